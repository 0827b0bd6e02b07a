// MXFP4: blocks of 32 values along a row share a power of two, a value is one of sixteen.
//
//   f = biased fp32 exponent of the block's largest magnitude, b = f == 255 ? 255 : max(f - 2, 0)
//   code = e2m1(x / 2^(b - 127)), ties to the even code, saturating; all codes 0 where b = 255 (the block holds an infinity or a NaN)
//
// Everything is exact up to the code's own rounding: the exponent is read from the bits of the maximum, the division is one by a power of
// two inside the conversion instruction (checked against the definition for every bf16 and fp16 value and millions of fp32 ones, subnormal ones
// and scales at both ends of the range among them).  The maximum is taken over the patterns without sign, where infinities and NaN are largest.
//
// Bound by HBM: a value is read once and becomes 17 / 32 bytes.  Along the rows a lane converts one vector of 16 bytes and the four lanes (fp32: eight)
// of a block join their maxima; rows whose length is a multiple of 32 are one flat array.  With the transposed copy of many values a lane holds 32 rows of one vector's
// columns in registers, which gives both directions from one read with no exchange but that of the maxima along the rows; eight lanes side by side and
// eight row blocks below each other make a wave, so that its loads and its transposed stores are whole 128-byte lines.
// Measured at 11000 x 7168 bf16: both directions 57 us (4.2 TB/s; without the stores of the row codes 47, without the transposed ones 45: two sets of
// writes beside the read are what is left), along the rows 33 (6.1 of values and codes together), back 29 (6.9), back from the transposed copy 38 (5.3).
// Other tiles of the two-way form (4 x 16 or 2 x 32 lanes, waves stacked instead of side by side) take 56 to 65 us, three waves to a SIMD the same 57.
#include "rows.hpp"

namespace fluxmi {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 32;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Lanes that share a block when each has one vector.
template <Row T>
constexpr int kShare = kBlock / kVec<T>;

// Running maximum over the magnitudes' patterns: of each half, or of the whole word.
template <Row T>
__device__ __forceinline__ uint32_t max_pattern(uint32_t a, uint32_t b) {
  if constexpr (T == Row::F32) return a > b ? a : b;
  else return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <Row T>
__device__ __forceinline__ uint32_t magnitude(uint32_t v) {
  return v & (T == Row::F32 ? 0x7fffffffu : 0x7fff7fffu);
}
template <Row T>
__device__ __forceinline__ uint32_t join_halves(uint32_t m) {
  if constexpr (T == Row::F32) return m;
  else return (m >> 16) > (m & 0xffffu) ? m >> 16 : m & 0xffffu;
}

// The maximum of 2, 4 or 8 neighbouring lanes, in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t max_of_lanes(uint32_t m) {
  auto with = [&](uint32_t o) { return m > o ? m : o; };
  m = with(__builtin_amdgcn_mov_dpp(m, 0xb1, 0xf, 0xf, false));                    // quad_perm [1,0,3,2]
  if constexpr (LANES >= 4) m = with(__builtin_amdgcn_mov_dpp(m, 0x4e, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
  if constexpr (LANES >= 8) m = with(__builtin_amdgcn_mov_dpp(m, 0x141, 0xf, 0xf, false));  // row_half_mirror: lane 7 - i of every 8
  return m;
}

// Scale byte of a block from the largest pattern of its magnitudes.
template <Row T>
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  uint32_t f;
  if constexpr (T == Row::F32) f = largest >> 23;
  else if constexpr (T == Row::BF16) f = largest >> 7;
  else f = __float_as_uint(f16_bits_to_float(static_cast<uint16_t>(largest))) >> 23;
  return f == 255 ? 255 : (f > 2 ? f - 2 : 0);
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7fc00000u : byte << 23));
}

// Two values (16-bit types: a pair in one word) to byte SEL of `old`.
template <Row T, int SEL>
__device__ __forceinline__ uint32_t convert2(uint32_t old, uint32_t pair, float scale) {
  if constexpr (T == Row::BF16) return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, pair), scale, SEL);
  else return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, pair), scale, SEL);
}
template <int SEL>
__device__ __forceinline__ uint32_t convert2f(uint32_t old, uint32_t lo, uint32_t hi, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, __uint_as_float(lo), __uint_as_float(hi), scale, SEL);
}

// A vector's codes: 4 bytes, fp32 the lower 2.
template <Row T>
__device__ __forceinline__ uint32_t convert_vector(const u32x4 v, float scale) {
  uint32_t c = 0;
  if constexpr (T == Row::F32) {
    c = convert2f<0>(c, v[0], v[1], scale);
    return convert2f<1>(c, v[2], v[3], scale);
  } else {
    c = convert2<T, 0>(c, v[0], scale);
    c = convert2<T, 1>(c, v[1], scale);
    c = convert2<T, 2>(c, v[2], scale);
    return convert2<T, 3>(c, v[3], scale);
  }
}

template <Row T>
__device__ __forceinline__ uint32_t vector_max(const u32x4 v) {
  uint32_t m = magnitude<T>(v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) m = max_pattern<T>(m, magnitude<T>(v[i]));
  return m;
}

// `count` elements (fewer than a vector) from p, zeros behind them.
template <Row T>
__device__ __forceinline__ u32x4 load_part(const uint8_t *p, int count) {
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) {
    if (i >= count) continue;
    if constexpr (T == Row::F32) v[i] = reinterpret_cast<const uint32_t *>(p)[i];
    else v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[i]) << (16 * (i & 1));
  }
  return v;
}

// ---- along the rows --------------------------------------------------------------------------------------------

template <Row T, bool NT>
__device__ __forceinline__ u32x4 load_vector(const uint8_t *p, int count) {
  return count >= kVec<T> ? load16<NT>(p) : load_part<T>(p, count);
}

// A vector's codes.
template <Row T>
__device__ __forceinline__ void store_codes(uint8_t *to, uint32_t c) {
  if constexpr (T == Row::F32) *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(c);
  else *reinterpret_cast<uint32_t *>(to) = c;
}

// One vector of the kShare of a block, in neighbouring lanes, all of which come here.
template <Row T>
__device__ __forceinline__ void quantise_vector(const u32x4 v, uint8_t *codes, uint8_t *scale, bool first_lane, bool stores = true) {
  const uint32_t byte = scale_byte<T>(max_of_lanes<kShare<T>>(join_halves<T>(vector_max<T>(v))));
  const uint32_t c = byte == 255 ? 0u : convert_vector<T>(v, scale_value(byte));
  if (!stores) return;
  store_codes<T>(codes, c);
  if (first_lane) *scale = static_cast<uint8_t>(byte);
}

// Rows of whole blocks: a vector to a lane, U of them in flight.
template <Row T, int U, bool NT>
__global__ __launch_bounds__(kThreads) void quant_flat_kernel(const uint8_t *__restrict__ x, size_t vectors, uint8_t *__restrict__ codes, uint8_t *__restrict__ scale) {
  const size_t at = static_cast<size_t>(blockIdx.x) * (kThreads * U) + threadIdx.x;
  u32x4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (at + u * kThreads < vectors) v[u] = load16<NT>(x + (at + u * kThreads) * 16);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = at + u * kThreads;
    if (i < vectors) quantise_vector<T>(v[u], codes + i * (kVec<T> / 2), scale + i / kShare<T>, (threadIdx.x & (kShare<T> - 1)) == 0);
  }
}

// Rows that end inside a block: a row to `1 << shift` lanes.
template <Row T, bool NT>
__global__ __launch_bounds__(kThreads) void quant_rows_kernel(const uint8_t *__restrict__ x, int64_t rows, int cols, int shift, uint8_t *__restrict__ codes,
                                                              uint8_t *__restrict__ scale) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads >> shift) + (threadIdx.x >> shift);
  if (row >= rows) return;
  const int vectors = (cols + kBlock - 1) / kBlock * kShare<T>;
  const uint8_t *const src = x + static_cast<size_t>(row) * cols * kElt<T>;
  for (int i = threadIdx.x & ((1 << shift) - 1); i < vectors; i += 1 << shift) {
    const size_t at = static_cast<size_t>(row) * vectors + i;
    quantise_vector<T>(load_vector<T, NT>(src + static_cast<size_t>(i) * 16, cols - i * kVec<T>), codes + at * (kVec<T> / 2), scale + at / kShare<T>,
                       (i & (kShare<T> - 1)) == 0);
  }
}

// ---- along the rows and along the columns -----------------------------------------------------------------------------

// One matrix of the batch, few values: a workgroup has 32 rows of 8 vectors, one to a thread, and reads them again from LDS by columns.  Its transposed stores are 16
// bytes from each column.
template <Row T>
__global__ __launch_bounds__(kThreads) void quant_tile_kernel(const uint8_t *__restrict__ x, int rows, int cols, int col_tiles, uint8_t *__restrict__ codes,
                                                              uint8_t *__restrict__ scale, uint8_t *__restrict__ codes_t, uint8_t *__restrict__ scale_t) {
  constexpr int V = kVec<T>, kPitch = 8 * 16 + 16;
  __shared__ __attribute__((aligned(16))) uint8_t tile[kBlock * kPitch];
  const int rt = blockIdx.x / col_tiles, ct = blockIdx.x - rt * col_tiles, kb = (cols + kBlock - 1) / kBlock, rb = (rows + kBlock - 1) / kBlock;
  const size_t matrix = static_cast<size_t>(blockIdx.y);
  {
    const int r = threadIdx.x >> 3, row = rt * kBlock + r, col = (ct * 8 + (threadIdx.x & 7)) * V;
    const size_t in_batch = matrix * rows + row, block = in_batch * kb + col / kBlock;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (row < rows && col < cols) v = load_vector<T, false>(x + (in_batch * cols + col) * kElt<T>, cols - col);
    *reinterpret_cast<u32x4 *>(tile + r * kPitch + (threadIdx.x & 7) * 16) = v;
    quantise_vector<T>(v, codes + block * 16 + col % kBlock / 2, scale + block, col % kBlock == 0, row < rows && col < kb * kBlock);
  }
  __syncthreads();
  const int c = threadIdx.x / kShare<T>, part = threadIdx.x % kShare<T>, col = ct * 8 * V + c;
  const uint8_t *const from = tile + part * V * kPitch + c * kElt<T>;
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (T == Row::F32) v[i] = *reinterpret_cast<const uint32_t *>(from + i * kPitch);
    else v[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(from + i * kPitch)) << (16 * (i & 1));
  }
  const size_t block = (matrix * cols + col) * rb + rt;
  quantise_vector<T>(v, codes_t + block * 16 + part * (V / 2), scale_t + block, part == 0, col < cols);
}

// One matrix of the batch.  A wave covers 8 vectors of columns x 8 blocks of 32 rows, a workgroup 4 waves side by side.
template <Row T, bool NT>
__global__ __launch_bounds__(kThreads, 2) void quant_both_kernel(const uint8_t *__restrict__ x, int rows, int cols, int row_tiles, int col_tiles,
                                                              uint8_t *__restrict__ codes, uint8_t *__restrict__ scale, uint8_t *__restrict__ codes_t,
                                                              uint8_t *__restrict__ scale_t) {
  constexpr int V = kVec<T>;
  // Neighbouring column tiles on one XCD (workgroups are dealt to the eight of them in turn): they share lines of the codes and of the scales.
  const int tiles = row_tiles * col_tiles, per_xcd = (tiles + 7) / 8, tile = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (static_cast<int>(blockIdx.x >> 3) >= per_xcd || tile >= tiles) return;
  const int rt = tile / col_tiles, ct = tile - rt * col_tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r0 = (rt * 8 + (lane >> 3)) * kBlock, c0 = ((ct * 4 + wave) * 8 + (lane & 7)) * V;
  const int kb = (cols + kBlock - 1) / kBlock, rb = (rows + kBlock - 1) / kBlock;
  const size_t matrix = static_cast<size_t>(blockIdx.y);
  x += matrix * rows * cols * kElt<T>;
  codes += matrix * rows * kb * 16;
  scale += matrix * rows * kb;
  codes_t += matrix * cols * rb * 16;
  scale_t += matrix * cols * rb;
  const int rows_here = rows - r0 < kBlock ? rows - r0 : kBlock, cols_here = cols - c0;  // (either may be negative)
  u32x4 v[kBlock];
  const uint8_t *const src = x + (static_cast<size_t>(r0) * cols + c0) * kElt<T>;
#pragma unroll
  for (int r = 0; r < kBlock; ++r) {
    v[r] = u32x4{0u, 0u, 0u, 0u};
    if (r < rows_here && cols_here > 0) {
      const uint8_t *const p = src + static_cast<size_t>(r) * cols * kElt<T>;
      v[r] = load_vector<T, NT>(p, cols_here);
    }
  }
  // Along the rows: kShare lanes have a block.
#pragma unroll
  for (int r = 0; r < kBlock; ++r) {
    const uint32_t byte = scale_byte<T>(max_of_lanes<kShare<T>>(join_halves<T>(vector_max<T>(v[r]))));
    const uint32_t c = byte == 255 ? 0u : convert_vector<T>(v[r], scale_value(byte));
    if (r < rows_here && c0 < kb * kBlock) {
      store_codes<T>(codes + (static_cast<size_t>(r0 + r) * kb * kBlock + c0) / 2, c);
      if ((lane & (kShare<T> - 1)) == 0) scale[static_cast<size_t>(r0 + r) * kb + c0 / kBlock] = static_cast<uint8_t>(byte);
    }
  }
  // Along the columns: 32 values of each are this lane's.
  u32x4 most = v[0];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    most[i] = magnitude<T>(v[0][i]);
#pragma unroll
    for (int r = 1; r < kBlock; ++r) most[i] = max_pattern<T>(most[i], magnitude<T>(v[r][i]));
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    uint32_t largest;
    if constexpr (T == Row::F32) largest = most[c];
    else largest = c & 1 ? most[c / 2] >> 16 : most[c / 2] & 0xffffu;
    const uint32_t byte = scale_byte<T>(largest);
    const float s = scale_value(byte);
    u32x4 o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w = 0;
      if constexpr (T == Row::F32) {
        w = convert2f<0>(w, v[8 * q][c], v[8 * q + 1][c], s);
        w = convert2f<1>(w, v[8 * q + 2][c], v[8 * q + 3][c], s);
        w = convert2f<2>(w, v[8 * q + 4][c], v[8 * q + 5][c], s);
        w = convert2f<3>(w, v[8 * q + 6][c], v[8 * q + 7][c], s);
      } else {
        // The column's halves of two rows to one word.
        auto pair = [&](int r) { return __builtin_amdgcn_perm(v[r + 1][c / 2], v[r][c / 2], c & 1 ? 0x07060302u : 0x05040100u); };
        w = convert2<T, 0>(w, pair(8 * q), s);
        w = convert2<T, 1>(w, pair(8 * q + 2), s);
        w = convert2<T, 2>(w, pair(8 * q + 4), s);
        w = convert2<T, 3>(w, pair(8 * q + 6), s);
      }
      o[q] = byte == 255 ? 0u : w;
    }
    if (rows_here > 0 && c < cols_here) {
      const size_t at = static_cast<size_t>(c0 + c) * rb + r0 / kBlock;
      store16(codes_t + at * 16, o);
      scale_t[at] = static_cast<uint8_t>(byte);
    }
  }
}

// ---- back ------------------------------------------------------------------------------------------------------

// A vector of values from its codes (4 bytes, fp32 the lower 2); `count` of them are there.
template <Row T, bool NT>
__device__ __forceinline__ void dequantise_vector(uint32_t c, uint32_t byte, uint8_t *out, int count) {
  const float s = scale_value(byte);
  u32x4 v;
  if constexpr (T == Row::F32) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    v = u32x4{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]), __float_as_uint(b[1])};
    if (byte == 255) v = u32x4{0x7fc00000u, 0x7fc00000u, 0x7fc00000u, 0x7fc00000u};
  } else if constexpr (T == Row::BF16) {
    v = u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
    if (byte == 255) v = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  } else {
    // Through fp32, which holds every value: the one rounding is that to fp16.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x2 p;
      if (i == 0) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
      else if (i == 1) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
      else if (i == 2) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
      else p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
      v[i] = float_to_f16_bits(p[0]) | static_cast<uint32_t>(float_to_f16_bits(p[1])) << 16;
    }
    if (byte == 255) v = u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
  }
  if (count >= kVec<T>) {
    store16<NT>(out, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec<T> - 1; ++i) {
    if (i >= count) continue;
    if constexpr (T == Row::F32) reinterpret_cast<uint32_t *>(out)[i] = v[i];
    else reinterpret_cast<uint16_t *>(out)[i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
  }
}

// Codes of vector i.
template <Row T>
__device__ __forceinline__ uint32_t load_codes(const uint8_t *codes, size_t i) {
  if constexpr (T == Row::F32) return reinterpret_cast<const uint16_t *>(codes)[i];
  else return reinterpret_cast<const uint32_t *>(codes)[i];
}

template <Row T, int U, bool NT>
__global__ __launch_bounds__(kThreads) void dequant_flat_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scale, size_t vectors, uint8_t *__restrict__ out) {
  const size_t at = static_cast<size_t>(blockIdx.x) * (kThreads * U) + threadIdx.x;
  uint32_t c[U], b[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = at + u * kThreads;
    if (i < vectors) {
      c[u] = load_codes<T>(codes, i);
      b[u] = scale[i / kShare<T>];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = at + u * kThreads;
    if (i < vectors) dequantise_vector<T, NT>(c[u], b[u], out + i * 16, kVec<T>);
  }
}

template <Row T, bool NT>
__global__ __launch_bounds__(kThreads) void dequant_rows_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scale, int64_t rows, int cols, int shift,
                                                                uint8_t *__restrict__ out) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads >> shift) + (threadIdx.x >> shift);
  if (row >= rows) return;
  const int vectors = (cols + kBlock - 1) / kBlock * kShare<T>;
  uint8_t *const dst = out + static_cast<size_t>(row) * cols * kElt<T>;
  for (int i = threadIdx.x & ((1 << shift) - 1); i * kVec<T> < cols; i += 1 << shift) {
    const size_t at = static_cast<size_t>(row) * vectors + i;
    dequantise_vector<T, NT>(load_codes<T>(codes, at), scale[at / kShare<T>], dst + static_cast<size_t>(i) * 16, cols - i * kVec<T>);
  }
}

// Lanes of a row that ends inside a block, as a power of two from one block's to 256.
template <Row T>
int row_shift(int64_t cols) {
  const int64_t vectors = (cols + kBlock - 1) / kBlock * kShare<T>;
  int shift = 2;
  while (shift < 8 && (int64_t{1} << shift) < vectors) ++shift;
  return shift;
}

// Workgroups of `items` work items, `per` to a workgroup; false: more than a launch has.
bool grid_of(int64_t items, int64_t per, dim3 *grid) {
  const int64_t n = (items + per - 1) / per;
  *grid = dim3(static_cast<unsigned>(n));
  return n * kThreads < (int64_t{1} << 32);
}

// From this many vectors on a lane has four of them in flight: below, one each spreads the work wider.
constexpr size_t kManyVectors = size_t{1} << 19;

// Values of this many bytes pass the caches by: they would only push out of them what is used again.
// Measured (us, ordinary and non-temporal), bf16 of 8192 columns: with both directions 25 and 23 at 64 MB, 41 and 35 at 96 MB, 104 and 96 at 256 MB;
// along the rows 14 and 16, 24 and 22, 59 and 53; back 15 and 13, 26 and 20, 60 and 49.  fp32 is alike.
constexpr size_t kStreamBytes = size_t{96} << 20;

// Up to so many values both directions go through LDS: many small workgroups, none of which waits for 32 loads of each lane.  Measured (us, in registers / through
// LDS): bf16 300 x 2048 9.8 / 2.7, 2800 x 4096 12.9 / 10.3, 4096 x 4096 14.9 / 13.2, 8192 x 4096 26 / 37; fp32 9.2 / 2.8, 17.4 / 14.1, 20.6 / 20.9, 43 / 43.  Rows
// that start inside lines: bf16 1024 x 7000 11.1 / 10.9, 4096 x 2800 12.8 / 13.0, 4100 x 5000 19 / 31; fp32 12.7 / 15.5, 17.2 / 17.0, 36 / 48.
template <Row T>
int64_t tile_values(int64_t cols) {
  return int64_t{1} << (cols * kElt<T> % 128 == 0 ? 24 : 22);
}

int check_sizes(const char *who, int64_t rows, int64_t cols) {
  FLUXMI_REQUIRE(rows >= 0 && cols >= 0, FLUXMI_ERR_INVALID_ARG, "%s: negative size (rows=%lld, cols=%lld)", who, static_cast<long long>(rows),
                 static_cast<long long>(cols));
  FLUXMI_REQUIRE(cols <= (int64_t{1} << 30), FLUXMI_ERR_UNSUPPORTED, "%s: cols=%lld exceeds 2^30", who, static_cast<long long>(cols));
  FLUXMI_REQUIRE(cols == 0 || rows <= (int64_t{1} << 40) / cols, FLUXMI_ERR_UNSUPPORTED, "%s: more than 2^40 values", who);
  return FLUXMI_OK;
}

}  // namespace
}  // namespace fluxmi

extern "C" int fluxmi_quant_mx(const void *x, int32_t row_type, int64_t batch, int64_t rows, int64_t cols, void *codes, void *scale, void *codes_t, void *scale_t,
                               void *stream) {
  using namespace fluxmi;
  Row type;
  int rc = check_type("quant_mx", row_type, &type);
  if (rc == FLUXMI_OK) rc = check_sizes("quant_mx", rows, cols);
  if (rc != FLUXMI_OK) return rc;
  FLUXMI_REQUIRE(batch >= 0 && batch <= 65535, FLUXMI_ERR_INVALID_ARG, "quant_mx: batch=%lld outside [0,65535]", static_cast<long long>(batch));
  FLUXMI_REQUIRE((codes_t == nullptr) == (scale_t == nullptr), FLUXMI_ERR_INVALID_ARG, "quant_mx: codes_t and scale_t go together");
  if (batch == 0 || rows == 0 || cols == 0) return FLUXMI_OK;
  rc = check_sizes("quant_mx", batch * rows, cols);
  if (rc != FLUXMI_OK) return rc;
  FLUXMI_REQUIRE(x != nullptr && codes != nullptr && scale != nullptr, FLUXMI_ERR_INVALID_ARG, "quant_mx: null pointer argument");
  FLUXMI_REQUIRE(aligned_to(x, type) && (reinterpret_cast<uintptr_t>(codes) & 3) == 0 && aligned16(codes_t), FLUXMI_ERR_INVALID_ARG,
                 "quant_mx: x is not aligned to its elements, codes to 4 or codes_t to 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto *const in = static_cast<const uint8_t *>(x);
  auto *const q = static_cast<uint8_t *>(codes), *const sc = static_cast<uint8_t *>(scale);
  dim3 grid;
  bool fits = true;
  auto launch = [&](auto t, auto nt) {
    constexpr Row T = decltype(t)::value;
    constexpr bool NT = decltype(nt)::value;
    if (codes_t != nullptr) {
      if constexpr (!NT) {
        if (batch * rows * cols <= tile_values<T>(cols)) {
          const int64_t row_tiles = (rows + kBlock - 1) / kBlock, col_tiles = (cols + 8 * kVec<T> - 1) / (8 * kVec<T>);
          fits = grid_of(row_tiles * col_tiles, 1, &grid);
          if (!fits) return;
          grid.y = static_cast<unsigned>(batch);
          hipLaunchKernelGGL(quant_tile_kernel<T>, grid, dim3(kThreads), 0, s, in, static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(col_tiles), q, sc,
                             static_cast<uint8_t *>(codes_t), static_cast<uint8_t *>(scale_t));
          return;
        }
      }
      const int64_t row_tiles = (rows + 8 * kBlock - 1) / (8 * kBlock), col_tiles = (cols + 32 * kVec<T> - 1) / (32 * kVec<T>);
      fits = grid_of((row_tiles * col_tiles + 7) / 8 * 8, 1, &grid) && row_tiles * col_tiles < (int64_t{1} << 23);
      if (!fits) return;
      grid.y = static_cast<unsigned>(batch);
      hipLaunchKernelGGL((quant_both_kernel<T, NT>), grid, dim3(kThreads), 0, s, in, static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(row_tiles),
                         static_cast<int>(col_tiles), q, sc, static_cast<uint8_t *>(codes_t), static_cast<uint8_t *>(scale_t));
    } else if (cols % kBlock == 0) {
      const size_t vectors = static_cast<size_t>(batch * rows) * cols / kVec<T>;
      const bool many = vectors >= kManyVectors;
      fits = grid_of(vectors, kThreads * (many ? 4 : 1), &grid);
      if (!fits) return;
      if (many) hipLaunchKernelGGL((quant_flat_kernel<T, 4, NT>), grid, dim3(kThreads), 0, s, in, vectors, q, sc);
      else if constexpr (!NT) hipLaunchKernelGGL((quant_flat_kernel<T, 1, false>), grid, dim3(kThreads), 0, s, in, vectors, q, sc);
    } else {
      const int shift = row_shift<T>(cols);
      fits = grid_of(batch * rows, kThreads >> shift, &grid);
      if (fits) hipLaunchKernelGGL((quant_rows_kernel<T, NT>), grid, dim3(kThreads), 0, s, in, batch * rows, static_cast<int>(cols), shift, q, sc);
    }
  };
  if (codes_t != nullptr)
    FLUXMI_REQUIRE(rows <= (int64_t{1} << 30), FLUXMI_ERR_UNSUPPORTED, "quant_mx: rows=%lld exceeds 2^30 with a transposed copy", static_cast<long long>(rows));
  const bool streamed = static_cast<size_t>(batch * rows) * cols * (type == Row::F32 ? 4 : 2) >= kStreamBytes;
  by_type(type, [&](auto t) {
    if (streamed) launch(t, std::true_type{});
    else launch(t, std::false_type{});
  });
  FLUXMI_REQUIRE(fits, FLUXMI_ERR_UNSUPPORTED, "quant_mx: batch=%lld rows=%lld cols=%lld is more than a launch covers", static_cast<long long>(batch),
                 static_cast<long long>(rows), static_cast<long long>(cols));
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}

extern "C" int fluxmi_dequant_mx(const void *codes, const void *scale, int64_t rows, int64_t cols, int32_t row_type, void *out, void *stream) {
  using namespace fluxmi;
  Row type;
  int rc = check_type("dequant_mx", row_type, &type);
  if (rc == FLUXMI_OK) rc = check_sizes("dequant_mx", rows, cols);
  if (rc != FLUXMI_OK) return rc;
  if (rows == 0 || cols == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(codes != nullptr && scale != nullptr && out != nullptr, FLUXMI_ERR_INVALID_ARG, "dequant_mx: null pointer argument");
  FLUXMI_REQUIRE(aligned_to(out, type) && (reinterpret_cast<uintptr_t>(codes) & 3) == 0, FLUXMI_ERR_INVALID_ARG,
                 "dequant_mx: out is not aligned to its elements or codes to 4 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto *const q = static_cast<const uint8_t *>(codes), *const sc = static_cast<const uint8_t *>(scale);
  auto *const o = static_cast<uint8_t *>(out);
  dim3 grid;
  bool fits = true;
  auto launch = [&](auto t, auto nt) {
    constexpr Row T = decltype(t)::value;
    constexpr bool NT = decltype(nt)::value;
    if (cols % kBlock == 0) {
      const size_t vectors = static_cast<size_t>(rows) * cols / kVec<T>;
      const bool many = vectors >= kManyVectors;
      fits = grid_of(vectors, kThreads * (many ? 4 : 1), &grid);
      if (!fits) return;
      if (many) hipLaunchKernelGGL((dequant_flat_kernel<T, 4, NT>), grid, dim3(kThreads), 0, s, q, sc, vectors, o);
      else if constexpr (!NT) hipLaunchKernelGGL((dequant_flat_kernel<T, 1, false>), grid, dim3(kThreads), 0, s, q, sc, vectors, o);
    } else {
      const int shift = row_shift<T>(cols);
      fits = grid_of(rows, kThreads >> shift, &grid);
      if (fits) hipLaunchKernelGGL((dequant_rows_kernel<T, NT>), grid, dim3(kThreads), 0, s, q, sc, rows, static_cast<int>(cols), shift, o);
    }
  };
  const bool streamed = static_cast<size_t>(rows) * cols * (type == Row::F32 ? 4 : 2) >= kStreamBytes;
  by_type(type, [&](auto t) {
    if (streamed) launch(t, std::true_type{});
    else launch(t, std::false_type{});
  });
  FLUXMI_REQUIRE(fits, FLUXMI_ERR_UNSUPPORTED, "dequant_mx: rows=%lld cols=%lld is more than a launch covers", static_cast<long long>(rows), static_cast<long long>(cols));
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}
