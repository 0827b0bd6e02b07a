// Activation checkpoints in 8 bits, and the gated activation between an expert's two products.
//
//   block of 32 values of a row, m its largest magnitude, f the biased fp32 exponent of m:
//     b = 255 and codes 0 where the block holds an infinity or a NaN, else max(f - 8 + (m > 1.75 * 2^(f - 127)), 0): the least scale
//         2^(b - 127) with m <= 448 times the scale, so that no code saturates
//     code = e4m3(x / 2^(b - 127)), ties to even; x beyond 15/8 times the type's largest power of two counts as that much, because the next code
//         up stands for a value that the type does not hold
//   out = silu(g) u, silu(g) = g s, s = 1 / (1 + exp(-g))
//   backwards, d the gradient of out: dg = d u s (1 + g (1 - s)), du = d g s
//
// All of it is fp32 inside, with one rounding to 16 bits at the end; values of a checkpoint are exact in fp32, scales and codes are exact up to the
// code's own rounding.
//
// Memory bounds all of it: every byte is read and written once.  A lane has eight values of a row (16 bytes in, 8 out), four lanes a block, whose maximum they find among
// themselves; rows of any length and start, whole vectors wherever eight values are left.  Of MI355X's 8 TB/s (a copy reaches 5.6, reading alone 6.9): swiglu with a checkpoint of
// 16384 x 2 x 14336 bf16 304 us, 6.2 TB/s, without one 227, 6.2; its gradient from 8 bits 384 us, 6.1 TB/s, from 16 bits 494, 5.7; a checkpoint of 16384 x 4096 39 us, 5.3 TB/s; calls below 10 MB take 5 to 6 us, which is the
// way through the call and not the memory.
#include "rows.hpp"

namespace fluxmi {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 32;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

// Largest magnitude that a code may stand for: 15/8 times the type's largest power of two, as a pattern of the type.
template <Row T>
constexpr uint32_t kLargest = T == Row::BF16 ? 0x7f70u : 0x7b80u;

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7fc00000u : byte << 23));
}

// The maximum of 4 neighbouring lanes, in each of them.
__device__ __forceinline__ uint32_t max_of_4_lanes(uint32_t m) {
  auto with = [&](uint32_t o) { return m > o ? m : o; };
  m = with(__builtin_amdgcn_mov_dpp(m, 0xb1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  m = with(__builtin_amdgcn_mov_dpp(m, 0x4e, 0xf, 0xf, false));  // quad_perm [2,3,0,1]
  return m;
}

// The largest pattern without sign of a vector's eight values.
template <Row T>
__device__ __forceinline__ uint32_t vector_max(const u32x4 v) {
  u16x2 m = __builtin_bit_cast(u16x2, v[0] & 0x7fff7fffu);
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
  return m[0] > m[1] ? m[0] : m[1];
}

template <Row T>
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  const uint32_t bits = T == Row::BF16 ? largest << 16 : __float_as_uint(f16_bits_to_float(static_cast<uint16_t>(largest)));
  const uint32_t f = bits >> 23, b = f + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return f == 255 ? 255 : (b > 8 ? b - 8 : 0);
}

// Eight codes.
template <Row T>
__device__ __forceinline__ u32x2 codes_of(const u32x4 v, uint32_t byte) {
  u32x2 c;
  const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte << 23);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t pair[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t w = v[2 * i + j], a = w & 0x7fff7fffu;
      const u16x2 most = {static_cast<uint16_t>(kLargest<T>), static_cast<uint16_t>(kLargest<T>)};
      pair[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), most)) | (w & 0x80008000u);
    }
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 two = {0, 0};
    if constexpr (T == Row::BF16) {
      two = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(two, __builtin_bit_cast(bf16x2, pair[0]), scale, false);
      two = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(two, __builtin_bit_cast(bf16x2, pair[1]), scale, true);
    } else {
      two = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(two, __builtin_bit_cast(f16x2, pair[0]), scale, false);
      two = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(two, __builtin_bit_cast(f16x2, pair[1]), scale, true);
    }
    c[i] = byte == 255 ? 0u : __builtin_bit_cast(uint32_t, two);
  }
  return c;
}

// `count` of a vector's eight values, zeros behind them; all of them where count >= 8.
template <Row T, bool NT>
__device__ __forceinline__ u32x4 load_some(const uint8_t *p, int count) {
  if (count >= 8) return load16<NT>(p);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[i]) << (16 * (i & 1));
  return v;
}
template <bool NT>
__device__ __forceinline__ void store_some(uint8_t *p, const u32x4 v, int count) {
  if (count >= 8) {
    store16<NT>(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < count) reinterpret_cast<uint16_t *>(p)[i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
}
template <bool NT>
__device__ __forceinline__ u32x2 load_codes(const uint8_t *p, int count) {
  if (count >= 8) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x2_any *>(p));
    else return *reinterpret_cast<const u32x2_any *>(p);
  }
  u32x2 v = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) v[i / 4] |= static_cast<uint32_t>(p[i]) << (8 * (i & 3));
  return v;
}
template <bool NT>
__device__ __forceinline__ void store_codes(uint8_t *p, const u32x2 c, int count) {
  if (count >= 8) {
    if constexpr (NT) __builtin_nontemporal_store(c, reinterpret_cast<u32x2_any *>(p));
    else *reinterpret_cast<u32x2_any *>(p) = c;
    return;
  }
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < count) p[i] = static_cast<uint8_t>(c[i / 4] >> (8 * (i & 3)));
}

// Eight codes' values.
__device__ __forceinline__ void values_of(const u32x2 c, uint32_t byte, float (&x)[8]) {
  const float scale = scale_value(byte);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], true);
    x[4 * i] = lo[0] * scale;
    x[4 * i + 1] = lo[1] * scale;
    x[4 * i + 2] = hi[0] * scale;
    x[4 * i + 3] = hi[1] * scale;
  }
}

__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// ---- a row's vectors -----------------------------------------------------------------------------------------
// A group of 2^lanes_log lanes has a row, or a piece of one where a row has more vectors than a workgroup has lanes.  Lane l of the group has the
// vectors l, l + lanes, .. of the piece; four neighbouring lanes have a block.
struct RowsArgs {
  const uint8_t *x, *grad;
  const uint8_t *in_scale;
  uint8_t *out, *grad_x;
  uint8_t *codes, *scale;
  int64_t rows;
  int32_t cols;    // of one half
  int32_t blocks;  // of one half: ceil(cols / 32)
  int32_t lanes_log, pieces, pad;
};

struct Place {
  int64_t row;
  int col;  // first of a vector's columns
  bool any;
};
__device__ __forceinline__ Place place_of(const RowsArgs &a) {
  const int group = threadIdx.x >> a.lanes_log, lane = threadIdx.x & ((1 << a.lanes_log) - 1);
  const int64_t item = static_cast<int64_t>(blockIdx.x) / a.pieces;
  const int piece = static_cast<int>(blockIdx.x - item * a.pieces);
  Place p;
  p.row = item * (kThreads >> a.lanes_log) + group;
  p.col = ((piece << a.lanes_log) + lane) * 8;
  p.any = p.row < a.rows && p.col < a.blocks * kBlock;
  return p;
}

template <Row T, bool GATED, bool KEEP, int PASS>
__global__ __launch_bounds__(kThreads) void checkpoint_kernel(const RowsArgs a) {
  const Place p = place_of(a);
  if (!p.any) return;  // (whole blocks of four lanes)
  const int count = a.cols - p.col;
  constexpr int halves = GATED ? 2 : 1;
  const uint8_t *x = a.x + (p.row * halves * a.cols + p.col) * 2;
  u32x4 v[halves];
#pragma unroll
  for (int h = 0; h < halves; ++h) v[h] = count > 0 ? load_some<T, PASS == 2>(x + static_cast<int64_t>(h) * a.cols * 2, count) : u32x4{0u, 0u, 0u, 0u};
  if constexpr (KEEP) {
#pragma unroll
    for (int h = 0; h < halves; ++h) {
      const uint32_t byte = scale_byte<T>(max_of_4_lanes(vector_max<T>(v[h])));
      if (count > 0) store_codes<PASS != 0>(a.codes + (p.row * halves + h) * a.cols + p.col, codes_of<T>(v[h], byte), count);
      if ((p.col & (kBlock - 1)) == 0) a.scale[(p.row * halves + h) * a.blocks + (p.col >> 5)] = static_cast<uint8_t>(byte);
    }
  }
  if constexpr (GATED) {
    if (count <= 0) return;
    float g[8], u[8], o[8];
    unpack<T>(v[0], g);
    unpack<T>(v[1], u);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = g[i] * sigmoid(g[i]) * u[i];
    store_some<PASS != 0>(a.out + (p.row * a.cols + p.col) * 2, pack<T>(o), count);
  }
}

// KEPT: from codes and scales, otherwise from 16 bits.  Without a gradient: the activation alone.
template <Row T, bool KEPT, int PASS>
__global__ __launch_bounds__(kThreads) void swiglu_backward_kernel(const RowsArgs a) {
  const Place p = place_of(a);
  const int count = a.cols - p.col;
  if (!p.any || count <= 0) return;
  float g[8], u[8], d[8], dg[8], du[8], o[8];
  if constexpr (KEPT) {
    const uint8_t *c = a.x + p.row * 2 * a.cols + p.col, *s = a.in_scale + p.row * 2 * a.blocks + (p.col >> 5);
    const u32x2 cg = load_codes<PASS == 2>(c, count), cu = load_codes<PASS == 2>(c + a.cols, count);
    values_of(cg, s[0], g);
    values_of(cu, s[a.blocks], u);
  } else {
    const uint8_t *x = a.x + (p.row * 2 * a.cols + p.col) * 2;
    unpack<T>(load_some<T, PASS == 2>(x, count), g);
    unpack<T>(load_some<T, PASS == 2>(x + static_cast<int64_t>(a.cols) * 2, count), u);
  }
  const int64_t at = (p.row * a.cols + p.col) * 2;
  if (a.grad == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = g[i] * sigmoid(g[i]) * u[i];
    store_some<PASS != 0>(a.out + at, pack<T>(o), count);
    return;
  }
  unpack<T>(load_some<T, PASS == 2>(a.grad + at, count), d);
  // Gradient times value comes first: times the slope of a gate that closes, a small gradient would be below fp32.  Only where gradient times value is beyond fp32 the slope
  // comes in between: there the gradient is over 1, and its product with a slope is in range.
  float slope[8], most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = sigmoid(g[i]), silu = g[i] * s, ud = d[i] * u[i];
    o[i] = silu * u[i];
    du[i] = d[i] * silu;
    slope[i] = s * (1.f + g[i] * (1.f - s));
    dg[i] = ud * slope[i];
    most = fmaxf(most, fabsf(ud));
  }
  if (most == INFINITY) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(d[i] * u[i]) == INFINITY) dg[i] = d[i] * slope[i] * u[i];
  }
  uint8_t *gx = a.grad_x + (p.row * 2 * a.cols + p.col) * 2;
  store_some<PASS != 0>(gx, pack<T>(dg), count);
  store_some<PASS != 0>(gx + static_cast<int64_t>(a.cols) * 2, pack<T>(du), count);
  if (a.out != nullptr) store_some<PASS != 0>(a.out + at, pack<T>(o), count);
}

// ---- host ----------------------------------------------------------------------------------------------------
int check_rows(const char *who, int32_t type, int64_t rows, int64_t cols, Row *row) {
  FLUXMI_REQUIRE(type == FLUXMI_ROWS_BF16 || type == FLUXMI_ROWS_FP16, FLUXMI_ERR_INVALID_ARG, "%s: type %d (bf16 and fp16 are built)", who, type);
  FLUXMI_REQUIRE(rows >= 0 && cols >= 0, FLUXMI_ERR_INVALID_ARG, "%s: negative rows or columns", who);
  FLUXMI_REQUIRE(cols <= (1 << 30), FLUXMI_ERR_UNSUPPORTED, "%s: more than 2^30 columns", who);
  *row = type == FLUXMI_ROWS_BF16 ? Row::BF16 : Row::F16;
  return FLUXMI_OK;
}

bool even(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

// Lanes and workgroups; *blocks = 0: nothing to do.
int plan_rows(const char *who, RowsArgs *a, uint32_t *grid) {
  *grid = 0;
  if (a->rows == 0 || a->cols == 0) return FLUXMI_OK;
  a->blocks = (a->cols + kBlock - 1) / kBlock;
  const int vectors = a->blocks * 4;
  a->lanes_log = 2;
  while (a->lanes_log < 8 && (1 << a->lanes_log) < vectors) ++a->lanes_log;
  a->pieces = (vectors + (1 << a->lanes_log) - 1) >> a->lanes_log;
  const int per = kThreads >> a->lanes_log;
  const int64_t groups = (a->rows + per - 1) / per;
  FLUXMI_REQUIRE(groups <= ((int64_t{1} << 32) / kThreads - 1) / a->pieces, FLUXMI_ERR_UNSUPPORTED, "%s: too many rows for one launch", who);
  *grid = static_cast<uint32_t>(groups * a->pieces);
  return FLUXMI_OK;
}

// f(type, PASS): 0, or results pass the caches by (1), or inputs as well (2).  A call of `bytes` in all; us with 0 / 1 / 2: swiglu with a checkpoint 16384 x 14336 339 / 326 / 304, 16384 x 4096
// 94 / 78 / 87, 20000 x 1407 41 / 42 / 60; its gradient from 8 bits 414 / 392 / 386, 115 / 98 / 108, 89 / 56 / 86.  Inputs of a few hundred MB are still cached where they
// were just made, and rows that do not start on lines would be fetched twice.
// Around 96 MiB results in the caches are what a reader right behind the call gains by: 4096 columns, a call alone on inputs from memory and with a read of its results, 0 / 1: with a checkpoint 48 MiB
// 12.7 / 11.5 and 15.2 / 15.6, 96 MiB 20.4 / 19.6 and 24.2 / 25.2, 192 MiB 37.3 / 35.6 and 42.1 / 44.7; gradient from 16 bits 11.8 / 9.9 and 20.6 / 20.6, 22.5 / 19.6 and 30.5 / 30.9, 39.0 / 36.4 and
// 51.4 / 55.0; checkpoint alone 12.4 / 12.0 and 15.7 / 16.4, 21.9 / 21.1 and 27.4 / 28.0, 39.2 / 38.4 and 48.7 / 50.1.  From 1 GiB on, 0 / 1 / 2 of 1100 MiB, alone: 198 / 191 / 184, 200 / 196 / 189, 199 / 202 / 202.
template <class F>
void by_half(Row t, int64_t bytes, int32_t cols, F &&f) {
  const int pass = bytes < (int64_t{96} << 20) ? 0 : (bytes < (int64_t{1} << 30) || cols % 64 != 0 ? 1 : 2);
  auto with = [&](auto T) {
    if (pass == 0) f(T, std::integral_constant<int, 0>{});
    else if (pass == 1) f(T, std::integral_constant<int, 1>{});
    else f(T, std::integral_constant<int, 2>{});
  };
  if (t == Row::BF16) with(std::integral_constant<Row, Row::BF16>{});
  else with(std::integral_constant<Row, Row::F16>{});
}

}  // namespace
}  // namespace fluxmi

using namespace fluxmi;

extern "C" int fluxmi_checkpoint_e4m3(const void *x, int32_t row_type, int64_t rows, int64_t cols, void *codes, void *scale, void *stream) {
  Row type;
  if (const int rc = check_rows("checkpoint_e4m3", row_type, rows, cols, &type)) return rc;
  RowsArgs a{};
  a.rows = rows;
  a.cols = static_cast<int32_t>(cols);
  uint32_t grid;
  if (const int rc = plan_rows("checkpoint_e4m3", &a, &grid)) return rc;
  if (grid == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(x && codes && scale, FLUXMI_ERR_INVALID_ARG, "checkpoint_e4m3: null pointer");
  FLUXMI_REQUIRE(even(x), FLUXMI_ERR_INVALID_ARG, "checkpoint_e4m3: x is not aligned to its elements");
  a.x = static_cast<const uint8_t *>(x);
  a.codes = static_cast<uint8_t *>(codes);
  a.scale = static_cast<uint8_t *>(scale);
  by_half(type, rows * cols * 3, a.cols, [&](auto T, auto PASS) {
    checkpoint_kernel<decltype(T)::value, false, true, decltype(PASS)::value><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  });
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}

extern "C" int fluxmi_swiglu(const void *x, int32_t row_type, int64_t rows, int64_t cols, void *out, void *codes, void *scale, void *stream) {
  Row type;
  if (const int rc = check_rows("swiglu", row_type, rows, cols, &type)) return rc;
  RowsArgs a{};
  a.rows = rows;
  a.cols = static_cast<int32_t>(cols);
  uint32_t grid;
  if (const int rc = plan_rows("swiglu", &a, &grid)) return rc;
  if (grid == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(x && out, FLUXMI_ERR_INVALID_ARG, "swiglu: null pointer");
  FLUXMI_REQUIRE((codes == nullptr) == (scale == nullptr), FLUXMI_ERR_INVALID_ARG, "swiglu: codes and scale come together");
  FLUXMI_REQUIRE(even(x) && even(out), FLUXMI_ERR_INVALID_ARG, "swiglu: a pointer is not aligned to its elements");
  a.x = static_cast<const uint8_t *>(x);
  a.out = static_cast<uint8_t *>(out);
  a.codes = static_cast<uint8_t *>(codes);
  a.scale = static_cast<uint8_t *>(scale);
  by_half(type, rows * cols * (codes != nullptr ? 8 : 6), a.cols, [&](auto T, auto PASS) {
    if (codes != nullptr) checkpoint_kernel<decltype(T)::value, true, true, decltype(PASS)::value><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
    else checkpoint_kernel<decltype(T)::value, true, false, decltype(PASS)::value><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  });
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}

extern "C" int fluxmi_swiglu_backward(const void *grad, const void *x, const void *x_scale, int32_t row_type, int64_t rows, int64_t cols, void *grad_x,
                                      void *out, void *stream) {
  Row type;
  if (const int rc = check_rows("swiglu_backward", row_type, rows, cols, &type)) return rc;
  RowsArgs a{};
  a.rows = rows;
  a.cols = static_cast<int32_t>(cols);
  uint32_t grid;
  if (const int rc = plan_rows("swiglu_backward", &a, &grid)) return rc;
  if (grid == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(x && (grad || out) && (grad != nullptr) == (grad_x != nullptr), FLUXMI_ERR_INVALID_ARG, "swiglu_backward: null pointer");
  FLUXMI_REQUIRE(even(grad) && (x_scale != nullptr || even(x)) && even(grad_x) && even(out), FLUXMI_ERR_INVALID_ARG,
                 "swiglu_backward: a pointer is not aligned to its elements");
  a.grad = static_cast<const uint8_t *>(grad);
  a.x = static_cast<const uint8_t *>(x);
  a.in_scale = static_cast<const uint8_t *>(x_scale);
  a.grad_x = static_cast<uint8_t *>(grad_x);
  a.out = static_cast<uint8_t *>(out);
  by_half(type, rows * cols * ((x_scale != nullptr ? 2 : 4) + (grad != nullptr ? 8 : 2)), a.cols, [&](auto T, auto PASS) {
    if (x_scale != nullptr) swiglu_backward_kernel<decltype(T)::value, true, decltype(PASS)::value><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
    else swiglu_backward_kernel<decltype(T)::value, false, decltype(PASS)::value><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  });
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}
