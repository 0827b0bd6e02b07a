// Tokens to the rows of their experts and back, with the gradients of both:
//
//   permute             rows[idx[t, j]] = x[t]; rows that no pair names are zeros
//   unpermute           out[t] = sum_j w[t, j] * rows[idx[t, j]]            (w = 1: the gradient of permute)
//   unpermute backward  grad_rows[idx[t, j]] = w[t, j] * g[t], rows that no pair names zeros;  grad_w[t, j] = <g[t], rows[idx[t, j]]>
//
// Bound by HBM.  All three go through the tokens and not through the rows: a token's own row is then read or written once in the whole
// launch, and the top-k rows once each, which is what the operators cannot do without; going through the rows would read x and g top-k
// times.  Groups of 8 to 256 lanes share a token, every lane moves 16-byte vectors at whatever alignment the rows have (the last one of a
// width that leaves a rest ends with the row and overlaps the one before it, 777 tokens top-8 2047 columns 8.5 -> 6.5 us; the backward pass, whose products would
// count twice, and rows shorter than a vector go by elements there), and a vector's top-k rows are requested before the first of them is used.
//
// Rows without a pair: the first workgroups of a launch that writes rows own a range of them each, read all of idx (4 bytes a pair, beside
// rows of kilobytes), mark in LDS which of their rows are named, and clear the others.  That needs neither a pass over the output before
// the launch nor the splits, and holds for any distinct indices, wherever they leave rows out.
#include "rows.hpp"

namespace fluxmi {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTopk = 64;
constexpr int kRowsOfClearer = 65536;  // most rows that one clearing workgroup owns: a bit each in 8 KiB of LDS

// The experts' rows are moved non-temporally (NT) from this size on, twice what the L2s hold; the tokens' own rows never.  us, ordinary -> NT, three
// sets of buffers in turn: permute 16384 tokens top-6 2048 columns 94 -> 81, 8192 top-2 4096 columns 42 -> 30; unpermute of the latter 41 -> 35,
// 4096 top-8 7168 columns 113 -> 99, its backward pass 212 -> 197, that of the
// former 71 -> 57.  Below, ordinary loads are the faster ones (the backward pass of 1000 top-4 1536 fp32 columns 13.1
// against 14.5).
constexpr size_t kStreamBytes = size_t{64} << 20;

__device__ __forceinline__ float load_as(const void *p, Row type, size_t i) {
  if (type == Row::F32) return static_cast<const float *>(p)[i];
  const uint16_t b = static_cast<const uint16_t *>(p)[i];
  return type == Row::F16 ? f16_bits_to_float(b) : bf16_bits_to_float(b);
}

__device__ __forceinline__ void store_as(void *p, Row type, size_t i, float v) {
  if (type == Row::F32) static_cast<float *>(p)[i] = v;
  else static_cast<uint16_t *>(p)[i] = type == Row::F16 ? float_to_f16_bits(v) : float_to_bf16_bits(v);
}

// The part of a launch that a workgroup computes: group of `1 << shift` lanes -> token.
struct Lanes {
  int token, lane, count;
};

// SUB: several tokens to a wave; otherwise the token is the same for all lanes of a wave, and so are the row indices.
template <bool SUB>
__device__ __forceinline__ Lanes my_token(int block, int shift) {
  const int group = threadIdx.x >> shift;
  return {block * (kThreads >> shift) + (SUB ? group : __builtin_amdgcn_readfirstlane(group)), static_cast<int>(threadIdx.x) & ((1 << shift) - 1), 1 << shift};
}

// Clears the rows of its range that no pair names.
__device__ void clear_unnamed(int clearer, int clearers, const int32_t *__restrict__ idx, int npairs, size_t row_bytes, uint8_t *__restrict__ rows) {
  __shared__ uint32_t named[kRowsOfClearer / 32];
  const int per = ((npairs + clearers - 1) / clearers + 31) & ~31, first = clearer * per;
  const int count = npairs - first < per ? npairs - first : per;
  if (count <= 0) return;
  const int words = (count + 31) >> 5;
  for (int i = threadIdx.x; i < words; i += kThreads) named[i] = 0;
  __syncthreads();
  const int quads = npairs >> 2;
  auto mark = [&](uint32_t row) {
    const uint32_t r = row - static_cast<uint32_t>(first);
    if (r < static_cast<uint32_t>(count)) atomicOr(&named[r >> 5], 1u << (r & 31));
  };
  for (int q0 = threadIdx.x; q0 < quads; q0 += 8 * kThreads) {
    u32x4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int q = q0 + u * kThreads;
      v[u] = q < quads ? load16(reinterpret_cast<const uint8_t *>(idx) + static_cast<size_t>(q) * 16) : u32x4{~0u, ~0u, ~0u, ~0u};
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) mark(v[u][i]);
  }
  if (static_cast<int>(threadIdx.x) < npairs - 4 * quads) mark(idx[4 * quads + threadIdx.x]);
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int w = 0; w < words; ++w) {
    uint32_t missing = ~static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(named[w])) & (0x11111111u << wave);
    if (count - w * 32 < 32) missing &= (1u << (count - w * 32)) - 1u;
    while (missing != 0) {
      const int bit = __ffs(missing) - 1;
      missing &= missing - 1;
      uint8_t *const dst = rows + static_cast<size_t>(first + w * 32 + bit) * row_bytes;
      const size_t nvec = row_bytes >> 4;
      for (size_t v = lane; v < nvec; v += 64) store16(dst + v * 16, u32x4{0u, 0u, 0u, 0u});
      for (size_t b = nvec * 16 + lane; b < row_bytes; b += 64) dst[b] = 0;
    }
  }
}

// Rows of `size` in vectors of `vec`: how many, and where the v-th begins.
__device__ __forceinline__ int vectors_of(int size, int vec) { return size < vec ? 0 : (size - 1) / vec + 1; }
__device__ __forceinline__ int vector_at(int v, int size, int vec) { return v < size / vec ? v * vec : size - vec; }

template <bool SUB, bool NT>
__global__ __launch_bounds__(kThreads) void permute_kernel(const uint8_t *__restrict__ in, const int32_t *__restrict__ idx, int ntokens, int topk,
                                                           size_t row_bytes, int shift, int clearers, uint8_t *__restrict__ rows) {
  const int npairs = ntokens * topk;
  if (static_cast<int>(blockIdx.x) < clearers) {
    clear_unnamed(blockIdx.x, clearers, idx, npairs, row_bytes, rows);
    return;
  }
  const Lanes me = my_token<SUB>(blockIdx.x - clearers, shift);
  if (me.token >= ntokens) return;
  constexpr int U = 4;
  const uint8_t *const src = in + static_cast<size_t>(me.token) * row_bytes;
  const int32_t *const my_idx = idx + static_cast<size_t>(me.token) * topk;
  const size_t nvec = row_bytes < 16 ? 0 : (row_bytes + 15) >> 4;
  for (size_t v0 = me.lane; v0 < nvec; v0 += U * me.count) {
    u32x4 x[U];
    size_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t v = v0 + u * me.count;
      at[u] = v * 16 + 16 <= row_bytes ? v * 16 : row_bytes - 16;
      if (v < nvec) x[u] = load16(src + at[u]);
    }
    for (int j = 0; j < topk; ++j) {
      const uint32_t r = my_idx[j];
      if (r >= static_cast<uint32_t>(npairs)) continue;
      uint8_t *const dst = rows + r * row_bytes;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * me.count < nvec) store16<NT>(dst + at[u], x[u]);
    }
  }
  if (row_bytes >= 16) return;
  for (size_t b = me.lane; b < row_bytes; b += me.count) {
    const uint8_t x = src[b];
    for (int j = 0; j < topk; ++j) {
      const uint32_t r = my_idx[j];
      if (r < static_cast<uint32_t>(npairs)) rows[r * row_bytes + b] = x;
    }
  }
}

// J pairs at a time, J * U vectors requested before the first is added; a token with more takes several rounds.  The sum runs over j in
// ascending order, in fp32 with one multiply-add per term, and is rounded once.
template <Row T, int J, int U, bool SUB, bool NT>
__global__ __launch_bounds__(kThreads) void unpermute_kernel(const uint8_t *__restrict__ rows, const int32_t *__restrict__ idx, const void *__restrict__ weights,
                                                             Row weight_type, int ntokens, int topk, int n, int shift, uint8_t *__restrict__ out) {
  Lanes me = my_token<SUB>(blockIdx.x, shift);
  if (me.token >= ntokens) return;
  // Few tokens: several workgroups to each.
  me.lane += blockIdx.y * me.count;
  me.count *= gridDim.y;
  const uint32_t npairs = static_cast<uint32_t>(ntokens) * topk;
  const size_t row_bytes = static_cast<size_t>(n) * kElt<T>, pair0 = static_cast<size_t>(me.token) * topk;
  const int nvec = vectors_of(n, kVec<T>);
  uint8_t *const dst = out + static_cast<size_t>(me.token) * row_bytes;
  auto byte_of = [&](int v) { return static_cast<size_t>(vector_at(v, n, kVec<T>)) * kElt<T>; };
  for (int v0 = me.lane; v0 < nvec; v0 += U * me.count) {
    float acc[U][kVec<T>] = {};
    for (int j0 = 0; j0 < topk; j0 += J) {
      u32x4 x[U][J];
      float w[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t r = ~0u;
        if (j0 + j < topk) r = idx[pair0 + j0 + j];
        const bool live = r < npairs;
        w[j] = 0.f;
        if (live) w[j] = weights ? load_as(weights, weight_type, pair0 + j0 + j) : 1.f;
        const uint8_t *const src = rows + (live ? r : 0) * row_bytes;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u][j] = u32x4{0u, 0u, 0u, 0u};
          if (live && v0 + u * me.count < nvec) x[u][j] = load16<NT>(src + byte_of(v0 + u * me.count));
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[kVec<T>];
          unpack<T>(x[u][j], f);
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) acc[u][i] = fmaf(w[j], f[i], acc[u][i]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * me.count < nvec) store16(dst + byte_of(v0 + u * me.count), pack<T>(acc[u]));
  }
  if (nvec > 0) return;
  for (int e = me.lane; e < n; e += me.count) {
    float acc = 0.f;
    for (int j = 0; j < topk; ++j) {
      const uint32_t r = idx[pair0 + j];
      if (r >= npairs) continue;
      acc = fmaf(weights ? load_as(weights, weight_type, pair0 + j) : 1.f, load_as(rows + r * row_bytes, T, e), acc);
    }
    store_as(dst, T, e, acc);
  }
}

// grad_rows and grad_weights, either of them only if given.  The products of a pair are summed per lane, then over the lanes of the token in a
// fixed order.
template <Row T, int J, bool SUB, bool NT>
__global__ __launch_bounds__(kThreads) void unpermute_backward_kernel(const uint8_t *__restrict__ grad, const uint8_t *__restrict__ rows,
                                                                      const int32_t *__restrict__ idx, const void *__restrict__ weights, Row weight_type,
                                                                      int ntokens, int topk, int n, int shift, int clearers,
                                                                      uint8_t *__restrict__ grad_rows, void *__restrict__ grad_weights) {
  const size_t row_bytes = static_cast<size_t>(n) * kElt<T>;
  if (static_cast<int>(blockIdx.x) < clearers) {
    clear_unnamed(blockIdx.x, clearers, idx, ntokens * topk, row_bytes, grad_rows);
    return;
  }
  __shared__ float partial[kThreads / 64][J];
  Lanes me = my_token<SUB>(blockIdx.x - clearers, shift);
  // (Lanes past the last token stay for the barriers.)
  const uint32_t npairs = me.token < ntokens ? static_cast<uint32_t>(ntokens) * topk : 0;
  if (me.token >= ntokens) me.token = n = 0;
  const size_t pair0 = static_cast<size_t>(me.token) * topk;
  const int nvec = n / kVec<T>;
  const uint8_t *const src = grad + static_cast<size_t>(me.token) * row_bytes;
  for (int j0 = 0; j0 < topk; j0 += J) {
    size_t at[J];
    bool live[J];
    float w[J], dot[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      uint32_t r = ~0u;
      if (j0 + j < topk) r = idx[pair0 + j0 + j];
      live[j] = r < npairs;
      at[j] = (live[j] ? r : 0) * row_bytes;
      w[j] = live[j] ? load_as(weights, weight_type, pair0 + j0 + j) : 0.f;
      dot[j] = 0.f;
    }
    auto load = [&](int v, u32x4 &gv, u32x4 (&x)[J]) {
      gv = load16(src + static_cast<size_t>(v) * 16);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        x[j] = u32x4{0u, 0u, 0u, 0u};
        if (grad_weights && live[j]) x[j] = load16<NT>(rows + at[j] + static_cast<size_t>(v) * 16);
      }
    };
    auto use = [&](int v, const u32x4 &gv, const u32x4 (&x)[J]) {
      float g[kVec<T>];
      unpack<T>(gv, g);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (!live[j]) continue;
        if (grad_rows) {
          float o[kVec<T>];
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) o[i] = w[j] * g[i];
          store16<NT>(grad_rows + at[j] + static_cast<size_t>(v) * 16, pack<T>(o));
        }
        if (grad_weights) {
          float f[kVec<T>];
          unpack<T>(x[j], f);
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) dot[j] = fmaf(g[i], f[i], dot[j]);
        }
      }
    };
    // Two vectors at a time with a pair or two (8192 tokens top-2 4096 columns 62 -> 58 us), one with more (2000 top-8 1024 columns 18, two 22).
    int v = me.lane;
    if constexpr (J <= 2) {
      for (; v + me.count < nvec; v += 2 * me.count) {
        u32x4 gv[2], x[2][J];
        load(v, gv[0], x[0]);
        load(v + me.count, gv[1], x[1]);
        use(v, gv[0], x[0]);
        use(v + me.count, gv[1], x[1]);
      }
    }
    for (; v < nvec; v += me.count) {
      u32x4 gv, x[J];
      load(v, gv, x);
      use(v, gv, x);
    }
    for (int e = nvec * kVec<T> + me.lane; e < n; e += me.count) {
      const float g = load_as(src, T, e);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (!live[j]) continue;
        if (grad_rows) store_as(grad_rows + at[j], T, e, w[j] * g);
        if (grad_weights) dot[j] = fmaf(g, load_as(rows + at[j], T, e), dot[j]);
      }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (int j = 0; j < J; ++j)
      for (int off = (me.count < 64 ? me.count : 64) >> 1; off > 0; off >>= 1) dot[j] += __shfl_xor(dot[j], off, 64);
    if (!SUB && me.count > 64) {
      __syncthreads();  // the round before has read its sums
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int j = 0; j < J; ++j) partial[threadIdx.x >> 6][j] = dot[j];
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int wave0 = (threadIdx.x >> 6) & ~((me.count >> 6) - 1);
        dot[j] = partial[wave0][j];
        for (int k = 1; k < me.count >> 6; ++k) dot[j] += partial[wave0 + k][j];
      }
    }
    if (me.lane == 0 && npairs > 0) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (j0 + j < topk) store_as(grad_weights, weight_type, pair0 + j0 + j, dot[j]);
    }
  }
}

// Lanes of a token, as a power of two from 8 to 256: a vector each where tokens are few, `per_lane` vectors each where there are enough of them
// to fill the 256 compute units without.
int lanes_shift(int64_t nvec, int ntokens, int per_lane) {
  int shift = 3;
  while (shift < 8 && (int64_t{1} << shift) < nvec) ++shift;
  while (shift > 3 && (int64_t{ntokens} << shift) > int64_t{2048} * kThreads && (int64_t{per_lane} << (shift - 1)) >= nvec) --shift;
  return shift;
}

// Workgroups that clear: one for every 32 rows, as clearing is what a launch with few rows waits for (1000 tokens, top-4, 1536 fp32 columns, 10 %
// dropped: 31 us with one for 512 rows, 13 with one for 32), but no more than 128, or as many as read 8 MB of idx together, as each reads all of it.
int clearer_count(int npairs) {
  const int by_rows = (npairs + kRowsOfClearer - 32) / (kRowsOfClearer - 31);
  const int most = (1 << 21) / npairs > 128 ? (1 << 21) / npairs : 128, wide = (npairs + 31) / 32 < most ? (npairs + 31) / 32 : most;
  return by_rows > wide ? by_rows : wide;
}

// Very many very short rows: what the clearing workgroups read, four bytes a pair for every kRowsOfClearer rows, would be more than the rows themselves.  They are all cleared
// before the launch then.
bool clear_first(int npairs, int64_t row_bytes) { return int64_t{npairs} * 4 / kRowsOfClearer > row_bytes; }

__global__ __launch_bounds__(kThreads) void clear_kernel(uint8_t *__restrict__ rows, size_t bytes) {
  const size_t step = static_cast<size_t>(gridDim.x) * kThreads, at = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x;
  for (size_t v = at; v < bytes / 16; v += step) store16(rows + v * 16, u32x4{0u, 0u, 0u, 0u});
  if (at < bytes % 16) rows[bytes / 16 * 16 + at] = 0;
}

void clear_all(int npairs, int64_t row_bytes, void *rows, hipStream_t s) {
  hipLaunchKernelGGL(clear_kernel, dim3(2048), dim3(kThreads), 0, s, static_cast<uint8_t *>(rows), static_cast<size_t>(npairs) * row_bytes);
}

// Workgroups of a launch, 0: more threads than a launch has.
unsigned grid_of(int ntokens, int shift, int clearers) {
  const int64_t grid = clearers + (int64_t{ntokens} + (kThreads >> shift) - 1) / (kThreads >> shift);
  return grid * kThreads < (int64_t{1} << 32) ? static_cast<unsigned>(grid) : 0;
}

int check_pairs(const char *who, const int32_t *idx, int32_t ntokens, int32_t topk) {
  FLUXMI_REQUIRE(ntokens >= 0, FLUXMI_ERR_INVALID_ARG, "%s: negative ntokens=%d", who, ntokens);
  FLUXMI_REQUIRE(topk >= 1 && topk <= kMaxTopk, FLUXMI_ERR_UNSUPPORTED, "%s: topk=%d outside [1,%d]", who, topk, kMaxTopk);
  FLUXMI_REQUIRE(static_cast<int64_t>(ntokens) * topk <= (int64_t{1} << 30), FLUXMI_ERR_UNSUPPORTED, "%s: ntokens*topk=%lld exceeds 2^30", who,
                 static_cast<long long>(ntokens) * topk);
  FLUXMI_REQUIRE(idx != nullptr || ntokens == 0, FLUXMI_ERR_INVALID_ARG, "%s: null scatter_index", who);
  FLUXMI_REQUIRE((reinterpret_cast<uintptr_t>(idx) & 3) == 0, FLUXMI_ERR_INVALID_ARG, "%s: scatter_index is not 4-byte aligned", who);
  return FLUXMI_OK;
}

// Pairs of a token that are requested together; top-k beyond 8 takes rounds of 8.
template <class F>
void by_topk(int topk, F &&f) {
  if (topk == 1) f(std::integral_constant<int, 1>{});
  else if (topk == 2) f(std::integral_constant<int, 2>{});
  else if (topk <= 4) f(std::integral_constant<int, 4>{});
  else if (topk <= 6) f(std::integral_constant<int, 6>{});
  else f(std::integral_constant<int, 8>{});
}

// f(several tokens to a wave, non-temporal)
template <class F>
void by_lanes(int shift, size_t row_bytes, F &&f) {
  const bool nt = row_bytes >= kStreamBytes;
  if (shift < 6) nt ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
  else nt ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}

}  // namespace
}  // namespace fluxmi

extern "C" int fluxmi_moe_permute(const void *in, const int32_t *scatter_index, int32_t ntokens, int32_t topk, int64_t row_bytes, void *rows, void *stream) {
  using namespace fluxmi;
  const int rc = check_pairs("moe_permute", scatter_index, ntokens, topk);
  if (rc != FLUXMI_OK) return rc;
  FLUXMI_REQUIRE(row_bytes >= 0 && row_bytes <= (int64_t{1} << 31), FLUXMI_ERR_INVALID_ARG, "moe_permute: row_bytes=%lld outside [0,2^31]",
                 static_cast<long long>(row_bytes));
  if (ntokens == 0 || row_bytes == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(in != nullptr && rows != nullptr, FLUXMI_ERR_INVALID_ARG, "moe_permute: null pointer argument");
  const int shift = lanes_shift((row_bytes + 15) / 16, ntokens, 4), clearers = clear_first(ntokens * topk, row_bytes) ? 0 : clearer_count(ntokens * topk);
  const unsigned grid = grid_of(ntokens, shift, clearers);
  FLUXMI_REQUIRE(grid > 0, FLUXMI_ERR_UNSUPPORTED, "moe_permute: ntokens=%d is too many for rows of %lld bytes", ntokens, static_cast<long long>(row_bytes));
  if (clearers == 0) clear_all(ntokens * topk, row_bytes, rows, static_cast<hipStream_t>(stream));
  by_lanes(shift, static_cast<size_t>(row_bytes) * ntokens * topk, [&](auto sub, auto nt) {
    hipLaunchKernelGGL((permute_kernel<decltype(sub)::value, decltype(nt)::value>), dim3(grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<const uint8_t *>(in), scatter_index, ntokens, topk, static_cast<size_t>(row_bytes), shift, clearers,
                       static_cast<uint8_t *>(rows));
  });
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}

extern "C" int fluxmi_moe_unpermute(const void *rows, int32_t row_type, const int32_t *scatter_index, const void *weights, int32_t weight_type,
                                    int32_t ntokens, int32_t topk, int32_t n, void *out, void *stream) {
  using namespace fluxmi;
  Row type, wtype;
  int rc = check_type("moe_unpermute", row_type, &type);
  if (rc == FLUXMI_OK) rc = check_type("moe_unpermute", weight_type, &wtype);
  if (rc == FLUXMI_OK) rc = check_pairs("moe_unpermute", scatter_index, ntokens, topk);
  if (rc != FLUXMI_OK) return rc;
  FLUXMI_REQUIRE(n >= 0, FLUXMI_ERR_INVALID_ARG, "moe_unpermute: negative n=%d", n);
  if (ntokens == 0 || n == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(rows != nullptr && out != nullptr, FLUXMI_ERR_INVALID_ARG, "moe_unpermute: null pointer argument");
  FLUXMI_REQUIRE(aligned_to(rows, type) && aligned_to(out, type) && aligned_to(weights, wtype), FLUXMI_ERR_INVALID_ARG,
                 "moe_unpermute: a pointer is not aligned to its elements");
  const int nvec = (static_cast<int64_t>(n) * (type == Row::F32 ? 4 : 2) + 15) / 16, shift = lanes_shift(nvec, ntokens, topk <= 2 ? 4 : 2);
  // us with one and with several workgroups to a token: 10 tokens top-8 7168 columns bf16 9.0 / 3.5, 100 tokens 12.9 / 5.2, 1000 tokens 30 / 25; 300 tokens top-4 4096 columns
  // 5.2 / 3.8, 1024 tokens 8.2 / 8.4.
  const unsigned parts = ntokens > 1024 || nvec <= kThreads ? 1 : nvec > 7 * kThreads ? 8 : (nvec + kThreads - 1) / kThreads;
  const unsigned grid = grid_of(ntokens, shift, 0);
  FLUXMI_REQUIRE(grid > 0, FLUXMI_ERR_UNSUPPORTED, "moe_unpermute: ntokens=%d is too many for n=%d", ntokens, n);
  by_type(type, [&](auto t) {
    by_topk(topk, [&](auto j) {
      by_lanes(shift, static_cast<size_t>(n) * kElt<decltype(t)::value> * ntokens * topk, [&](auto sub, auto nt) {
        constexpr int J = decltype(j)::value, U = J == 1 ? 4 : J == 2 ? 2 : 1;
        hipLaunchKernelGGL((unpermute_kernel<decltype(t)::value, J, U, decltype(sub)::value, decltype(nt)::value>), dim3(grid, parts), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), static_cast<const uint8_t *>(rows), scatter_index, weights, wtype, ntokens, topk, n, shift,
                           static_cast<uint8_t *>(out));
      });
    });
  });
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}

extern "C" int fluxmi_moe_unpermute_backward(const void *grad_out, const void *rows, int32_t row_type, const int32_t *scatter_index, const void *weights,
                                             int32_t weight_type, int32_t ntokens, int32_t topk, int32_t n, void *grad_rows, void *grad_weights,
                                             void *stream) {
  using namespace fluxmi;
  Row type, wtype;
  int rc = check_type("moe_unpermute_backward", row_type, &type);
  if (rc == FLUXMI_OK) rc = check_type("moe_unpermute_backward", weight_type, &wtype);
  if (rc == FLUXMI_OK) rc = check_pairs("moe_unpermute_backward", scatter_index, ntokens, topk);
  if (rc != FLUXMI_OK) return rc;
  FLUXMI_REQUIRE(n >= 0, FLUXMI_ERR_INVALID_ARG, "moe_unpermute_backward: negative n=%d", n);
  if (ntokens == 0 || (n == 0 && grad_weights == nullptr)) return FLUXMI_OK;
  FLUXMI_REQUIRE(weights != nullptr && (n == 0 || (grad_out != nullptr && (rows != nullptr || grad_weights == nullptr))) &&
                     (grad_rows != nullptr || grad_weights != nullptr || n == 0),
                 FLUXMI_ERR_INVALID_ARG, "moe_unpermute_backward: null pointer argument");
  FLUXMI_REQUIRE(aligned_to(rows, type) && aligned_to(grad_out, type) && aligned_to(grad_rows, type) && aligned_to(weights, wtype) &&
                     aligned_to(grad_weights, wtype),
                 FLUXMI_ERR_INVALID_ARG, "moe_unpermute_backward: a pointer is not aligned to its elements");
  const int64_t row_bytes = int64_t{n} * (type == Row::F32 ? 4 : 2);
  const bool clears = grad_rows != nullptr && n > 0;
  const int shift = lanes_shift(n / (type == Row::F32 ? 4 : 8), ntokens, 4), clearers = clears && !clear_first(ntokens * topk, row_bytes) ? clearer_count(ntokens * topk) : 0;
  const unsigned grid = grid_of(ntokens, shift, clearers);
  FLUXMI_REQUIRE(grid > 0, FLUXMI_ERR_UNSUPPORTED, "moe_unpermute_backward: ntokens=%d is too many for n=%d", ntokens, n);
  if (clears && clearers == 0) clear_all(ntokens * topk, row_bytes, grad_rows, static_cast<hipStream_t>(stream));
  by_type(type, [&](auto t) {
    by_topk(topk, [&](auto j) {
      by_lanes(shift, static_cast<size_t>(n) * kElt<decltype(t)::value> * ntokens * topk, [&](auto sub, auto nt) {
        hipLaunchKernelGGL((unpermute_backward_kernel<decltype(t)::value, decltype(j)::value, decltype(sub)::value, decltype(nt)::value>),
                           dim3(grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                           static_cast<const uint8_t *>(grad_out), static_cast<const uint8_t *>(rows), scatter_index, weights, wtype, ntokens, topk, n, shift,
                           clearers, static_cast<uint8_t *>(grad_rows), grad_weights);
      });
    });
  });
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}
