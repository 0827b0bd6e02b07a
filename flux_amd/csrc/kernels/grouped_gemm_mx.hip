// Grouped product of MXFP4 operands: D[r, n] = row_scale[r] * sum_k A[row(r), k] * B[e(r), n, k].
//
// The MFMA takes the packed codes and the scale bytes as they lie in memory: of 16 x 16 x 128 a lane holds 16 bytes of codes, one block of 32
// values (lane l: row l & 15, block l >> 4), and the block's scale byte in a register of its own.  B's rows are the MFMA's rows, so that a lane's
// four sums are neighbouring columns of one row of D.
//
// Few rows per expert: the weights are read once and everything else is small.  A workgroup has 64 columns of an expert and up to 64 of its
// rows; its four waves split K in turns of 512 values and add their sums through LDS in a fixed order.
#include "rows.hpp"

namespace fluxmi {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kCols = 64;    // columns of a workgroup
constexpr int kTurn = 512;   // values of K a wave takes at a time: 256 bytes of codes, 16 of scales of each row
constexpr int kMaxExperts = 1024;

struct MxParams {
  const uint8_t *a, *a_scale, *b, *b_scale;
  uint8_t *d;
  const int32_t *splits, *gather_a;
  const float *row_scale;
  int32_t nexperts, max_rows, n, kb, a_rows;  // kb: blocks of a row
  Row d_type;
};

#if defined(__HIP_DEVICE_COMPILE__)

// Rows row0 .. row0 + rows of the sorted rows, all of expert e; rows == 0: there is no such item.
struct Item {
  int e, row0, rows;
};

// The item-th piece of at most `most` rows, experts in order.  Negative counts are 0, rows past max_rows do not exist.
__device__ __forceinline__ Item locate(const MxParams &p, int item, int most) {
  if (p.splits == nullptr) {
    const int row0 = item * most, rest = p.max_rows - row0;
    return {0, row0, rest < 0 ? 0 : (rest < most ? rest : most)};
  }
  const int lane = threadIdx.x & 63;
  int row_carry = 0, item_carry = 0;
  for (int e0 = 0; e0 < p.nexperts; e0 += 64) {
    int r = e0 + lane < p.nexperts ? p.splits[e0 + lane] : 0;
    r = r < 0 ? 0 : (r > p.max_rows ? p.max_rows : r);
    const int incl = wave_inclusive_scan(r);  // (at most 64 * 2^24 more than the carry, see the host's check)
    int begin = row_carry + incl - r, end = row_carry + incl;
    begin = begin > p.max_rows ? p.max_rows : begin;
    end = end > p.max_rows ? p.max_rows : end;
    row_carry = __builtin_amdgcn_readlane(end, 63);
    const int items = (end - begin + most - 1) / most, items_end = item_carry + wave_inclusive_scan(items);
    item_carry = __builtin_amdgcn_readlane(items_end, 63);
    const uint64_t hit = __ballot(item < items_end);
    if (hit != 0) {
      const int src = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      const int first = __builtin_amdgcn_readlane(items_end - items, src), end_row = __builtin_amdgcn_readlane(end, src);
      const int row0 = __builtin_amdgcn_readlane(begin, src) + (item - first) * most, rest = end_row - row0;
      return {e0 + src, row0, rest < most ? rest : most};
    }
  }
  return {0, 0, 0};
}

// The row of A that sorted row r reads.
__device__ __forceinline__ int a_row(const MxParams &p, int r) {
  if (p.gather_a == nullptr) return r;
  const int x = p.gather_a[r];
  return x < 0 ? 0 : (x >= p.a_rows ? p.a_rows - 1 : x);
}

__device__ __forceinline__ f32x4 mfma(const u32x4 w, const u32x4 x, uint32_t w_scale, uint32_t x_scale, f32x4 c) {
  const i32x8 wa = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3]), 0, 0, 0, 0};
  const i32x8 xa = {static_cast<int>(x[0]), static_cast<int>(x[1]), static_cast<int>(x[2]), static_cast<int>(x[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xa, c, 4, 4, 0, w_scale, 0, x_scale);
}

__device__ __forceinline__ void store_one(uint8_t *d, Row type, size_t i, float v) {
  if (type == Row::F32) reinterpret_cast<float *>(d)[i] = v;
  else reinterpret_cast<uint16_t *>(d)[i] = type == Row::BF16 ? float_to_bf16_bits(v) : float_to_f16_bits(v);
}

// Codes and scales of a lane's blocks of one turn: block 4 s + g of the turn, s = 0 .. 3, with g = lane >> 4.  What lies past the end of the row is zero codes
// with scale byte 0 in both operands.
struct Turn {
  u32x4 code[4];
  uint32_t scale[4];
};

__device__ __forceinline__ void load_turn(Turn &t, const uint8_t *codes, const uint8_t *scales, int turn, int kb) {
  const int g = (threadIdx.x & 63) >> 4, first = turn * 16;
  if (first + 16 <= kb) {
#pragma unroll
    for (int s = 0; s < 4; ++s) t.code[s] = load16(codes + (first + 4 * s + g) * 16);
    const u32x4 sc = load16(scales + first);
#pragma unroll
    for (int s = 0; s < 4; ++s) t.scale[s] = sc[s] >> (8 * g);  // the MFMA takes the lowest byte
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      t.code[s] = u32x4{0u, 0u, 0u, 0u};
      t.scale[s] = 0;
      if (first + 4 * s + g < kb) {
        t.code[s] = load16(codes + (first + 4 * s + g) * 16);
        t.scale[s] = scales[first + 4 * s + g];
      }
    }
  }
}

#endif  // __HIP_DEVICE_COMPILE__

template <int MT>
__global__ __launch_bounds__(kThreads) void mx_few_rows_kernel(const MxParams p, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ f32x4 sums[3][MT * 4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x / tiles_n, n0 = (blockIdx.x - item * tiles_n) * kCols;
  const Item it = locate(p, item, MT * 16);
  if (it.rows <= 0) return;
  const size_t row_bytes = static_cast<size_t>(p.kb) * 16;
  const uint8_t *w[4], *ws[4], *x[MT], *xs[MT];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + j * 16 + (lane & 15);
    const size_t row = static_cast<size_t>(it.e) * p.n + (n < p.n ? n : p.n - 1);  // (columns past the end are not stored)
    w[j] = p.b + row * row_bytes;
    ws[j] = p.b_scale + row * p.kb;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = i * 16 + (lane & 15);
    const size_t row = a_row(p, it.row0 + (m < it.rows ? m : it.rows - 1));
    x[i] = p.a + row * row_bytes;
    xs[i] = p.a_scale + row * p.kb;
  }
  f32x4 acc[MT][4] = {};
  const int turns = (p.kb + 15) / 16;
  for (int t = wave; t < turns; t += 4) {
    Turn wt[4], xt[MT];
#pragma unroll
    for (int j = 0; j < 4; ++j) load_turn(wt[j], w[j], ws[j], t, p.kb);
#pragma unroll
    for (int i = 0; i < MT; ++i) load_turn(xt[i], x[i], xs[i], t, p.kb);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma(wt[j].code[s], xt[i].code[s], wt[j].scale[s], xt[i].scale[s], acc[i][j]);
  }
  // Wave w finishes the blocks of column group w.
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j != wave) sums[wave < j ? wave : wave - 1][i * 4 + j][lane] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = i * 16 + (lane & 15);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 4; ++v) {  // the waves' sums in order
      f32x4 own = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j == wave) own = acc[i][j];
      sum += v == wave ? own : sums[v < wave ? v : v - 1][i * 4 + wave][lane];
    }
    if (m >= it.rows) continue;
    const int r = it.row0 + m;
    const float scale = p.row_scale ? p.row_scale[r] : 1.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int n = n0 + wave * 16 + (lane >> 4) * 4 + v;
      if (n < p.n) store_one(p.d, p.d_type, static_cast<size_t>(r) * p.n + n, sum[v] * scale);
    }
  }
#endif  // __HIP_DEVICE_COMPILE__
}

int check_args(const fluxmi_mx_gemm_args *args) {
  FLUXMI_REQUIRE(args != nullptr, FLUXMI_ERR_INVALID_ARG, "grouped_gemm_mx: null args");
  const fluxmi_mx_gemm_args &a = *args;
  FLUXMI_REQUIRE(a.nexperts >= 1 && a.nexperts <= kMaxExperts, FLUXMI_ERR_UNSUPPORTED, "grouped_gemm_mx: nexperts=%d outside [1,%d]", a.nexperts, kMaxExperts);
  FLUXMI_REQUIRE(a.max_rows >= 0 && a.n >= 0 && a.k >= 1 && a.a_rows >= 0, FLUXMI_ERR_INVALID_ARG,
                 "grouped_gemm_mx: bad sizes (max_rows=%d, n=%d, k=%d, a_rows=%d)", a.max_rows, a.n, a.k, a.a_rows);
  FLUXMI_REQUIRE(a.max_rows <= (1 << 24), FLUXMI_ERR_UNSUPPORTED, "grouped_gemm_mx: max_rows=%d exceeds 2^24", a.max_rows);
  FLUXMI_REQUIRE(a.splits != nullptr || a.nexperts == 1, FLUXMI_ERR_INVALID_ARG, "grouped_gemm_mx: null splits with nexperts=%d", a.nexperts);
  FLUXMI_REQUIRE(a.d_type >= 0 && a.d_type <= 2, FLUXMI_ERR_INVALID_ARG, "grouped_gemm_mx: unknown type %d of d", a.d_type);
  const int64_t row_bytes = (int64_t{a.k} + 31) / 32 * 16, limit = int64_t{1} << 31;
  FLUXMI_REQUIRE(a.n * row_bytes < limit && a.a_rows * row_bytes < limit, FLUXMI_ERR_UNSUPPORTED,
                 "grouped_gemm_mx: codes of one expert or of A reach 2 GiB (n=%d, a_rows=%d, k=%d)", a.n, a.a_rows, a.k);
  if (a.max_rows == 0 || a.n == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(a.a != nullptr && a.a_scale != nullptr && a.b != nullptr && a.b_scale != nullptr && a.d != nullptr, FLUXMI_ERR_INVALID_ARG,
                 "grouped_gemm_mx: null a / a_scale / b / b_scale / d");
  FLUXMI_REQUIRE(a.a_rows >= (a.gather_a != nullptr ? 1 : a.max_rows), FLUXMI_ERR_INVALID_ARG, "grouped_gemm_mx: a_rows=%d is too few for max_rows=%d", a.a_rows,
                 a.max_rows);
  const uintptr_t d = reinterpret_cast<uintptr_t>(a.d);
  FLUXMI_REQUIRE(aligned16(a.a) && aligned16(a.b) && (d & (a.d_type == FLUXMI_ROWS_FP32 ? 3u : 1u)) == 0, FLUXMI_ERR_INVALID_ARG,
                 "grouped_gemm_mx: a or b is not 16-byte aligned, or d not to its elements");
  return FLUXMI_OK;
}

template <int MT>
int launch_few_rows(const MxParams &p, hipStream_t s) {
  const int tiles_n = (p.n + kCols - 1) / kCols;
  // Pieces of rows: at most one that is not full for each expert with rows.
  const int64_t items = p.max_rows / (MT * 16) + (p.nexperts < p.max_rows ? p.nexperts : p.max_rows), grid = items * tiles_n;
  FLUXMI_REQUIRE(grid * kThreads < (int64_t{1} << 32), FLUXMI_ERR_UNSUPPORTED, "grouped_gemm_mx: max_rows=%d and n=%d are more than a launch covers", p.max_rows, p.n);
  hipLaunchKernelGGL(mx_few_rows_kernel<MT>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s, p, tiles_n);
  return FLUXMI_OK;
}

}  // namespace
}  // namespace fluxmi

extern "C" size_t fluxmi_grouped_gemm_mx_workspace_bytes(const fluxmi_mx_gemm_args *) { return 0; }

extern "C" int fluxmi_grouped_gemm_mx(const fluxmi_mx_gemm_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace fluxmi;
  int rc = check_args(args);
  if (rc != FLUXMI_OK || args->max_rows == 0 || args->n == 0) return rc;
  const size_t need = fluxmi_grouped_gemm_mx_workspace_bytes(args);
  FLUXMI_REQUIRE(need == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= need), FLUXMI_ERR_WORKSPACE,
                 "grouped_gemm_mx: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  MxParams p;
  p.a = static_cast<const uint8_t *>(args->a);
  p.a_scale = static_cast<const uint8_t *>(args->a_scale);
  p.b = static_cast<const uint8_t *>(args->b);
  p.b_scale = static_cast<const uint8_t *>(args->b_scale);
  p.d = static_cast<uint8_t *>(args->d);
  p.splits = args->splits;
  p.gather_a = args->gather_a;
  p.row_scale = args->row_scale;
  p.nexperts = args->nexperts;
  p.max_rows = args->max_rows;
  p.n = args->n;
  p.kb = (args->k + 31) / 32;
  p.a_rows = args->a_rows;
  p.d_type = args->d_type == FLUXMI_ROWS_BF16 ? Row::BF16 : args->d_type == FLUXMI_ROWS_FP32 ? Row::F32 : Row::F16;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int average = p.max_rows / p.nexperts;
  rc = average <= 16 ? launch_few_rows<1>(p, s) : average <= 32 ? launch_few_rows<2>(p, s) : launch_few_rows<4>(p, s);
  if (rc != FLUXMI_OK) return rc;
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}
