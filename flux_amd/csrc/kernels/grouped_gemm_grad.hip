// Gradients of the grouped product D[r, :] = X[r, :] W[e(r)]^T (W[e] is [n, k]):
//
//   of its input    dX[r, k] = sum_n G[r, n] W[e(r)][n, k]              rows that belong to no expert are 0
//   of its weights  dW[e][n, k] = sum_{r in e} G[r, n] X[r, k]          0 for an expert without rows
//
// Sums are fp32 in MFMAs of 16 x 16 x 32, with one rounding at the end (to 16 bits; none to fp32); with `accumulate` the old value is added before it.
//
// What is summed over lies across the rows of W, X and, for the weights, G: a lane of the MFMA needs eight values of one column, from eight rows.  The
// rows go to LDS as they lie in memory and come back through the transposing LDS read: 16 lanes together read four rows of 16 columns, and each of
// them gets the four values of one column.
//
// Here: pieces of 128 x 128 on four waves, one step in LDS and the next in registers, for operands of any width and start and for small products; the weights' sums are cut into parts
// of 256 rows or more where pieces are few, so that the card is full.  Latency and barriers bound them: 8 experts 1024 x 1024, 2048 rows 15 us (weights), 26 (input); at the large
// sizes of grouped_gemm_grad_tiles.hip, which computes what is larger, they take 2360 and 2460 where its tiles take 1435 and 1470.  Operands that tiles refuse cost more: 8 experts
// 14336 x 4092, 16384 rows 5130 (weights), 6130 (from 8 bits) and 6510 (input), most of it loads element by element; 14336 x 4096 with an input off 16 bytes 2820 (weights).
#include "grouped_gemm_grad_tiles.hpp"

namespace fluxmi {
namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 128;     // rows and columns of a piece of the result
constexpr int kStep = 32;       // what a step sums over
constexpr int kAcross = 272;    // bytes from one row of LDS to the next: 128 columns, and 16 bytes off the banks of the row before
constexpr int kAlong = 80;      // 32 columns, and 16 bytes

#if defined(__HIP_DEVICE_COMPILE__)

typedef u32x4 u32x4_any __attribute__((aligned(1)));  // at any address: one instruction on this hardware
typedef u32x2 u32x2_any __attribute__((aligned(1)));

// `count` of eight elements of 16 bits, zeros behind them.  VEC: all eight or none, on 16 bytes.
template <bool VEC>
__device__ __forceinline__ u32x4 load8(const uint8_t *p, int count) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if constexpr (VEC) {
    if (count > 0) v = *reinterpret_cast<const u32x4 *>(p);
  } else {
    if (count >= 8) return *reinterpret_cast<const u32x4_any *>(p);
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < count) v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[i]) << (16 * (i & 1));
  }
  return v;
}
// The same of eight codes, as values of 16 bits.
template <bool VEC, bool F16>
__device__ __forceinline__ u32x4 load8_codes(const uint8_t *p, int count, const uint8_t *scale) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (count <= 0) return v;
  u32x2 c = {0u, 0u};
  if constexpr (VEC) {
    c = *reinterpret_cast<const u32x2 *>(p);
  } else if (count >= 8) {
    c = *reinterpret_cast<const u32x2_any *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < count) c[i / 4] |= static_cast<uint32_t>(p[i]) << (8 * (i & 3));
  }
  const uint32_t byte = *scale;
  const float s = __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7fc00000u : byte << 23));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto x = i & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8(c[i / 2], true) : __builtin_amdgcn_cvt_pk_f32_fp8(c[i / 2], false);
    v[i] = pack2<F16>(x[0] * s, x[1] * s);
  }
  return v;
}

// The fragment of 16 columns (from byte `col` of a row on) over the 32 rows of a step: lane l has column l % 16 of rows 8 (l / 16) .. + 7.
__device__ __forceinline__ u32x4 read_across(uint32_t lds, int col) {
  const int l = lane_id(), g = l >> 4, i = l & 15;
  const uint32_t at = lds + (8 * g + (i >> 2)) * kAcross + col * 2 + (i & 3) * 8;
  const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(uintptr_t)at));
  const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(uintptr_t)(at + 4 * kAcross)));
  return {lo[0], lo[1], hi[0], hi[1]};
}

template <bool F16>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

#endif  // __HIP_DEVICE_COMPILE__

// A piece of 128 x 128 of the result on four waves, 64 x 64 to each.  VEC: n and k are multiples of 8 and the operands start on 16 bytes (codes: 8).
template <bool F16, Grad G, bool VEC>
__global__ __launch_bounds__(kThreads) void grad_piece_kernel(const GradArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool INPUT = G == Grad::INPUT;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kStep * kAcross + (INPUT ? kPiece * kAlong : kStep * kAcross)];
  const uint32_t cols_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)smem));
  const uint32_t rows_lds = cols_lds + kStep * kAcross;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 1, wc = wave & 1;  // 64 rows and columns of the piece

  // ---- which piece: rows out_row0 .. + out_rows of the result, columns col0 .., and what it sums over ------------
  const int tiles_k = (a.k + kPiece - 1) / kPiece;
  const int item = blockIdx.x;
  const int kt = item % tiles_k, rest = item / tiles_k, col0 = kt * kPiece;
  int e, out_rows, steps;
  int64_t out_row0;
  const uint8_t *grad0, *other0, *scale0 = nullptr;  // first row (INPUT: of grad; otherwise of both) that the piece reads
  int sum_over;                                    // rows, INPUT: columns of grad
  int grad_col0 = 0;
  if constexpr (INPUT) {
    const RowTile t = row_tile<kPiece>(a, rest);
    if (t.rows <= 0) return;
    e = t.e;
    out_rows = t.rows;
    out_row0 = t.row0;
    sum_over = e < a.nexperts ? a.n : 0;
    grad0 = a.grad + static_cast<int64_t>(t.row0) * a.n * 2;
    other0 = a.other + static_cast<int64_t>(e < a.nexperts ? e : 0) * a.n * a.k * 2;
  } else {
    const int tiles_n = (a.n + kPiece - 1) / kPiece;
    const int part = rest % a.parts, nt = rest / a.parts % tiles_n;
    e = rest / a.parts / tiles_n;
    grad_col0 = nt * kPiece;
    out_rows = a.n - grad_col0 < kPiece ? a.n - grad_col0 : kPiece;
    out_row0 = static_cast<int64_t>(e) * a.n + grad_col0;
    const ExpertRows x = rows_of_expert(a, e);
    const int all = (x.end - x.begin + kStep - 1) / kStep, first = static_cast<int>(static_cast<int64_t>(all) * part / a.parts) * kStep;
    int last = static_cast<int>(static_cast<int64_t>(all) * (part + 1) / a.parts) * kStep;
    if (last > x.end - x.begin) last = x.end - x.begin;
    sum_over = last - first;
    const int64_t row0 = x.begin + first;
    grad0 = a.grad + row0 * a.n * 2;
    other0 = a.other + row0 * a.k * (G == Grad::WEIGHT_8BIT ? 1 : 2);
    if constexpr (G == Grad::WEIGHT_8BIT) scale0 = a.scale + row0 * ((a.k + 31) / 32);
  }
  steps = (sum_over + kStep - 1) / kStep;

  // ---- fills: two vectors of either operand to a thread, through registers ----------------------------------------
  u32x4 fc[2], fr[2];
  auto load = [&](int s) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = (tid >> 4) + q * 16, c = (tid & 15) * 8, row = s * kStep + r;  // 16 vectors to a row
      const int count = row < sum_over ? a.k - col0 - c : 0;
      if constexpr (G == Grad::WEIGHT_8BIT)
        fc[q] = load8_codes<VEC, F16>(other0 + static_cast<int64_t>(row) * a.k + col0 + c, count,
                                      scale0 + static_cast<int64_t>(row) * ((a.k + 31) / 32) + (col0 + c) / 32);
      else fc[q] = load8<VEC>(other0 + (static_cast<int64_t>(row) * a.k + col0 + c) * 2, count);
      if constexpr (INPUT) {
        const int m = (tid >> 2) + q * 64, n = s * kStep + (tid & 3) * 8;  // four vectors to a row
        fr[q] = load8<VEC>(grad0 + (static_cast<int64_t>(m) * a.n + n) * 2, m < out_rows ? a.n - n : 0);
      } else {
        fr[q] = load8<VEC>(grad0 + (static_cast<int64_t>(row) * a.n + grad_col0 + c) * 2, row < sum_over ? a.n - grad_col0 - c : 0);
      }
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = (tid >> 4) + q * 16, c = (tid & 15) * 8;
      *reinterpret_cast<u32x4 *>(smem + r * kAcross + c * 2) = fc[q];
      if constexpr (INPUT) *reinterpret_cast<u32x4 *>(smem + kStep * kAcross + ((tid >> 2) + q * 64) * kAlong + (tid & 3) * 16) = fr[q];
      else *reinterpret_cast<u32x4 *>(smem + kStep * kAcross + r * kAcross + c * 2) = fr[q];
    }
  };

  f32x4 acc[4][4];  // [row block][column block]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (steps > 0) load(0);
  for (int s = 0; s < steps; ++s) {
    __syncthreads();
    store();
    __syncthreads();
    if (s + 1 < steps) load(s + 1);
    u32x4 rf[4], cf[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cf[i] = read_across(cols_lds, wc * 64 + i * 16);
      if constexpr (INPUT) rf[i] = *reinterpret_cast<const u32x4 *>(smem + kStep * kAcross + (wr * 64 + i * 16 + (lane & 15)) * kAlong + (lane >> 4) * 16);
      else rf[i] = read_across(rows_lds, wr * 64 + i * 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma<F16>(cf[j], rf[i], acc[i][j]);
  }

  // ---- lane l has columns 4 (l / 16) .. + 3 of row l % 16 of a block ----------------------------------------------
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = wr * 64 + i * 16 + (lane & 15), c = wc * 64 + j * 16 + (lane >> 4) * 4;
      if (!INPUT && a.parts > 1) {
        *reinterpret_cast<f32x4 *>(a.partial + ((static_cast<int64_t>(item) * kPiece + r) * kPiece + c)) = acc[i][j];
      } else if (r < out_rows) {
        store4<F16>(a, (out_row0 + r) * a.k + col0 + c, acc[i][j], a.k - col0 - c, (a.k & 3) == 0);
      }
    }
#endif
}

// The parts of a piece's sums, added in their order.
template <bool F16>
__global__ __launch_bounds__(kThreads) void grad_join_kernel(const GradArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int tiles_k = (a.k + kPiece - 1) / kPiece, tiles_n = (a.n + kPiece - 1) / kPiece;
  const int piece = blockIdx.x >> 4, r = (blockIdx.x & 15) * 8 + (threadIdx.x >> 5), c = (threadIdx.x & 31) * 4;
  const int kt = piece % tiles_k, nt = piece / tiles_k % tiles_n, e = piece / tiles_k / tiles_n;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < a.parts; ++part) {
    const int64_t item = ((static_cast<int64_t>(e) * tiles_n + nt) * a.parts + part) * tiles_k + kt;
    v += *reinterpret_cast<const f32x4 *>(a.partial + (item * kPiece + r) * kPiece + c);
  }
  const int n = nt * kPiece + r, k = kt * kPiece + c;
  if (n < a.n) store4<F16>(a, (static_cast<int64_t>(e) * a.n + n) * a.k + k, v, a.k - k, (a.k & 3) == 0);
#endif
}

constexpr int kClearBlocks = 256;

// Rows past the sum of the splits to 0: an even share of their bytes to each workgroup, whole 16 bytes but at the ends.
__global__ __launch_bounds__(kThreads) void clear_rest_kernel(const GradArgs a, int64_t row_bytes) {
#if defined(__HIP_DEVICE_COMPILE__)
  int carry = 0;
  for (int e0 = 0; e0 < a.nexperts; e0 += 64) rows_of_lane(a, e0, carry);
  uint8_t *const first = a.out + carry * row_bytes, *const last = a.out + a.rows * row_bytes;
  uint8_t *head = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(first) + 15) & ~uintptr_t{15});
  if (head > last) head = last;
  const int64_t vectors = (last - head) / 16;
  if (blockIdx.x == 0) {
    for (uint8_t *p = first + threadIdx.x; p < head; p += kThreads) *p = 0;
    for (uint8_t *p = head + vectors * 16 + threadIdx.x; p < last; p += kThreads) *p = 0;
  }
  for (int64_t v = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; v < vectors; v += kClearBlocks * kThreads)
    *reinterpret_cast<u32x4 *>(head + v * 16) = u32x4{0u, 0u, 0u, 0u};
#endif
}

// ---- host ----------------------------------------------------------------------------------------------------
int check_product(const char *who, int32_t type, int32_t nexperts, int64_t rows, int64_t n, int64_t k) {
  FLUXMI_REQUIRE(type == FLUXMI_ROWS_BF16 || type == FLUXMI_ROWS_FP16, FLUXMI_ERR_INVALID_ARG, "%s: type %d (bf16 and fp16 are built)", who, type);
  FLUXMI_REQUIRE(nexperts >= 0 && rows >= 0 && n >= 0 && k >= 0, FLUXMI_ERR_INVALID_ARG, "%s: a negative size", who);
  FLUXMI_REQUIRE(nexperts <= 1024, FLUXMI_ERR_UNSUPPORTED, "%s: nexperts=%d (at most 1024)", who, nexperts);
  FLUXMI_REQUIRE(rows <= kGradMaxRows, FLUXMI_ERR_UNSUPPORTED, "%s: %lld rows (at most 2^24)", who, static_cast<long long>(rows));
  FLUXMI_REQUIRE(n <= (1 << 24) && k <= (1 << 24), FLUXMI_ERR_UNSUPPORTED, "%s: n or k is over 2^24", who);
  return FLUXMI_OK;
}

// Pieces are dealt to workgroups of 256 threads, of which a launch has at most 2^24 - 1.
constexpr int64_t kMostItems = (int64_t{1} << 24) - 1;

int64_t tiles_of(int64_t v) { return (v + kPiece - 1) / kPiece; }

// Parts of an expert's rows: as many as fill the card with pieces twice over, of 256 rows at least on average.
int parts_of(int32_t nexperts, int64_t rows, int64_t n, int64_t k) {
  const int64_t pieces = nexperts * tiles_of(n) * tiles_of(k);
  if (pieces == 0 || pieces >= 512) return 1;
  int64_t parts = (512 + pieces - 1) / pieces;
  const int64_t most = rows / nexperts / 256;
  if (parts > most) parts = most;
  return parts < 1 ? 1 : static_cast<int>(parts);
}

bool on(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <Grad G>
void launch_pieces(const GradArgs &a, bool f16, bool vec, uint32_t grid, hipStream_t stream) {
  if (f16) {
    if (vec) grad_piece_kernel<true, G, true><<<grid, kThreads, 0, stream>>>(a);
    else grad_piece_kernel<true, G, false><<<grid, kThreads, 0, stream>>>(a);
  } else {
    if (vec) grad_piece_kernel<false, G, true><<<grid, kThreads, 0, stream>>>(a);
    else grad_piece_kernel<false, G, false><<<grid, kThreads, 0, stream>>>(a);
  }
}

}  // namespace
}  // namespace fluxmi

using namespace fluxmi;

extern "C" size_t fluxmi_moe_dgrad_workspace_bytes(int32_t nexperts, int64_t rows, int64_t n, int64_t k) {
  if (check_product("moe_dgrad", FLUXMI_ROWS_BF16, nexperts, rows, n, k) != FLUXMI_OK) return 0;
  return grad_tiles_workspace_bytes(Grad::INPUT, nexperts, rows, n, k);
}

extern "C" int fluxmi_moe_dgrad(const void *grad, const void *weight, int32_t row_type, const int32_t *splits, int32_t nexperts, int64_t rows, int64_t n,
                                int64_t k, void *grad_input, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int rc = check_product("moe_dgrad", row_type, nexperts, rows, n, k)) return rc;
  if (rows == 0 || k == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(grad_input && (n == 0 || grad) && (n == 0 || nexperts == 0 || weight) && (nexperts == 0 || splits), FLUXMI_ERR_INVALID_ARG,
                 "moe_dgrad: null pointer");
  FLUXMI_REQUIRE(on(grad, 2) && on(weight, 2) && on(splits, 4) && on(grad_input, 8), FLUXMI_ERR_INVALID_ARG,
                 "moe_dgrad: grad and weight must be aligned to their elements, splits to 4 bytes, grad_input to 8");
  GradArgs a{};
  a.grad = static_cast<const uint8_t *>(grad);
  a.other = static_cast<const uint8_t *>(weight);
  a.out = static_cast<uint8_t *>(grad_input);
  a.splits = splits;
  a.nexperts = nexperts;
  a.rows = static_cast<int32_t>(rows);
  a.n = static_cast<int32_t>(n);
  a.k = static_cast<int32_t>(k);
  a.parts = 1;
  a.partial = static_cast<float *>(workspace);
  const size_t need = fluxmi_moe_dgrad_workspace_bytes(nexperts, rows, n, k);
  FLUXMI_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && on(workspace, 16)), FLUXMI_ERR_WORKSPACE,
                 "moe_dgrad: workspace of %zu bytes, 16-byte aligned, expected, got %zu", need, workspace_bytes);
  if (grad_tiles_take(Grad::INPUT, a) && grad_tiles_are_faster(Grad::INPUT, nexperts, rows, n, k)) return launch_grad_tiles(Grad::INPUT, row_type == FLUXMI_ROWS_FP16, a, stream);
  // Every expert and the rows of none end with a tile that may be partial.
  const int64_t row_tiles = rows / kPiece + (rows < nexperts ? rows : nexperts) + 1, items = row_tiles * tiles_of(k);
  FLUXMI_REQUIRE(items <= kMostItems, FLUXMI_ERR_UNSUPPORTED, "moe_dgrad: too many rows and columns for one launch");
  const bool vec = n % 8 == 0 && k % 8 == 0 && on(grad, 16) && on(weight, 16);
  launch_pieces<Grad::INPUT>(a, row_type == FLUXMI_ROWS_FP16, vec, static_cast<uint32_t>(items), static_cast<hipStream_t>(stream));
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}

extern "C" size_t fluxmi_moe_wgrad_workspace_bytes(int32_t nexperts, int64_t rows, int64_t n, int64_t k) {
  if (check_product("moe_wgrad", FLUXMI_ROWS_BF16, nexperts, rows, n, k) != FLUXMI_OK) return 0;
  const int parts = parts_of(nexperts, rows, n, k);
  const size_t pieces = parts > 1 ? static_cast<size_t>(nexperts * tiles_of(n) * tiles_of(k)) * parts * kPiece * kPiece * sizeof(float) : 0;
  const size_t tiles = grad_tiles_workspace_bytes(Grad::WEIGHT, nexperts, rows, n, k);
  return pieces > tiles ? pieces : tiles;  // (which of them computes a call also depends on alignment)
}

extern "C" int fluxmi_moe_wgrad(const void *grad, const void *input, const void *input_scale, int32_t row_type, const int32_t *splits, int32_t nexperts,
                                int64_t rows, int64_t n, int64_t k, void *grad_weight, int32_t out_type, int32_t accumulate, void *workspace,
                                size_t workspace_bytes, void *stream) {
  if (const int rc = check_product("moe_wgrad", row_type, nexperts, rows, n, k)) return rc;
  FLUXMI_REQUIRE(out_type == row_type || out_type == FLUXMI_ROWS_FP32, FLUXMI_ERR_INVALID_ARG, "moe_wgrad: out_type %d (the rows' type and fp32 are built)", out_type);
  if (nexperts == 0 || n == 0 || k == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(grad_weight && splits && (rows == 0 || (grad && input)), FLUXMI_ERR_INVALID_ARG, "moe_wgrad: null pointer");
  FLUXMI_REQUIRE(on(grad, 2) && (input_scale != nullptr || on(input, 2)) && on(splits, 4) && on(grad_weight, 16), FLUXMI_ERR_INVALID_ARG,
                 "moe_wgrad: grad and input must be aligned to their elements, splits to 4 bytes, grad_weight to 16");
  GradArgs a{};
  a.grad = static_cast<const uint8_t *>(grad);
  a.other = static_cast<const uint8_t *>(input);
  a.scale = static_cast<const uint8_t *>(input_scale);
  a.out = static_cast<uint8_t *>(grad_weight);
  a.splits = splits;
  a.nexperts = nexperts;
  a.rows = static_cast<int32_t>(rows);
  a.n = static_cast<int32_t>(n);
  a.k = static_cast<int32_t>(k);
  a.out_f32 = out_type == FLUXMI_ROWS_FP32;
  a.accumulate = accumulate != 0;
  a.parts = parts_of(nexperts, rows, n, k);
  const Grad kind = input_scale != nullptr ? Grad::WEIGHT_8BIT : Grad::WEIGHT;
  const bool tiles = grad_tiles_take(kind, a) && grad_tiles_are_faster(kind, nexperts, rows, n, k);
  const int64_t pieces = nexperts * tiles_of(n) * tiles_of(k), items = pieces * a.parts;
  FLUXMI_REQUIRE(tiles || items <= kMostItems, FLUXMI_ERR_UNSUPPORTED, "moe_wgrad: too many experts, rows and columns for one launch");
  const size_t need = fluxmi_moe_wgrad_workspace_bytes(nexperts, rows, n, k);
  FLUXMI_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && on(workspace, 16)), FLUXMI_ERR_WORKSPACE,
                 "moe_wgrad: workspace of %zu bytes, 16-byte aligned, expected, got %zu", need, workspace_bytes);
  a.partial = static_cast<float *>(workspace);
  if (tiles) return launch_grad_tiles(kind, row_type == FLUXMI_ROWS_FP16, a, stream);
  const bool f16 = row_type == FLUXMI_ROWS_FP16;
  const bool vec = n % 8 == 0 && k % 8 == 0 && on(grad, 16) && on(input, input_scale != nullptr ? 8 : 16);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (input_scale != nullptr) launch_pieces<Grad::WEIGHT_8BIT>(a, f16, vec, static_cast<uint32_t>(items), s);
  else launch_pieces<Grad::WEIGHT>(a, f16, vec, static_cast<uint32_t>(items), s);
  FLUXMI_HIP_CHECK(hipGetLastError());
  if (a.parts > 1) {
    if (f16) grad_join_kernel<true><<<static_cast<uint32_t>(pieces * 16), kThreads, 0, s>>>(a);
    else grad_join_kernel<false><<<static_cast<uint32_t>(pieces * 16), kThreads, 0, s>>>(a);
    FLUXMI_HIP_CHECK(hipGetLastError());
  }
  return FLUXMI_OK;
}

extern "C" int fluxmi_moe_clear_rest(void *data, const int32_t *splits, int32_t nexperts, int64_t rows, int64_t row_bytes, void *stream) {
  if (const int rc = check_product("moe_clear_rest", FLUXMI_ROWS_BF16, nexperts, rows, 0, 0)) return rc;
  FLUXMI_REQUIRE(row_bytes >= 0 && row_bytes <= (int64_t{1} << 31), FLUXMI_ERR_INVALID_ARG, "moe_clear_rest: row_bytes=%lld", static_cast<long long>(row_bytes));
  if (rows == 0 || row_bytes == 0) return FLUXMI_OK;
  FLUXMI_REQUIRE(data && (nexperts == 0 || splits), FLUXMI_ERR_INVALID_ARG, "moe_clear_rest: null pointer");
  FLUXMI_REQUIRE(on(splits, 4), FLUXMI_ERR_INVALID_ARG, "moe_clear_rest: splits are not 4-byte aligned");
  GradArgs a{};
  a.out = static_cast<uint8_t *>(data);
  a.splits = splits;
  a.nexperts = nexperts;
  a.rows = static_cast<int32_t>(rows);
  clear_rest_kernel<<<kClearBlocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a, row_bytes);
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}
