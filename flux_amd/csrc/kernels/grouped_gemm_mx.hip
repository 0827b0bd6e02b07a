// Grouped product of MXFP4 operands: D[r, n] = row_scale[r] * sum_k A[row(r), k] * B[e(r), n, k].
//
// The MFMA takes the packed codes and the scale bytes as they lie in memory: of 16 x 16 x 128 a lane holds 16 bytes of codes, one block of 32
// values (lane l: row l & 15, block l >> 4), and the block's scale byte in a register of its own.  B's rows are the MFMA's rows, so that a lane's
// four sums are neighbouring columns of one row of D.
//
// Bound by the weights' bytes with few rows per expert, by the MFMAs and what feeds them with many.  Five kernels:
//  * streams (mx_stream_kernel), where there is less work than the card has room for: a wave, or two or four that split K, has 16 or 32 rows and 32 or 64 columns of
//    an expert and streams through LDS on its own;
//  * panels of 64 or 128 rows and 128 columns (mx_panel_kernel);
//  * the dual tiles of 256 x 256 (grouped_gemm_dual.hip);
//  * for many rows and what those do not take (K up to 512, more than 128 experts), mx_tile_kernel;
//  * for few rows whose scales are not on whole words (K that is no multiple of 128), mx_few_rows_kernel, whose four waves split K in turns of 512 values and load
//    straight into registers.  The others want a copy of such scales, of all experts.
//
// The tiles of this file: 256 x 256 on eight waves through a ring of four stages in LDS, a stage 128 values of K (64 bytes a row), filled by loads that write
// LDS.  The waves of a SIMD take turns: while one computes a stage, the other reads its fragments and requests fills.  Scales come 16 bytes a row for four
// stages, and lie in registers while those are computed.
#include "grouped_gemm_dual.hpp"
#include "rows.hpp"

namespace fluxmi {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kCols = 64;    // columns of a workgroup
constexpr int kMaxExperts = 1024;
constexpr int kPlanCus = 256;  // compute units that the choice of a kernel reckons with

struct MxParams {
  const uint8_t *a, *a_scale, *b, *b_scale;
  uint8_t *d;
  const int32_t *splits, *gather_a;
  const float *row_scale;
  int32_t nexperts, max_rows, n, kb, a_rows;  // kb: blocks of a row
  int32_t scale_stride;                       // bytes from row to row of the scales
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

// BYTE: the byte of both scale registers that the MFMA takes.
template <int BYTE>
__device__ __forceinline__ f32x4 mfma(const u32x4 w, const u32x4 x, uint32_t w_scale, uint32_t x_scale, f32x4 c) {
  const i32x8 wa = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3]), 0, 0, 0, 0};
  const i32x8 xa = {static_cast<int>(x[0]), static_cast<int>(x[1]), static_cast<int>(x[2]), static_cast<int>(x[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xa, c, 4, 4, BYTE, w_scale, BYTE, x_scale);
}

__device__ __forceinline__ void store_one(uint8_t *d, Row type, size_t i, float v) {
  if (type == Row::F32) reinterpret_cast<float *>(d)[i] = v;
  else reinterpret_cast<uint16_t *>(d)[i] = type == Row::BF16 ? float_to_bf16_bits(v) : float_to_f16_bits(v);
}

// Eight neighbouring results of one row, from column n on.
__device__ __forceinline__ void store_eight(const MxParams &p, int r, int n, const float (&v)[8]) {
  const size_t at = static_cast<size_t>(r) * p.n + n;
  if (n + 8 <= p.n) {
    if (p.d_type == Row::F32) {
      store16(p.d + at * 4, pack<Row::F32>(reinterpret_cast<const float(&)[4]>(v[0])));
      store16(p.d + at * 4 + 16, pack<Row::F32>(reinterpret_cast<const float(&)[4]>(v[4])));
    } else {
      store16(p.d + at * 2, p.d_type == Row::BF16 ? pack<Row::BF16>(v) : pack<Row::F16>(v));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (n + k < p.n) store_one(p.d, p.d_type, at + k, v[k]);
  }
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

// ---- tiles -----------------------------------------------------------------------------------------------------

// A tile: rows row0 .. row0 + rows of the sorted rows, all of expert e, columns from n0 on; rows == 0: there is no such tile.
struct TileItem {
  int e, row0, rows, n0;
};

// Workgroup -> tile.  Experts in order; an expert's rows are dealt to its row tiles evenly in units of 32, and its tiles are walked in groups of up to 8 row tiles,
// column by column.  Workgroups come to the eight XCDs in turn: each XCD has one stretch of that order, so that its L2 holds what its tiles share.
__device__ __forceinline__ TileItem locate_tile(const MxParams &p, int block, int tiles_n, int bm, int bn) {
  const int lane = threadIdx.x & 63;
  int row_carry = 0, piece_carry = 0, begin = 0, rows = 0, pieces_end = 0;
  auto scan = [&](int e0) {
    int r = 0;
    if (e0 + lane < p.nexperts) r = p.splits ? p.splits[e0 + lane] : p.max_rows;
    r = r < 0 ? 0 : (r > p.max_rows ? p.max_rows : r);
    const int incl = wave_inclusive_scan(r);
    int end = row_carry + incl;
    begin = end - r > p.max_rows ? p.max_rows : end - r;
    end = end > p.max_rows ? p.max_rows : end;
    rows = end - begin;
    row_carry = __builtin_amdgcn_readlane(end, 63);
    pieces_end = piece_carry + wave_inclusive_scan((rows + bm - 1) / bm);
    piece_carry = __builtin_amdgcn_readlane(pieces_end, 63);
  };
  for (int e0 = 0; e0 < p.nexperts; e0 += 64) scan(e0);
  const int per_xcd = (piece_carry * tiles_n + 7) / 8, i = block >> 3, item = (block & 7) * per_xcd + i;
  if (i >= per_xcd || item >= piece_carry * tiles_n) return {0, 0, 0, 0};
  row_carry = piece_carry = 0;
  for (int e0 = 0; e0 < p.nexperts; e0 += 64) {
    if (p.nexperts > 64) scan(e0);
    const uint64_t hit = __ballot(item < pieces_end * tiles_n);
    if (hit == 0) continue;
    const int src = __ffsll(static_cast<unsigned long long>(hit)) - 1;
    const int e_begin = __builtin_amdgcn_readlane(begin, src), e_rows = __builtin_amdgcn_readlane(rows, src);
    const int m_tiles = (e_rows + bm - 1) / bm, local = item - (__builtin_amdgcn_readlane(pieces_end, src) - m_tiles) * tiles_n;
    const int groups = (m_tiles + 7) / 8, per_group = (m_tiles + groups - 1) / groups;
    const int group = local / (per_group * tiles_n), group_rows = m_tiles - group * per_group < per_group ? m_tiles - group * per_group : per_group;
    const int in_group = local - group * per_group * tiles_n, nt = in_group / group_rows, mt = group * per_group + in_group - nt * group_rows;
    const int units = (e_rows + 31) / 32, per = units / m_tiles, longer = units - per * m_tiles;
    const int m0 = 32 * (mt * per + (mt < longer ? mt : longer)), height = 32 * (per + (mt < longer ? 1 : 0));
    TileItem t;
    t.e = __builtin_amdgcn_readfirstlane(e0 + src);
    t.row0 = __builtin_amdgcn_readfirstlane(e_begin + m0);
    t.rows = __builtin_amdgcn_readfirstlane(e_rows - m0 < height ? e_rows - m0 : height);
    t.n0 = __builtin_amdgcn_readfirstlane(nt * bn);
    return t;
  }
  return {0, 0, 0, 0};
}

#define FLUXMI_LGKM0() __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8))
#define FLUXMI_VMCNT(vm) __builtin_amdgcn_s_waitcnt(((vm)&15) | (((vm) >> 4) << 14) | (7 << 4) | (15 << 8))

// (Scales of a row's end are read 16 bytes at a time: words behind the last row's are zeros and not fetched, see buffer_of in grouped_gemm_rows.hpp.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void *base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, static_cast<int>(bytes), 0x00020000);
}

// 16 bytes a lane to LDS at `dst` + 16 * lane, zeros from an offset past the buffer.  (The scalar registers may come from vector instructions: five wait states
// lie between the statement's start and the load.)
__device__ __forceinline__ void fill(uint32_t dst, uint32_t off, __amdgpu_buffer_rsrc_t r, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(dst), "v"(off), "s"(r), "s"(soff) : "memory");
}

// The same, of bytes that are read once.
__device__ __forceinline__ void fill_once(uint32_t dst, uint32_t off, __amdgpu_buffer_rsrc_t r, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds" : : "s"(dst), "v"(off), "s"(r), "s"(soff) : "memory");
}

constexpr uint32_t kNoRow = 0x80000000u;  // a byte offset past every operand

// The column of a tile that row R of B's part of a stage holds: of 32 rows, lane group g finds columns 8 g .. 8 g + 7 in its sums of the two blocks of 16.
__device__ __forceinline__ int column_of(int R) { return (R & ~31) + 8 * ((R & 15) >> 2) + 4 * ((R >> 4) & 1) + (R & 3); }

#endif  // __HIP_DEVICE_COMPILE__

// MI x NJ blocks of 16 rows x 16 columns to a wave, WM x WN = 8 waves to a tile.
template <int MI, int NJ, int WM, int WN>
struct Tile {
  static constexpr int BM = MI * 16 * WM, BN = NJ * 16 * WN;
  static constexpr int XF = BM / 128, WF = BN / 128;            // fills of a wave for a stage
  static constexpr int kScaleFills = (BM + BN) / 64;             // fills of a tile for the scales of four stages, one or none to a wave
  static constexpr int kStage = (BM + BN) * 64, kStages = 4;
  static constexpr int kLds = kStage * kStages + (BM + BN) * 16;  // the ring, and the scales of four stages
  static_assert(WM * WN == 8 && BM % 128 == 0 && BN % 128 == 0 && kScaleFills <= 8, "");
};

template <int MI, int NJ, int WM, int WN>
__global__ __launch_bounds__(512, 2) void mx_tile_kernel(const MxParams p, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = Tile<MI, NJ, WM, WN>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const TileItem t = locate_tile(p, blockIdx.x, tiles_n, C::BM, C::BN);
  if (t.rows <= 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)smem));
  const int row_bytes = p.kb * 16, stages = (p.kb + 3) / 4;

  // ---- fills: LDS row R lies at R * 64, its chunk c of 16 bytes at slot c ^ turn(R >> 2); a fill covers 16 rows, lane l row l >> 2 and slot l & 3.  The turns
  // 0, 3, 2, 1 of every 16 rows keep the 16 lanes that LDS serves together (rows 0 to 3 and 12 to 15 of one lane group, 4 to 11 of the next) off each other's banks.
  auto turn = [](int q) { return -q & 3; };
  const int chunk = (lane & 3) ^ turn(lane >> 4);
  const auto xr = buffer_of(p.a, static_cast<int64_t>(p.a_rows) * row_bytes);
  const auto wr = buffer_of(p.b + static_cast<int64_t>(t.e) * p.n * row_bytes, static_cast<int64_t>(p.n) * row_bytes);
  const int scale_fill = wave % C::kScaleFills;  // (waves without one of their own repeat another's)
  const bool scales_of_a = scale_fill * 64 < C::BM;
  const auto sr = buffer_of(scales_of_a ? p.a_scale : p.b_scale + static_cast<int64_t>(t.e) * p.n * p.scale_stride,
                            static_cast<int64_t>(scales_of_a ? p.a_rows : p.n) * p.scale_stride);
  uint32_t xoff[C::XF], woff[C::WF], soff;
#pragma unroll
  for (int q = 0; q < C::XF; ++q) {
    const int m = (wave * C::XF + q) * 16 + (lane >> 2);
    xoff[q] = m < t.rows ? static_cast<uint32_t>(a_row(p, t.row0 + m)) * row_bytes + chunk * 16 : kNoRow;
  }
#pragma unroll
  for (int q = 0; q < C::WF; ++q) {
    const int n = t.n0 + column_of((wave * C::WF + q) * 16 + (lane >> 2));
    woff[q] = n < p.n ? static_cast<uint32_t>(n) * row_bytes + chunk * 16 : kNoRow;
  }
  {
    const int R = scale_fill * 64 + lane;  // A's rows, then B's
    if (R < C::BM) {
      soff = R < t.rows ? static_cast<uint32_t>(a_row(p, t.row0 + R)) * p.scale_stride : kNoRow;
    } else {
      const int n = t.n0 + column_of(R - C::BM);
      soff = n < p.n ? static_cast<uint32_t>(n) * p.scale_stride : kNoRow;
    }
  }
  // Stage s, into slot s mod 4; blocks past the end of the rows, and stages past the last, are zeros.
  auto fill_stage = [&](int s, int slot) {
    if (slot == 0) fill(lds0 + C::kStage * C::kStages + scale_fill * 1024, soff, sr, (s >> 2) * 16);
    const bool in = s * 4 + chunk < p.kb;
    const uint32_t dst = lds0 + slot * C::kStage;
#pragma unroll
    for (int q = 0; q < C::XF; ++q) fill(dst + (wave * C::XF + q) * 1024, in ? xoff[q] : kNoRow, xr, s * 64);
#pragma unroll
    for (int q = 0; q < C::WF; ++q) fill(dst + C::BM * 64 + (wave * C::WF + q) * 1024, in ? woff[q] : kNoRow, wr, s * 64);
  };

  // ---- fragments ---------------------------------------------------------------------------------------------
  typedef const __attribute__((address_space(3))) u32x4 *LdsFrag;
  // Wave rows: of both halves of the tile's rows MI / 2 blocks each, so that few rows are shared out evenly.
  const uint32_t in_rows = (lane & 15) * 64 + (((lane >> 4) ^ turn(lane >> 2)) * 16);
  const uint32_t xread = lds0 + wm * (MI * 8) * 64 + in_rows, wread = lds0 + (C::BM + wn * NJ * 16) * 64 + in_rows;
  const uint32_t in_scales = lds0 + C::kStage * C::kStages + (lane & 15) * 16;
  const uint32_t xsread = in_scales + wm * (MI * 8) * 16, wsread = in_scales + (C::BM + wn * NJ * 16) * 16;
  const bool has0 = wm * (MI * 8) < t.rows, has1 = C::BM / 2 + wm * (MI * 8) < t.rows;  // rows of the tile in the wave's halves
  u32x4 x[MI], w[NJ];
  uint32_t xs[MI], ws[NJ];  // byte s: the scale of this lane's block in stage s of four
  // 16 bytes of a row's scales, byte 4 s + g for the lanes of group g in stage s -> the lane's four.
  const uint32_t pick = 0x0c0c0400u + 0x0101u * (lane >> 4);
  auto scales_of = [&](uint32_t at) {
    const u32x4 v = *reinterpret_cast<LdsFrag>(at);
    const uint32_t lo = __builtin_amdgcn_perm(v[1], v[0], pick), hi = __builtin_amdgcn_perm(v[3], v[2], pick);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  };
  auto read_stage = [&](int slot) {
    const uint32_t xat = xread + slot * C::kStage, wat = wread + slot * C::kStage;
#pragma unroll
    for (int j = 0; j < NJ; ++j) w[j] = *reinterpret_cast<LdsFrag>(wat + j * 1024);
#pragma unroll
    for (int i = 0; i < MI; ++i) x[i] = *reinterpret_cast<LdsFrag>(xat + (i / (MI / 2)) * (C::BM / 2) * 64 + (i % (MI / 2)) * 1024);
    if (slot == 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) ws[j] = scales_of(wsread + j * 256);
#pragma unroll
      for (int i = 0; i < MI; ++i) xs[i] = scales_of(xsread + (i / (MI / 2)) * (C::BM / 2) * 16 + (i % (MI / 2)) * 256);
    }
  };
  f32x4 acc[MI][NJ] = {};
  auto compute = [&](auto SLOT) {
    constexpr int slot = decltype(SLOT)::value;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 0 ? !has0 : !has1) continue;
#pragma unroll
      for (int i = h * (MI / 2); i < (h + 1) * (MI / 2); ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mfma<slot>(w[j], x[i], ws[j], xs[i], acc[i][j]);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto sync = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // ---- the loop over K ----------------------------------------------------------------------------------------
  // The four waves of a group, one to a SIMD, compute a stage while the others read their fragments and request fills; a barrier ends the phase for both.
  // Both groups run the same code, the second one phase behind: the first reads stage s in phase 2 s - 1 and computes it in 2 s, the second reads it in
  // 2 s and computes it in 2 s + 1.  Whoever reads stage s requests s + 3, whose slot was that of stage s - 1, which nobody reads after phase 2 s - 2.
  // Stage s + 1 has to have come when phase 2 s ends; then stages s + 2 and s + 3 of a wave may be on their way.
  constexpr int kFills = C::XF + C::WF;
  const bool behind = wave >= 4;
  fill_stage(0, 0);
  fill_stage(1, 1);
  fill_stage(2, 2);
  FLUXMI_VMCNT(2 * kFills);
  sync();
  if (behind) sync();
  auto stage = [&](auto SLOT, int s) {
    constexpr int slot = decltype(SLOT)::value, kYounger = 2 * kFills + (slot == 1 || slot == 2 ? 1 : 0);  // (scales come with every fourth stage)
    read_stage(slot);
    fill_stage(s + 3, (slot + 3) & 3);
    if (behind) FLUXMI_VMCNT(kYounger);
    FLUXMI_LGKM0();
    sync();
    compute(SLOT);
    if (!behind) FLUXMI_VMCNT(kYounger);
    sync();
  };
  for (int s = 0;;) {
    stage(std::integral_constant<int, 0>{}, s);
    if (++s == stages) break;
    stage(std::integral_constant<int, 1>{}, s);
    if (++s == stages) break;
    stage(std::integral_constant<int, 2>{}, s);
    if (++s == stages) break;
    stage(std::integral_constant<int, 3>{}, s);
    if (++s == stages) break;
  }
  if (!behind) sync();
  FLUXMI_VMCNT(0);  // fills past the end write zeros: LDS is this workgroup's until they have

  // ---- results: lane group g has columns 8 g .. 8 g + 7 of each 32, of row lane & 15 of each block ------------------
  float rs[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = (i / (MI / 2)) * (C::BM / 2) + wm * (MI * 8) + (i % (MI / 2)) * 16 + (lane & 15);
    rs[i] = p.row_scale && m < t.rows ? p.row_scale[t.row0 + m] : 1.f;
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = (i / (MI / 2)) * (C::BM / 2) + wm * (MI * 8) + (i % (MI / 2)) * 16 + (lane & 15);
    if (m >= t.rows) continue;
#pragma unroll
    for (int jg = 0; jg < NJ / 2; ++jg) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = acc[i][2 * jg + k / 4][k % 4] * rs[i];
      store_eight(p, t.row0 + m, t.n0 + wn * NJ * 16 + jg * 32 + (lane >> 4) * 8, v);
    }
  }
#endif  // __HIP_DEVICE_COMPILE__
}

// ---- panels ----------------------------------------------------------------------------------------------------

// MI x 2 blocks of 16 x 16 to a wave, 2 x 4 waves: up to 32 MI rows and 128 columns of one expert.  LDS holds S steps of 256 values of K.
template <int MI>
struct Panel {
  static constexpr int S = 3;
  static constexpr int BM = 32 * MI, BN = 128;
  static constexpr int XF = BM / 32, WF = 4;  // fills of a step, of each of the four waves that request them
  static constexpr int kW = S * BM * 128, kXs = kW + S * BN * 128, kWs = kXs + 2 * BM * 16, kLds = kWs + 2 * BN * 16;  // (scales: of two pairs of steps)
  static_assert(MI % 2 == 0 && kLds <= 160 * 1024, "");
};

// A step is a line of 128 bytes of each row.  All waves read the panel's rows of A from one copy in LDS, which leaves more of it to the weights on their way than the
// streams have, whose waves have a copy each; two workgroups of 64 rows to a compute unit.  Bound by the weights' bytes: 9 to 48 rows of 8 experts 4096 x 14336 43
// to 47 us (5.9 to 5.5 TB/s), 32 rows of 32 experts 2048 x 7168 47, 7168 x 2048 57 (4.8).  Waves 0 to 3 request A's lines, waves 4 to 7 B's.  More steps in LDS
// take workgroups off the compute unit (five of B: 52 and 71 us), two steps let its loads run dry (65 instead of 45 for 24 rows 4096 x 14336).
template <int MI>
__global__ __launch_bounds__(512, 2) void mx_panel_kernel(const MxParams p, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = Panel<MI>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const TileItem t = locate_tile(p, blockIdx.x, tiles_n, C::BM, C::BN);
  if (t.rows <= 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)smem));
  const int row_bytes = p.kb * 16, steps = (p.kb + 7) / 8;
  const bool of_a = wave < 4;  // whose fills this wave requests
  const uint8_t *const codes = of_a ? p.a : p.b + static_cast<int64_t>(t.e) * p.n * row_bytes;
  const uint8_t *const scales = of_a ? p.a_scale : p.b_scale + static_cast<int64_t>(t.e) * p.n * p.scale_stride;
  const int64_t rows_of = of_a ? p.a_rows : p.n;
  const auto cr = buffer_of(codes, rows_of * row_bytes), sr = buffer_of(scales, rows_of * p.scale_stride);
  // ---- fills: rows of 128 bytes as in the streams; wave q of four has the fills q, q + 4 ... of 8 rows each.  (Of B: four of them.)
  uint32_t off[C::XF > C::WF ? C::XF : C::WF], soff = kNoRow;
  const int place = (lane & 7) ^ (lane >> 4);
  const uint32_t chunk = (((place & 3) * 2 + (place >> 2)) ^ (wn & 1)) * 16;  // (fill q * 4 + wn has the parity of wn)
#pragma unroll
  for (int q = 0; q < (C::XF > C::WF ? C::XF : C::WF); ++q) {
    const int R = (q * 4 + wn) * 8 + (lane >> 3);
    if (of_a) {
      off[q] = R < t.rows ? static_cast<uint32_t>(a_row(p, t.row0 + R)) * row_bytes + chunk : kNoRow;
    } else {
      const int n = t.n0 + column_of(R);
      off[q] = n < p.n ? static_cast<uint32_t>(n) * row_bytes + chunk : kNoRow;
    }
  }
  const int scale_fill = of_a ? wn % (C::BM / 64) : wn & 1;  // of 64 rows each (more waves than fills: some repeat another's)
  {
    const int R = scale_fill * 64 + lane;
    if (of_a) {
      if (R < t.rows) soff = static_cast<uint32_t>(a_row(p, t.row0 + R)) * p.scale_stride;
    } else {
      const int n = t.n0 + column_of(R);
      if (n < p.n) soff = static_cast<uint32_t>(n) * p.scale_stride;
    }
  }
  // Step s, into `slot`; blocks past the end of the rows are zero codes, and what lies there instead of their scales is masked when it is used.  With the first step of
  // a pair come the scales of both.
  auto fill_step = [&](int s, int slot) {
    if ((s & 1) == 0)
      fill(lds0 + (of_a ? C::kXs + ((s >> 1) & 1) * (C::BM * 16) : C::kWs + ((s >> 1) & 1) * (C::BN * 16)) + scale_fill * 1024, s < steps ? soff : kNoRow, sr, (s >> 1) * 16);
    const bool in = s * 8 + static_cast<int>(chunk >> 4) < p.kb;
    if (of_a) {
#pragma unroll
      for (int q = 0; q < C::XF; ++q) fill(lds0 + slot * (C::BM * 128) + (q * 4 + wn) * 1024, in ? off[q] : kNoRow, cr, s * 128);
    } else {
#pragma unroll
      for (int q = 0; q < C::WF; ++q) fill_once(lds0 + C::kW + slot * (C::BN * 128) + (q * 4 + wn) * 1024, in ? off[q] : kNoRow, cr, s * 128);
    }
  };
  // ---- fragments: lane group g has chunks 2 g and 2 g + 1 of a line in two MFMAs, and bytes 2 g and 2 g + 1 of the line's 8 scales.
  typedef const __attribute__((address_space(3))) u32x4 *LdsFrag;
  typedef const __attribute__((address_space(3))) uint16_t *LdsPair;
  const int g = lane >> 4, r = lane & 15;
  const uint32_t in_rows0 = r * 128 + ((g ^ ((lane >> 1) & 7)) * 16), in_rows1 = r * 128 + (((4 + g) ^ ((lane >> 1) & 7)) * 16);
  // Wave rows: of both halves of the panel's rows MI / 2 blocks each, so that few rows are shared out evenly.
  auto block_row = [&](int i) { return (i / (MI / 2)) * (C::BM / 2) + wm * (MI * 8) + (i % (MI / 2)) * 16; };
  const bool has0 = block_row(0) < t.rows, has1 = block_row(MI / 2) < t.rows;
  f32x4 acc[MI][2] = {};
  auto compute = [&](auto PARITY, int s, int slot) {
    constexpr int PAR = decltype(PARITY)::value;
    const uint32_t x_at = lds0 + slot * (C::BM * 128), w_at = lds0 + C::kW + slot * (C::BN * 128) + wn * 4096;
    const uint32_t xs_at = lds0 + C::kXs + ((s >> 1) & 1) * (C::BM * 16) + r * 16 + PAR * 8 + g * 2;
    const uint32_t ws_at = lds0 + C::kWs + ((s >> 1) & 1) * (C::BN * 16) + wn * 512 + r * 16 + PAR * 8 + g * 2;
    const int first = s * 8 + 2 * g;  // this lane's two blocks
    const uint32_t known = first + 1 < p.kb ? 0xffffu : first < p.kb ? 0xffu : 0u;
    u32x4 w[2][2];
    uint32_t ws[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      w[j][0] = *reinterpret_cast<LdsFrag>(w_at + in_rows0 + j * 2048);
      w[j][1] = *reinterpret_cast<LdsFrag>(w_at + in_rows1 + j * 2048);
      ws[j] = *reinterpret_cast<LdsPair>(ws_at + j * 256) & known;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 0 ? !has0 : !has1) continue;
#pragma unroll
      for (int i = h * (MI / 2); i < (h + 1) * (MI / 2); ++i) {
        const u32x4 x0 = *reinterpret_cast<LdsFrag>(x_at + in_rows0 + block_row(i) * 128), x1 = *reinterpret_cast<LdsFrag>(x_at + in_rows1 + block_row(i) * 128);
        const uint32_t xs = *reinterpret_cast<LdsPair>(xs_at + block_row(i) * 16) & known;
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma<0>(w[j][0], x0, ws[j], xs, acc[i][j]);
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma<1>(w[j][1], x1, ws[j], xs, acc[i][j]);
      }
    }
  };
  auto sync = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // ---- the loop over K: after the barrier of step s its operands are there, and what step s - 1 had is free.  A wave requests step s + 2 then, and waits for step
  // s + 1 at the end, when the fills of step s + 2 may be on their way, with a pair's scales if s is even.
  fill_step(0, 0);
  fill_step(1, 1);
  if (of_a) FLUXMI_VMCNT(C::XF);
  else FLUXMI_VMCNT(C::WF);
  sync();
  int slot = 0;
  auto step = [&](auto PARITY, int s) {
    constexpr int PAR = decltype(PARITY)::value;
    fill_step(s + 2, slot == 0 ? 2 : slot - 1);
    __builtin_amdgcn_sched_barrier(0);
    compute(PARITY, s, slot);
    FLUXMI_LGKM0();
    if (of_a) FLUXMI_VMCNT(C::XF + 1 - PAR);
    else FLUXMI_VMCNT(C::WF + 1 - PAR);
    sync();
    slot = slot == 2 ? 0 : slot + 1;
  };
  for (int s = 0; s < steps; s += 2) {  // (an odd last step has one of zeros behind it)
    step(std::integral_constant<int, 0>{}, s);
    step(std::integral_constant<int, 1>{}, s + 1);
  }
  FLUXMI_VMCNT(0);  // fills past the end write zeros: LDS is this workgroup's until they have

  // ---- results: lane group g has columns 8 g .. 8 g + 7 of the wave's 32, of row r of each block
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = block_row(i) + r;
    if (m >= t.rows) continue;
    const float scale = p.row_scale ? p.row_scale[t.row0 + m] : 1.f;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = acc[i][k / 4][k % 4] * scale;
    store_eight(p, t.row0 + m, t.n0 + wn * 32 + g * 8, v);
  }
#endif  // __HIP_DEVICE_COMPILE__
}

// Scales in rows of a multiple of 16 bytes, zeros behind their end: A's rows, then those of all experts.
__global__ __launch_bounds__(kThreads) void mx_pad_scales_kernel(const uint8_t *__restrict__ a, int64_t a_rows, const uint8_t *__restrict__ b, int64_t b_rows, int kb, int stride,
                                                                 uint8_t *__restrict__ out) {
  const int per_row = stride / 16;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < (a_rows + b_rows) * per_row; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / per_row;
    const int c = static_cast<int>(i - row * per_row) * 16;
    const uint8_t *const src = (row < a_rows ? a + row * kb : b + (row - a_rows) * kb) + c;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (c + 16 <= kb) {
      v = load16(src);
    } else {
      for (int k = 0; k < kb - c; ++k) v[k / 4] |= static_cast<uint32_t>(src[k]) << (8 * (k & 3));
    }
    store16(out + i * 16, v);
  }
}

// MT blocks of 16 rows x NJ blocks of 16 columns, P waves that split K.
template <int MT, int NJ, int P>
struct Stream {
  static constexpr int kX = NJ * 4096, kScales = kX + MT * 4096, kStage = kScales + 2048;  // of a stage: codes of B, of A, scales of B, of A
  static constexpr int kFills = 4 * (NJ + MT) + 2, kWaveLds = 2 * kStage, kLds = P * kWaveLds;
};

// A wave is on its own until the end: it requests a turn's 512 values of K of its columns and rows into one half of its LDS while it computes the other half's, with
// no barrier.  Weights come in whole lines, eight rows of 128 bytes to a load, and non-temporally, as nobody else reads them.
template <int MT, int NJ, int P>
__global__ __launch_bounds__(64 * P) void mx_stream_kernel(const MxParams p, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = Stream<MT, NJ, P>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = P == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x / tiles_n, n0 = (blockIdx.x - item * tiles_n) * (NJ * 16);
  const Item it = locate(p, item, MT * 16);
  if (it.rows <= 0) return;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)smem)) + wave * C::kWaveLds;
  const int row_bytes = p.kb * 16, turns = (p.kb + 15) / 16;
  const auto xr = buffer_of(p.a, static_cast<int64_t>(p.a_rows) * row_bytes), xsr = buffer_of(p.a_scale, static_cast<int64_t>(p.a_rows) * p.scale_stride);
  const auto wr = buffer_of(p.b + static_cast<int64_t>(it.e) * p.n * row_bytes, static_cast<int64_t>(p.n) * row_bytes);
  const auto wsr = buffer_of(p.b_scale + static_cast<int64_t>(it.e) * p.n * p.scale_stride, static_cast<int64_t>(p.n) * p.scale_stride);
  // LDS row R of 128 bytes: its chunks of 16 bytes in the order 0, 2, 4, 6, 1, 3, 5, 7, the c-th of them at slot c ^ ((R >> 1) & 7); a fill covers 8 rows, lane l row
  // l >> 3 and slot l & 7.  (The 16 lanes that LDS serves together, of two lane groups, are so on banks of their own.)
  uint32_t xoff[2 * MT], woff[2 * NJ];
  const int place = (lane & 7) ^ (lane >> 4);  // of even fills; odd ones: ^ 4
  const uint32_t chunk0 = ((place & 3) * 2 + (place >> 2)) * 16;
#pragma unroll
  for (int q = 0; q < 2 * NJ; ++q) {
    const int n = n0 + column_of(q * 8 + (lane >> 3));
    woff[q] = n < p.n ? static_cast<uint32_t>(n) * row_bytes + (chunk0 ^ ((q & 1) * 16)) : kNoRow;
  }
  const int ns = n0 + column_of(lane);
  const uint32_t wsoff = lane < NJ * 16 && ns < p.n ? static_cast<uint32_t>(ns) * p.scale_stride : kNoRow;
#pragma unroll
  for (int q = 0; q < 2 * MT; ++q) {
    const int m = q * 8 + (lane >> 3);
    xoff[q] = m < it.rows ? static_cast<uint32_t>(a_row(p, it.row0 + m)) * row_bytes + (chunk0 ^ ((q & 1) * 16)) : kNoRow;
  }
  const uint32_t xsoff = lane < it.rows ? static_cast<uint32_t>(a_row(p, it.row0 + lane)) * p.scale_stride : kNoRow;  // (lanes past the rows' blocks: not read)
  // Blocks past the end of the rows are zero codes; what lies there instead of their scales is masked when it is used.
  auto fill_turn_of = [&](auto LAST, int t, int slot) {
    constexpr bool kLast = decltype(LAST)::value;
    const uint32_t dst = lds0 + slot * C::kStage;
    auto in_row = [&](uint32_t off, int q, int h) {
      if constexpr (kLast) return t * 16 + h * 8 + static_cast<int>((chunk0 >> 4) ^ (q & 1)) < p.kb ? off : kNoRow;
      else return off;
    };
    fill_once(dst + C::kScales, wsoff, wsr, t * 16);
#pragma unroll
    for (int q = 0; q < 4 * NJ; ++q) fill_once(dst + q * 1024, in_row(woff[q % (2 * NJ)], q, q / (2 * NJ)), wr, t * 256 + q / (2 * NJ) * 128);
    fill(dst + C::kScales + 1024, xsoff, xsr, t * 16);
#pragma unroll
    for (int q = 0; q < 4 * MT; ++q) fill(dst + C::kX + q * 1024, in_row(xoff[q % (2 * MT)], q, q / (2 * MT)), xr, t * 256 + q / (2 * MT) * 128);
  };
  auto fill_turn = [&](int t, int slot) {
    if (t * 16 + 16 <= p.kb) fill_turn_of(std::false_type{}, t, slot);
    else fill_turn_of(std::true_type{}, t, slot);
  };
  // Lane group g has chunks 2 g and 2 g + 1 of a line in two MFMAs, and their scales are bytes 2 g and 2 g + 1 of the line's 8.
  typedef const __attribute__((address_space(3))) u32x4 *LdsFrag;
  typedef const __attribute__((address_space(3))) uint32_t *LdsWord;
  const int g = lane >> 4, r = lane & 15;
  const uint32_t in_rows0 = r * 128 + ((g ^ ((lane >> 1) & 7)) * 16), in_rows1 = r * 128 + (((4 + g) ^ ((lane >> 1) & 7)) * 16);
  const uint32_t in_scales = C::kScales + r * 16 + (g >> 1) * 4, pick = 0x05040100u + 0x02020202u * (g & 1);
  f32x4 acc[MT][NJ] = {};
  int slot = 0;
  if (wave < turns) fill_turn(wave, 0);
  if (wave + P < turns) fill_turn(wave + P, 1);
  for (int t = wave; t < turns; t += P) {
    if (t + P < turns) FLUXMI_VMCNT(C::kFills);
    else FLUXMI_VMCNT(0);
    asm volatile("" ::: "memory");
    const uint32_t at = lds0 + slot * C::kStage;
    u32x4 w[NJ][4], x[MT][4];
    uint32_t ws[NJ], xs[MT];
    uint32_t known = ~0u;  // bytes of blocks that the rows have
    if (t * 16 + 16 > p.kb) {
      known = 0;
#pragma unroll
      for (int m = 0; m < 4; ++m) known |= t * 16 + (m >> 1) * 8 + 2 * g + (m & 1) < p.kb ? 0xffu << (8 * m) : 0u;
    }
    auto scales_of = [&](uint32_t a) { return __builtin_amdgcn_perm(*reinterpret_cast<LdsWord>(a + 8), *reinterpret_cast<LdsWord>(a), pick) & known; };
#pragma unroll
    for (int j = 0; j < NJ; ++j) ws[j] = scales_of(at + in_scales + j * 256);
#pragma unroll
    for (int i = 0; i < MT; ++i) xs[i] = scales_of(at + in_scales + 1024 + i * 256);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        w[j][2 * h] = *reinterpret_cast<LdsFrag>(at + in_rows0 + h * NJ * 2048 + j * 2048);
        w[j][2 * h + 1] = *reinterpret_cast<LdsFrag>(at + in_rows1 + h * NJ * 2048 + j * 2048);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        x[i][2 * h] = *reinterpret_cast<LdsFrag>(at + C::kX + in_rows0 + h * MT * 2048 + i * 2048);
        x[i][2 * h + 1] = *reinterpret_cast<LdsFrag>(at + C::kX + in_rows1 + h * MT * 2048 + i * 2048);
      }
    }
    FLUXMI_LGKM0();  // all of this half is in registers: the turn after the next may come into it
    __builtin_amdgcn_sched_barrier(0);
    if (t + 2 * P < turns) fill_turn(t + 2 * P, slot);
    auto multiply = [&](auto M) {
      constexpr int m = decltype(M)::value;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mfma<m>(w[j][m], x[i][m], ws[j], xs[i], acc[i][j]);
    };
    multiply(std::integral_constant<int, 0>{});
    multiply(std::integral_constant<int, 1>{});
    multiply(std::integral_constant<int, 2>{});
    multiply(std::integral_constant<int, 3>{});
    slot ^= 1;
  }
  // The waves' sums, in their order; wave v stores every P-th group of 16 rows x 32 columns from the v-th on.
  typedef __attribute__((address_space(3))) f32x4 *LdsSums;
  if constexpr (P > 1) {
    FLUXMI_VMCNT(0);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) *reinterpret_cast<LdsSums>(lds0 + (i * NJ + j) * 1024 + lane * 16) = acc[i][j];
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < MT * NJ / 2; ++q) {
    if (P > 1 && q % P != wave) continue;
    const int i = q / (NJ / 2), jg = q % (NJ / 2), m = i * 16 + r;
    f32x4 sum[2] = {acc[i][2 * jg], acc[i][2 * jg + 1]};
    if constexpr (P > 1) {
      const uint32_t first = lds0 - wave * C::kWaveLds + (i * NJ + 2 * jg) * 1024 + lane * 16;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        sum[k] = *reinterpret_cast<LdsSums>(first + k * 1024);
        for (int v = 1; v < P; ++v) sum[k] += *reinterpret_cast<LdsSums>(first + v * C::kWaveLds + k * 1024);
      }
    }
    if (m >= it.rows) continue;
    const float scale = p.row_scale ? p.row_scale[it.row0 + m] : 1.f;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = sum[k / 4][k % 4] * scale;
    store_eight(p, it.row0 + m, n0 + jg * 32 + g * 8, v);
  }
#endif  // __HIP_DEVICE_COMPILE__
}

__global__ __launch_bounds__(kThreads) void mx_few_rows_kernel(const MxParams p, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int MT = 1;
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
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma<0>(wt[j].code[s], xt[i].code[s], wt[j].scale[s], xt[i].scale[s], acc[i][j]);
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

int launch_few_rows(const MxParams &p, hipStream_t s) {
  const int tiles_n = (p.n + kCols - 1) / kCols;
  // Pieces of rows: at most one that is not full for each expert with rows.
  const int64_t items = p.max_rows / 16 + (p.nexperts < p.max_rows ? p.nexperts : p.max_rows), grid = items * tiles_n;
  FLUXMI_REQUIRE(grid * kThreads < (int64_t{1} << 32), FLUXMI_ERR_UNSUPPORTED, "grouped_gemm_mx: max_rows=%d and n=%d are more than a launch covers", p.max_rows, p.n);
  hipLaunchKernelGGL(mx_few_rows_kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s, p, tiles_n);
  return FLUXMI_OK;
}

template <int MT, int NJ, int P>
int launch_stream(const MxParams &p, hipStream_t s) {
  using C = Stream<MT, NJ, P>;
  static std::atomic<uint64_t> lds_done{0};
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(mx_stream_kernel<MT, NJ, P>), C::kLds, lds_done);
  if (rc != FLUXMI_OK) return rc;
  const int tiles_n = (p.n + NJ * 16 - 1) / (NJ * 16);
  const int64_t items = p.max_rows / (MT * 16) + (p.nexperts < p.max_rows ? p.nexperts : p.max_rows), grid = items * tiles_n;
  FLUXMI_REQUIRE(grid * 64 * P < (int64_t{1} << 32), FLUXMI_ERR_UNSUPPORTED, "grouped_gemm_mx: max_rows=%d and n=%d are more than a launch covers", p.max_rows, p.n);
  hipLaunchKernelGGL((mx_stream_kernel<MT, NJ, P>), dim3(static_cast<unsigned>(grid)), dim3(64 * P), C::kLds, s, p, tiles_n);
  return FLUXMI_OK;
}

template <int MI, int NJ, int WM, int WN>
int launch_tiles(const MxParams &p, hipStream_t s) {
  using C = Tile<MI, NJ, WM, WN>;
  static std::atomic<uint64_t> lds_done{0};
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(mx_tile_kernel<MI, NJ, WM, WN>), C::kLds, lds_done);
  if (rc != FLUXMI_OK) return rc;
  const int tiles_n = (p.n + C::BN - 1) / C::BN;
  const int64_t pieces = p.max_rows / C::BM + (p.nexperts < p.max_rows ? p.nexperts : p.max_rows), grid = (pieces * tiles_n + 7) / 8 * 8;
  FLUXMI_REQUIRE(grid * 512 < (int64_t{1} << 32), FLUXMI_ERR_UNSUPPORTED, "grouped_gemm_mx: max_rows=%d and n=%d are more than a launch covers", p.max_rows, p.n);
  hipLaunchKernelGGL((mx_tile_kernel<MI, NJ, WM, WN>), dim3(static_cast<unsigned>(grid)), dim3(512), C::kLds, s, p, tiles_n);
  return FLUXMI_OK;
}

template <int MI>
int launch_panel(const MxParams &p, hipStream_t s) {
  using C = Panel<MI>;
  static std::atomic<uint64_t> lds_done{0};
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(mx_panel_kernel<MI>), C::kLds, lds_done);
  if (rc != FLUXMI_OK) return rc;
  const int tiles_n = (p.n + C::BN - 1) / C::BN;
  const int64_t pieces = p.max_rows / C::BM + (p.nexperts < p.max_rows ? p.nexperts : p.max_rows), grid = (pieces * tiles_n + 7) / 8 * 8;
  FLUXMI_REQUIRE(grid * 512 < (int64_t{1} << 32), FLUXMI_ERR_UNSUPPORTED, "grouped_gemm_mx: max_rows=%d and n=%d are more than a launch covers", p.max_rows, p.n);
  hipLaunchKernelGGL((mx_panel_kernel<MI>), dim3(static_cast<unsigned>(grid)), dim3(512), C::kLds, s, p, tiles_n);
  return FLUXMI_OK;
}

// The call as the dual tiles take it.
GemmParams dual_params(const fluxmi_mx_gemm_args &a) {
  GemmParams p{};
  p.a = static_cast<const uint8_t *>(a.a);
  p.b[0] = static_cast<const uint8_t *>(a.b);
  p.d[0] = a.d;
  p.splits = a.splits;
  p.gather_a = a.gather_a;
  p.row_scale = a.row_scale;
  p.scalar = 1.f;
  p.nexperts = a.nexperts;
  p.max_rows = a.max_rows;
  p.a_rows = a.a_rows;
  p.n = a.n;
  p.k = (a.k + 31) / 32 * 32;  // the codes past the end are zeros
  p.d_fp32 = a.d_type == FLUXMI_ROWS_FP32;
  p.half_is_f16 = a.d_type == FLUXMI_ROWS_FP16;
  p.ngroups = 1;
  p.raster_rows = 8;
  p.a_scale = static_cast<const float *>(a.a_scale);
  p.b_scale = static_cast<const float *>(a.b_scale);
  return p;
}

// Which kernel computes a call.
enum class Form { FEW_ROWS, STREAM, PANEL, DUAL, TILES };
struct Plan {
  Form form;
  int row_blocks, col_blocks, waves;  // STREAM: blocks of 16 rows and of 16 columns of an item, waves that split K; PANEL: row blocks of 32
  size_t workspace;                   // scales in rows of whole 16 bytes
};

// By the rows of an expert on average and by how many workgroups the card gets.  us, rows a fifth more and less on every other expert:
//  streams / panels of 64 / of 128 / dual tiles
//  few panels: one token of two experts 4096 x 14336 (64 panels) 13 / 33, 14336 x 4096 (224) 13.8 / 14.4 / - / 26; 4 experts 4096 x 7168 (128), 9 rows 14 / 20, 20 rows
//  16 / 21, 40 rows 22 / 23; one expert 4096 x 4096, 60 rows 6.4 / 15 / 15 / 25, 256 rows (128) 14 / 14 / 19 / 28, 512 rows (256) 27 / 16 / 20 / 27, 1024 rows (512; 256
//  of 128 rows) 50 / 26 / 21 / 29; 2 experts 14336 x 4096 (224), 30 rows 21 / 16 / 17 / 26; 6 experts 4096 x 7168 (192), 20 rows 23.3 / 22.4
//  up to 48 rows: 8 experts 4096 x 14336 (256), 5 rows 49 / 42, 9 rows 49 / 43, 24 rows 54 / 45 / 48 / 69; 14336 x 4096 (896), 5 rows 46 / 46, 9 rows 47 / 47, 24 rows
//  61 / 51 / 62 / 61, 48 rows - / 57 / 67 / 63; 32 experts 2048 x 7168 (512), 9 rows 52 / 43, 32 rows 78 / 47 / 54 / 53; 7168 x 2048, 32 rows 77 / 57 / 70 / 67
//  more: 8 experts 4096 x 14336 (256 of 128 rows), 60 rows - / 82 / 52 / 75, 100 rows - / 84 / 60 / 79; 32 experts 2048 x 7168 (512), 60 rows - / 72 / 59 / 58, 100 rows
//  - / 95 / 65 / 63; 14336 x 4096 (896), 60 rows - / 82 / 71 / 67; one expert 4096 x 14336, 1024 rows (256) 161 / 74 / 54 / 68, 2048 rows (512) - / 145 / 106 / 84.
// The waves of a stream: one token of two experts 4096 x 14336 (256 streams) 16.3 / 13.0 / 13.4 of one, two and four that split K, with 896 (14336 x 4096) 13.8 / 15.7;
// of 32 rows one expert 4096 x 4096, 128 rows (512 streams) 9.4 / 9.5 / 12.5, 1024 x 4096, 256 rows (256) 8.1 / 6.0 / 6.8, 128 rows (128) 8.0 / 5.9 / 5.6.  64 columns of
// 32 rows: one expert 4096 x 14336, 256 rows (1024 streams) 46 -> 37, with fewer streams it is slower.
// Scales that are not on words (K = 2880), few rows straight to registers / streams and panels with a copy of all scales: 32 experts of 5760 columns, 1 row each 65 / 85,
// 16 rows 73 / 92, 20 rows 115 / 93, 48 rows 165 / 100; 128 experts of 768, 1 row 35 / 53, 16 rows 42 / 56, 20 rows 66 / 57; 8 experts of 4096, 16 rows 13.0 / 19.7, 20 to
// 32 rows the same, 48 rows 24.1 / 21.6; only with one or two experts would 48 rows still be better off (2880 columns 11.0 / 13.0).  K = 2816, which needs neither: 32 experts of
// 5760 columns, 1 row 51, 32 rows 60 (K = 2880: 97, the copy 15 of them and the panels 80: rows of 1440 bytes do not start on lines).
// What keeps the dual tiles off (K up to 512, more than 128 experts) goes to the tiles of this file, which are slower (8 experts 14336 x 4224, 194 rows 102 -> 110, 1200 rows
// 379 -> 431; 4095 x 14336, 600 rows 195 -> 245).  Panels of 256 rows would be as good as the dual tiles at 194 rows 4096 x 14336 (86 / 91) and worse where some experts have
// more than 256 (4 experts of 176 and 264 rows 8192 x 4096 58 / 40).
Plan plan_of(const fluxmi_mx_gemm_args &a, const GemmParams &dual, int cus) {
  const int64_t rows = a.max_rows, experts = a.nexperts, active = rows < experts ? rows : experts, kb = (int64_t{a.k} + 31) / 32;
  const int64_t each = (rows + active - 1) / active;  // rows of an expert on average
  auto pieces = [&](int64_t high, int64_t wide) { return active * ((each + high - 1) / high) * ((a.n + wide - 1) / wide); };
  auto scales_on = [&](int64_t bytes) {
    return kb % bytes == 0 && (reinterpret_cast<uintptr_t>(a.a_scale) | reinterpret_cast<uintptr_t>(a.b_scale)) % static_cast<uintptr_t>(bytes) == 0;
  };
  const size_t padded = static_cast<size_t>(a.a_rows + experts * a.n) * ((kb + 15) / 16 * 16), unless_words = scales_on(4) ? 0 : padded;
  if (!scales_on(4) && rows <= 16 * experts) return {Form::FEW_ROWS, 0, 0, 0, 0};
  const int64_t low_panels = pieces(64, 128);
  if (low_panels < (each <= 10 ? 240 : 160)) {
    const bool two = each > 10;
    const int64_t streams = pieces(two ? 32 : 16, 32);
    const bool wide = two && streams >= 1024;
    return {Form::STREAM, two ? 2 : 1, wide ? 4 : 2, streams >= (two ? 512 : 768) ? 1 : streams >= 192 ? 2 : 4, unless_words};
  }
  if (each <= 48 || low_panels <= cus) return {Form::PANEL, 2, 0, 0, unless_words};
  if (pieces(128, 128) <= cus) return {Form::PANEL, 4, 0, 0, unless_words};
  if (dual_takes_mx(dual)) return {Form::DUAL, 0, 0, 0, kb % 4 == 0 ? 0 : padded};
  return {Form::TILES, 0, 0, 0, scales_on(16) ? 0 : padded};
}

}  // namespace
}  // namespace fluxmi

extern "C" size_t fluxmi_grouped_gemm_mx_workspace_bytes(const fluxmi_mx_gemm_args *args) {
  if (args == nullptr || args->nexperts < 1 || args->max_rows < 1 || args->n < 1 || args->k < 1 || args->a_rows < 0) return 0;
  return fluxmi::plan_of(*args, fluxmi::dual_params(*args), fluxmi::kPlanCus).workspace;
}

extern "C" int fluxmi_grouped_gemm_mx_launch_info(const fluxmi_mx_gemm_args *args, fluxmi_mx_launch_info *info) {
  using namespace fluxmi;
  FLUXMI_REQUIRE(args != nullptr && info != nullptr, FLUXMI_ERR_INVALID_ARG, "grouped_gemm_mx_launch_info: null args / info");
  *info = fluxmi_mx_launch_info{};
  const int rc = check_args(args);
  if (rc != FLUXMI_OK || args->max_rows == 0 || args->n == 0) return rc;
  const Plan plan = plan_of(*args, dual_params(*args), kPlanCus);
  switch (plan.form) {
    case Form::FEW_ROWS:
      *info = {FLUXMI_MX_FEW_ROWS, 16, kCols, kThreads / 64};
      break;
    case Form::STREAM:
      *info = {FLUXMI_MX_STREAM, 16 * plan.row_blocks, 16 * plan.col_blocks, plan.waves};
      break;
    case Form::PANEL:
      *info = {FLUXMI_MX_PANEL, 32 * plan.row_blocks, 128, 1};
      break;
    case Form::DUAL:
      *info = {FLUXMI_MX_DUAL, 256, 256, 1};
      break;
    case Form::TILES:
      *info = {FLUXMI_MX_TILES, 256, 256, 1};
      break;
  }
  return FLUXMI_OK;
}

extern "C" int fluxmi_grouped_gemm_mx(const fluxmi_mx_gemm_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace fluxmi;
  int rc = check_args(args);
  if (rc != FLUXMI_OK || args->max_rows == 0 || args->n == 0) return rc;
  GemmParams dual = dual_params(*args);
  const Plan plan = plan_of(*args, dual, kPlanCus);
  FLUXMI_REQUIRE(plan.workspace == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= plan.workspace), FLUXMI_ERR_WORKSPACE,
                 "grouped_gemm_mx: workspace of %zu bytes needed, %zu given", plan.workspace, workspace_bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
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
  p.scale_stride = p.kb;
  p.d_type = args->d_type == FLUXMI_ROWS_BF16 ? Row::BF16 : args->d_type == FLUXMI_ROWS_FP32 ? Row::F32 : Row::F16;
  if (plan.workspace > 0) {
    p.scale_stride = (p.kb + 15) / 16 * 16;
    const int64_t a_rows = p.a_rows, b_rows = int64_t{p.nexperts} * p.n, groups = (a_rows + b_rows) * (p.scale_stride / 16);
    const unsigned grid = static_cast<unsigned>(groups / kThreads < 8192 ? groups / kThreads + 1 : 8192);
    uint8_t *const padded = static_cast<uint8_t *>(workspace);
    hipLaunchKernelGGL(mx_pad_scales_kernel, dim3(grid), dim3(kThreads), 0, s, p.a_scale, a_rows, p.b_scale, b_rows, p.kb, p.scale_stride, padded);
    p.a_scale = padded;
    p.b_scale = padded + a_rows * p.scale_stride;
    dual.a_scale = reinterpret_cast<const float *>(p.a_scale);
    dual.b_scale = reinterpret_cast<const float *>(p.b_scale);
  }
  switch (plan.form) {
    case Form::STREAM:
      if (plan.col_blocks == 4) rc = launch_stream<2, 4, 1>(p, s);
      else if (plan.row_blocks == 2) rc = plan.waves == 1 ? launch_stream<2, 2, 1>(p, s) : plan.waves == 2 ? launch_stream<2, 2, 2>(p, s) : launch_stream<2, 2, 4>(p, s);
      else rc = plan.waves == 1 ? launch_stream<1, 2, 1>(p, s) : plan.waves == 2 ? launch_stream<1, 2, 2>(p, s) : launch_stream<1, 2, 4>(p, s);
      break;
    case Form::PANEL:
      rc = plan.row_blocks == 2 ? launch_panel<2>(p, s) : launch_panel<4>(p, s);
      break;
    case Form::DUAL: {
      // Up to four workgroups to a tile, which is cut in pieces when these still fit the card.
      const int64_t tiles = (int64_t{p.max_rows} / 256 + (p.nexperts < p.max_rows ? p.nexperts : p.max_rows)) * ((p.n + 255) / 256), cus = fluxmi_device_cu_count();
      rc = launch_grouped_gemm_dual_mx(dual, static_cast<int>(tiles * 4 < cus ? tiles * 4 : cus), s);
      break;
    }
    case Form::FEW_ROWS:
      rc = launch_few_rows(p, s);
      break;
    case Form::TILES:
      rc = launch_tiles<8, 4, 2, 4>(p, s);
      break;
  }
  if (rc != FLUXMI_OK) return rc;
  FLUXMI_HIP_CHECK(hipGetLastError());
  return FLUXMI_OK;
}
