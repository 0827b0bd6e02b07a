// Gradients of the grouped product (grouped_gemm_grad.hip has the formulas) by tiles of 256 x 256 of the result.
//
//  * Four waves, one to a SIMD, 128 x 128 to each: 256 sums in accumulation registers, two sets of fragments of 16 x 32 in vector registers.  A step
//    sums over 32 values: 64 MFMAs of 16 x 16 x 32 on one set, while the other is read from LDS for the next step and the step four further on is
//    requested.
//  * LDS holds four steps of both operands, 16 KiB each, filled by loads that go there directly.  An operand whose rows are what is summed over ("across": W,
//    X, and G for the weights' gradient) lies in rows of 256 columns, 512 bytes; 16 columns of a row (32 bytes) are at place s ^ f(row), f = row % 4 + 4 (row / 8 % 2), so
//    that the eight rows which half a wave reads together are on different banks.  G for the input's gradient lies in rows of 32 values, 64 bytes.
//  * A fragment of an "across" operand comes back through the transposing read, twice four rows of 16 columns.
//  * A step that is not whole is fetched as far as the sum goes, and the rest of it is cleared in LDS; rows and columns past the end of the result are not fetched: what
//    LDS held there reaches no result that is stored.
//  * A checkpoint's codes and scale bytes (WEIGHT_8BIT) are fetched like the rest, and each wave turns what it fetched to values of 16 bits two steps ahead, in LDS, beside the
//    MFMAs; the values are exact in the rows' type.
//  * One workgroup to a compute unit computes several tiles, in turns or (weights of several experts, four turns or more) from a queue to each XCD.  The next tile's first four steps are
//    requested before a tile's results go out, through a window in LDS and in whole lines.  The last turn's tiles are cut along the sum where that is cheaper, and joined in
//    the parts' order: results have the same bits in every launch.
//
// What bounds it on MI355X (us): large products the board's power, 8 experts 14336 x 4096, 16384 rows: input 1470, weights 1435, 1.31 to 1.34 PFLOP/s, MFMA 77 and 68 % busy at 1.6 to 1.8 GHz
// (zero operands reach 1.75 PFLOP/s).  Many small experts what lies between two tiles' sums, about 7 to each of 25 to 45, with MFMA 57 and 46 % busy: 64 skewed experts, 93000 rows, input
// 1408 x 2048 525, weights 1400 x 2040 to fp32 606 (1408 x 2048, whose rows begin on lines, 560).  Weights from 8 bits, 32 experts 2048 x 7168 to fp32, 32768 rows: 1060, the conversion a
// tenth of it, MFMA 39 % busy.  Few rows the read of W: 74 rows on 8 experts 14336 x 4096 167, 5.7 TB/s.  Results that are added to what is there wait for it store by store: the same
// weights to bf16 2020, from 8 bits to fp32 1970, 1400 x 2040 to fp32 920.
// Also built: without the window 1594 for weights (neighbouring lanes store to different rows); row blocks left out one by one in tiles of any height + 7 to 10 %; small and large
// experts in turn from the queues 668 where the largest come first 631.
#include "grouped_gemm_grad_tiles.hpp"

#include <type_traits>
#include <utility>

namespace fluxmi {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 256;
constexpr int kStep = 32;
constexpr int kSlot = 16384;           // bytes of one operand's step
constexpr int kSlots = 4;
constexpr int kCodeSlot = 8192, kScaleSlot = 1024;  // WEIGHT_8BIT: a step's codes, and its scales in words
// The columns' operand in kSlots slots (WEIGHT_8BIT: two, of converted values), the rows' operand in kSlots, then codes and scales.
constexpr int rows_at(Grad g) { return (g == Grad::WEIGHT_8BIT ? 2 : kSlots) * kSlot; }
constexpr int codes_at() { return rows_at(Grad::WEIGHT_8BIT) + kSlots * kSlot; }
constexpr int scales_at() { return codes_at() + kSlots * kCodeSlot; }
// Behind them a window of each wave, through which results go out, and the experts' tables: where their rows end, and (INPUT) their tiles or (otherwise) the order
// they are taken in.
constexpr int kWindow = 2048;
constexpr int windows_at(Grad g) { return g == Grad::WEIGHT_8BIT ? scales_at() + kSlots * kScaleSlot : rows_at(g) + kSlots * kSlot; }
constexpr int tables_at(Grad g) { return windows_at(g) + kThreads / 64 * kWindow; }
constexpr int lds_bytes(Grad g) { return tables_at(g) + 2 * 4 * kMaxExperts + 32; }

// Division of numbers below 2^24 by one that the host knows.
struct Divisor {
  uint32_t by, factor, shift;
};
Divisor divisor(int64_t by) {
  Divisor d{static_cast<uint32_t>(by), 0, 24};
  while ((int64_t{1} << (d.shift - 24)) < by) ++d.shift;
  d.factor = static_cast<uint32_t>(((uint64_t{1} << d.shift) + by - 1) / by);
  return d;
}
__device__ __forceinline__ int divide(int x, Divisor d) { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(x)) * d.factor) >> d.shift); }

// Queues: eight of them, one to an XCD, a counter each (a line apart) of the tiles that were fetched from it beyond every workgroup's first; then the experts, those with most
// rows first.
constexpr int kQueueLine = 32, kQueueExperts = 8 * kQueueLine;
constexpr size_t kQueueBytes = (kQueueExperts + kMaxExperts) * sizeof(int32_t);

// Every workgroup computes one tile in a turn.  Where the last turn's tiles are at most half as many as workgroups, their sums may be cut into parts, which a second
// kernel joins: tiles [0, whole), then `parts` of each of `cut` tiles.  In 1/128 us, a step takes 64, and parts cost their way through memory (15 for a tile of 256 rows,
// written and read) and the second kernel (512): the cheapest number of them is taken.  us, 8 experts, none / cut as here: input 14336 x 4096, 16384 rows 1564 / 1470, 74 rows 240 / 202.
constexpr int kMostParts = 16;
struct Turns {
  int whole, cut, parts;
};
struct Cutting {
  int32_t steps, height;  // of a tile's sum, and its rows, on average
};
__host__ __device__ inline Turns turns_of(int tiles, int grid, Cutting c) {
  const int whole = tiles / grid * grid, cut = tiles - whole, each = cut * (c.height * 15) / kTile;
  int parts = 1, best = c.steps * 64 - 512;
  auto consider = [&](auto P) {
    constexpr int p = decltype(P)::value;
    const int cost = c.steps * 64 / p + each * p;
    if (cut * p <= grid && cost < best) best = cost, parts = p;
  };
  consider(std::integral_constant<int, 2>{});
  consider(std::integral_constant<int, 3>{});
  consider(std::integral_constant<int, 4>{});
  consider(std::integral_constant<int, 6>{});
  consider(std::integral_constant<int, 8>{});
  consider(std::integral_constant<int, 12>{});
  consider(std::integral_constant<int, kMostParts>{});
  if (cut == 0 || parts == 1) return {tiles, 0, 1};
  return {whole, cut, parts};
}

struct TileArgs {
  GradArgs a;
  Cutting cutting;
  int32_t grid;           // workgroups, a multiple of 8
  int32_t turns;          // tiles that a workgroup computes at most
  Divisor per_expert, per_group;  // an expert's tiles; those of eight along the result's rows
  int32_t *queue;         // NULL: tiles are dealt in turns; otherwise workgroups fetch them: counters, then the experts by their rows
};

#if defined(__HIP_DEVICE_COMPILE__)

#define FLUXMI_VMCNT(vm) __builtin_amdgcn_s_waitcnt(((vm)&15) | (((vm) >> 4) << 14) | (7 << 4) | (15 << 8))
#define FLUXMI_LGKM0() __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8))

typedef const __attribute__((address_space(3))) u32x4 *LdsFrag;

template <class F, int... I>
__device__ __forceinline__ void static_for_seq(F &f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int END, class F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for_seq(f, std::make_integer_sequence<int, END>{});
}

// Pinned to the accumulation registers: given the builtin, the compiler spreads the sums over both files and moves them about.  FIRST: a sum begins.
template <bool F16, bool FIRST>
__device__ __forceinline__ void mfma(f32x4 &acc, const u32x4 &a, const u32x4 &b) {
  if constexpr (F16) {
    if constexpr (FIRST) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "=a"(acc) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
  } else {
    if constexpr (FIRST) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=a"(acc) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
  }
}

// Block `block` of a wave's rows, unless the tile has no more than `blocks` of them.  One statement with its branch: as a branch that the compiler sees, the sums' registers
// would be moved about.
template <bool F16, bool FIRST>
__device__ __forceinline__ void row_block(f32x4 (&acc)[8], const u32x4 (&c)[8], const u32x4 &r, int block, int blocks) {
#define FLUXMI_ROW_BLOCK(MFMA, D)                                                                                                                   \
  asm volatile("s_cmp_gt_i32 %17, %18\n\ts_cbranch_scc0 .Lrow_block%=\n\t" MFMA " %0, %8, %16, " D("%0") "\n\t" MFMA " %1, %9, %16, " D("%1") "\n\t"      \
               MFMA " %2, %10, %16, " D("%2") "\n\t" MFMA " %3, %11, %16, " D("%3") "\n\t" MFMA " %4, %12, %16, " D("%4") "\n\t"                       \
               MFMA " %5, %13, %16, " D("%5") "\n\t" MFMA " %6, %14, %16, " D("%6") "\n\t" MFMA " %7, %15, %16, " D("%7") "\n.Lrow_block%=:"          \
               : "+a"(acc[0]), "+a"(acc[1]), "+a"(acc[2]), "+a"(acc[3]), "+a"(acc[4]), "+a"(acc[5]), "+a"(acc[6]), "+a"(acc[7])                       \
               : "v"(c[0]), "v"(c[1]), "v"(c[2]), "v"(c[3]), "v"(c[4]), "v"(c[5]), "v"(c[6]), "v"(c[7]), "v"(r), "s"(blocks), "i"(block)              \
               : "scc")
#define FLUXMI_SAME(x) x
#define FLUXMI_ZERO(x) "0"
  if constexpr (F16 && FIRST) FLUXMI_ROW_BLOCK("v_mfma_f32_16x16x32_f16", FLUXMI_ZERO);
  else if constexpr (F16) FLUXMI_ROW_BLOCK("v_mfma_f32_16x16x32_f16", FLUXMI_SAME);
  else if constexpr (FIRST) FLUXMI_ROW_BLOCK("v_mfma_f32_16x16x32_bf16", FLUXMI_ZERO);
  else FLUXMI_ROW_BLOCK("v_mfma_f32_16x16x32_bf16", FLUXMI_SAME);
#undef FLUXMI_ROW_BLOCK
#undef FLUXMI_SAME
#undef FLUXMI_ZERO
}

// A sum's block, read where it is used: the compiler would copy all of them to vector registers ahead of the branches of the stores.
__device__ __forceinline__ f32x4 sums_of(const f32x4 &acc) {
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(acc[i]));
    v[i] = x;
  }
  return v;
}

// Sixteen bytes (BYTE: one, to a word) of each lane to LDS, from base + AT on.  Not the builtin: with it the compiler lets every LDS read wait for all loads.  The load comes five wait
// states after the statement's start: what a scalar register needs that a vector instruction wrote (v_readlane, with which the compiler brings back spilled ones: words of the buffer
// among them), and it does not look into asm for that.
template <bool BYTE, int AT>
__device__ __forceinline__ void load_to_lds(uint32_t base, uint32_t off, __amdgpu_buffer_rsrc_t rsrc) {
  if constexpr (BYTE) asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 3\n\tbuffer_load_ubyte %2, %3, 0 offen lds" : : "s"(base), "i"(AT), "v"(off), "s"(rsrc) : "memory", "scc");
  else asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 3\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" : : "s"(base), "i"(AT), "v"(off), "s"(rsrc) : "memory", "scc");
}
// The same behind two MFMAs, beside which the wait states cost little.  us, MFMA and load as statements without a wait / this / MFMA and load apart, the load with its wait: weights
// 14336 x 4096, 16384 rows 1432 / 1435 / 1455 to 1480; 2048 x 7168 from 8 bits, 32768 rows 1046 / 1059 / 1063; input 1466 / 1467 / 1476 to 1488.
template <bool F16, bool FIRST, bool BYTE, int AT>
__device__ __forceinline__ void mfma_and_load(f32x4 &acc0, f32x4 &acc1, const u32x4 &c0, const u32x4 &c1, const u32x4 &r, uint32_t base, uint32_t off, __amdgpu_buffer_rsrc_t rsrc) {
#define FLUXMI_MFMA_AND_LOAD(MFMA, D, LOAD)                                                                                                         \
  asm volatile("s_add_u32 m0, %5, %6\n\t" MFMA " %0, %2, %4, " D("%0") "\n\ts_nop 1\n\t" MFMA " %1, %3, %4, " D("%1") "\n\t" LOAD                 \
               " %7, %8, 0 offen lds"                                                                                                               \
               : "+a"(acc0), "+a"(acc1) : "v"(c0), "v"(c1), "v"(r), "s"(base), "i"(AT), "v"(off), "s"(rsrc) : "memory", "scc")
#define FLUXMI_SAME(x) x
#define FLUXMI_ZERO(x) "0"
#define FLUXMI_OF_SIZE(MFMA, D)                                             \
  do {                                                                      \
    if constexpr (BYTE) FLUXMI_MFMA_AND_LOAD(MFMA, D, "buffer_load_ubyte"); \
    else FLUXMI_MFMA_AND_LOAD(MFMA, D, "buffer_load_dwordx4");              \
  } while (0)
  if constexpr (F16 && FIRST) FLUXMI_OF_SIZE("v_mfma_f32_16x16x32_f16", FLUXMI_ZERO);
  else if constexpr (F16) FLUXMI_OF_SIZE("v_mfma_f32_16x16x32_f16", FLUXMI_SAME);
  else if constexpr (FIRST) FLUXMI_OF_SIZE("v_mfma_f32_16x16x32_bf16", FLUXMI_ZERO);
  else FLUXMI_OF_SIZE("v_mfma_f32_16x16x32_bf16", FLUXMI_SAME);
#undef FLUXMI_MFMA_AND_LOAD
#undef FLUXMI_OF_SIZE
#undef FLUXMI_SAME
#undef FLUXMI_ZERO
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7fc00000u : byte << 23)); }

// Two of sixteen codes of one block to values of 16 bits.
template <bool F16>
__device__ __forceinline__ void convert_pair(const u32x4 codes, float scale, u32x4 (&v)[2], int pair) {
  const int w = pair >> 1;
  uint32_t x;
  if constexpr (F16) {
    x = pair & 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[w], scale, true))
                 : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[w], scale, false));
  } else {
    x = pair & 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w], scale, true))
                 : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w], scale, false));
  }
  v[pair >> 2][pair & 3] = x;
}

// A tile of the result and where its operands begin.
struct Tile {
  int e, row0, rows, col0, cols;  // row0: column of grad for weights, otherwise 0; rows = 0: there is no such tile
  int part, slot;  // part < 0: the whole sum; otherwise its sums go to place `slot` of the parts'
  int begin;    // INPUT: first of the columns of G that it sums over
  int sum_over;
  int first;  // of the rows that it sums over (INPUT: reads)
  int64_t out_row0;
};

// The lane, opaque to the compiler: what is computed from it is not kept in registers through the loops.
__device__ __forceinline__ int fresh_lane() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l;
}

#endif  // __HIP_DEVICE_COMPILE__

// FEW: most tiles have far fewer rows than 256 (INPUT).
template <bool F16, Grad G, bool FEW>
__global__ __launch_bounds__(kThreads, 1) void grad_tile_kernel(const TileArgs args) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool INPUT = G == Grad::INPUT, EIGHT = G == Grad::WEIGHT_8BIT;
  const GradArgs &a = args.a;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)smem));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave >> 1, wc = wave & 1;
  const int tiles_k = (a.k + kTile - 1) / kTile, tiles_n = (a.n + kTile - 1) / kTile;
  const int64_t rpitch = static_cast<int64_t>(a.n) * 2, cpitch = static_cast<int64_t>(a.k) * (EIGHT ? 1 : 2);
  const int blocks = (a.k + 31) / 32;

  // ---- the experts' rows and tiles, in LDS ------------------------------------------------------------------------
  typedef __attribute__((address_space(3))) int *LdsInt;
  const LdsInt row_ends = (LdsInt)(uintptr_t)(lds0 + tables_at(G)), tile_ends = row_ends + kMaxExperts, order = tile_ends, mail = tile_ends + kMaxExperts;
  int all_rows = 0, row_tiles = 0;
  for (int e0 = 0; e0 < a.nexperts; e0 += 64) {  // (the same from every wave)
    const ExpertRows x = rows_of_lane(a, e0, all_rows);
    row_ends[e0 + lane] = x.end;
    if (!INPUT && args.queue != nullptr) order[e0 + lane] = e0 + lane < a.nexperts ? args.queue[kQueueExperts + e0 + lane] : 0;
    if constexpr (INPUT) {
      const int end = row_tiles + wave_inclusive_scan((x.end - x.begin + kTile - 1) / kTile);
      tile_ends[e0 + lane] = end;
      row_tiles = __builtin_amdgcn_readlane(end, 63);
    }
  }
  __syncthreads();
  const int expert_tiles = row_tiles;
  if constexpr (INPUT) row_tiles += (a.rows - all_rows + kTile - 1) / kTile;  // the rows that belong to no expert
  const Turns turns = turns_of((INPUT ? row_tiles : a.nexperts * tiles_n) * tiles_k, args.grid, args.cutting);

  // Tile number `item`.  An expert's (INPUT: all) tiles lie in groups of eight along the result's rows, walked column by column.
  auto describe = [&](int item, int part) {
    Tile t{};
    t.part = part;
    const int e = INPUT ? 0 : divide(item, args.per_expert), local = INPUT ? item : item - e * static_cast<int>(args.per_expert.by);
    const int group = divide(local, args.per_group), in_group = local - group * static_cast<int>(args.per_group.by);
    const int high = (INPUT ? row_tiles : tiles_n) - group * 8, height = high < 8 ? high : 8;
    const int kt = height == 8 ? in_group >> 3 : in_group / height, rt = group * 8 + in_group - kt * height;
    t.col0 = kt * kTile;
    t.cols = a.k - t.col0 < kTile ? a.k - t.col0 : kTile;
    if constexpr (INPUT) {
      t.e = a.nexperts;
      int begin = all_rows + (rt - expert_tiles) * kTile, end = a.rows;
      if (rt < expert_tiles) {
        for (int e0 = 0;; e0 += 64) {
          const int ends = tile_ends[e0 + lane];
          const uint64_t hit = __ballot(e0 + lane < a.nexperts && rt < ends);
          if (hit == 0) continue;
          const int src = __ffsll(static_cast<unsigned long long>(hit)) - 1;
          t.e = e0 + src;
          const int first = t.e > 0 ? __builtin_amdgcn_readfirstlane(row_ends[t.e - 1]) : 0;
          end = __builtin_amdgcn_readfirstlane(row_ends[t.e]);
          begin = first + (rt - (__builtin_amdgcn_readlane(ends, src) - (end - first + kTile - 1) / kTile)) * kTile;
          break;
        }
      }
      t.rows = end - begin < kTile ? end - begin : kTile;
      t.out_row0 = t.first = begin;
      t.sum_over = t.e < a.nexperts ? a.n : 0;
    } else {
      t.e = args.queue != nullptr ? __builtin_amdgcn_readfirstlane(order[e]) : e;
      t.row0 = rt * kTile;
      t.rows = a.n - t.row0 < kTile ? a.n - t.row0 : kTile;
      t.out_row0 = static_cast<int64_t>(t.e) * a.n + t.row0;
      t.first = t.e > 0 ? __builtin_amdgcn_readfirstlane(row_ends[t.e - 1]) : 0;
      t.sum_over = __builtin_amdgcn_readfirstlane(row_ends[t.e]) - t.first;
    }
    if (t.part >= 0) {
      const int all = (t.sum_over + kStep - 1) / kStep, from = all * t.part / turns.parts * kStep, to = all * (t.part + 1) / turns.parts * kStep;
      t.sum_over = (to < t.sum_over ? to : t.sum_over) - from;
      if constexpr (INPUT) t.begin = from;
      else t.first += from;
    }
    return t;
  };
  // This workgroup's tile of a turn.  Workgroups are dealt to the eight XCDs in turn; those on one XCD take neighbouring tiles.
  const int home = blockIdx.x & 7, place = blockIdx.x >> 3;
  auto tile_of_turn = [&](int turn) {
    int item = turn * args.grid + home * (args.grid >> 3) + place;
    if (item < turns.whole) return describe(item, -1);
    item -= turns.whole;
    if (item >= turns.cut * turns.parts) return Tile{};
    const int part = item / turns.cut;
    Tile t = describe(turns.whole + item - part * turns.cut, part);
    t.slot = item;
    return t;
  };
  // Tile at a place of a queue: 32 neighbouring tiles (as many as an XCD has compute units) are dealt to each queue in turn, so that those that an XCD has at a time share
  // their rows of G and X.  us by 8 / 16 / 32 / 64: 64 skewed experts 1400 x 2040 to fp32 628 / 607 / 613 / 779 (the largest expert's tiles in one queue), to fp16 540 / 524 / 514 /
  // 673; 128 of them 792 / 762 / 750 / 812; 8 experts 14336 x 4096, 16384 rows 1449 / 1452 / 1445 / 1441.
  auto tile_of_queue = [&](int queue, int at) {
    const int item = ((at & ~31) + queue * 4) * 8 + (at & 31);
    return item < a.nexperts * tiles_n * tiles_k ? describe(item, -1) : Tile{};
  };

  // ---- fills: four instructions of a wave to either operand's step ------------------------------------------------
  // Across: an instruction fills two rows, lane l place l % 32 (of 16 bytes) of row l / 32; along: 16 rows, lane l place l % 4 of row l / 4.
  // Codes: four rows, lane l chunk l % 16 (of 16 columns) of row l / 16; scales: the eight rows whose codes this wave fetches, a word to each byte.
  constexpr int kColFills = EIGHT ? 3 : 4, kFills = kColFills + 4;
  uint32_t coff[4], roff[4];
  constexpr uint32_t kNowhere = 0xfffffff0u;  // past every buffer's end: rows and columns that the tile does not have are not fetched
  // The step that is requested next: where it begins, and how much of the sum (INPUT: of the tile's rows of G, in bytes) is left there.
  const uint8_t *rnext = nullptr, *cnext = nullptr, *snext = nullptr;
  int left = 0, rbytes = 0;
  int row_blocks = 0;
  int steps = 0, rest = 0;  // rest: values of the last step
  auto begin_tile = [&](const Tile &t) {
    const int lane = fresh_lane();
    left = __builtin_amdgcn_readfirstlane(t.sum_over);
    steps = left > 0 ? (left + kStep - 1) / kStep : 1;  // (a sum of nothing is a step that is cleared)
    rest = left - (steps - 1) * kStep;
    row_blocks = (__builtin_amdgcn_readfirstlane(t.rows) - wr * 16 + 31) / 32;
    const int64_t first = __builtin_amdgcn_readfirstlane(t.first);
    rnext = a.grad + first * rpitch;
    if constexpr (INPUT) {
      const int e = __builtin_amdgcn_readfirstlane(t.e), begin = __builtin_amdgcn_readfirstlane(t.begin);
      cnext = a.other + (static_cast<int64_t>(e < a.nexperts ? e : 0) * a.n + begin) * cpitch;
      rnext += begin * 2;
      rbytes = __builtin_amdgcn_readfirstlane(t.rows) * static_cast<int>(rpitch) - begin * 2;
    } else {
      cnext = a.other + first * cpitch;
    }
    if constexpr (EIGHT) snext = a.scale + first * blocks;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = wave * 8 + i * 2 + (lane >> 5), f = (row & 3) | ((row >> 1) & 4);
      const int col = (((lane & 31) >> 1) ^ f) * 16 + (lane & 1) * 8;
      if constexpr (EIGHT) {
        const int c = (lane & 15) * 16, b = lane & 7;
        if (i < 2) coff[i] = c < t.cols ? static_cast<uint32_t>((wave * 8 + i * 4 + (lane >> 4)) * cpitch) + t.col0 + c : kNowhere;
        else if (i == 2) coff[i] = static_cast<uint32_t>((wave * 8 + (lane >> 3)) * blocks) + t.col0 / 32 + (b * 32 < t.cols ? b : 0);
      } else {
        coff[i] = col < t.cols ? static_cast<uint32_t>(row * cpitch) + (t.col0 + col) * 2u : kNowhere;
      }
      if constexpr (INPUT) {
        const int r = wave * 64 + i * 16 + (lane >> 2), c = (lane & 3) ^ ((r >> 1) & 3);
        roff[i] = r < t.rows ? static_cast<uint32_t>(r * rpitch) + c * 16u : kNowhere;
      } else {
        roff[i] = col < t.rows ? static_cast<uint32_t>(row * rpitch) + (t.row0 + col) * 2u : kNowhere;
      }
    }
  };
  const int64_t cstep = kStep * cpitch, rstep = INPUT ? kStep * 2 : kStep * rpitch, sstep = static_cast<int64_t>(kStep) * blocks;
  __amdgpu_buffer_rsrc_t crsrc, rrsrc, srsrc;
  // The buffers of the step that is requested next; what lies behind their end is not fetched.
  auto next_buffers = [&]() {
    auto buffer = [](const uint8_t *p, int bytes) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, bytes, 0x00020000); };
    int rows = left < kStep ? left : kStep;
    asm("" : "+s"(rows));  // (as one clamp it would be computed in vector registers)
    rows = rows < 0 ? 0 : rows;
    crsrc = buffer(cnext, rows * static_cast<int>(cpitch));
    cnext += cstep;
    if constexpr (EIGHT) {
      srsrc = buffer(snext, rows * blocks);
      snext += sstep;
    }
    rrsrc = buffer(rnext, INPUT ? (rbytes < 0 || rows == 0 ? 0 : rbytes) : rows * static_cast<int>(rpitch));
    rnext += rstep;
    if constexpr (INPUT) rbytes -= kStep * 2;
    left -= kStep;
  };
  const uint32_t cdst = lds0 + wave * 4096, rdst = cdst + rows_at(G), codes = lds0 + codes_at() + wave * 2048, scales = lds0 + scales_at() + wave * 256;
  using std::integral_constant;

  f32x4 acc[8][8];  // [row block][column block]

  // ---- fragment addresses -------------------------------------------------------------------------------------------
  uint32_t cfrag[8], rfrag[8];
  {
    const int g = lane >> 4, i = lane & 15, t = 8 * g + (i >> 2), f = (t & 3) | ((t >> 1) & 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cfrag[j] = lds0 + t * 512 + ((wc * 8 + j) ^ f) * 32 + (i & 3) * 8;
      if constexpr (INPUT) rfrag[j] = lds0 + rows_at(G) + (wr * 16 + i) * 64 + (g ^ ((i >> 1) & 3)) * 16;
      else rfrag[j] = lds0 + rows_at(G) + t * 512 + ((2 * j + wr) ^ f) * 32 + (i & 3) * 8;
    }
  }
  u32x4 ca[8], ra[8], cb[8], rb[8];
  // Read R of the 32 (INPUT: 24) that a step's fragments take, from slot SLOT.
  constexpr int kReads = INPUT ? 24 : 32;
  auto read_one = [&](auto SLOT, auto R, u32x4(&cf)[8], u32x4(&rf)[8]) {
    constexpr int slot = decltype(SLOT)::value, r = decltype(R)::value;
    if constexpr (r < 16) {
      const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(uintptr_t)(cfrag[r / 2] + (EIGHT ? slot % 2 : slot) * kSlot + (r & 1) * 2048)));
      cf[r / 2][(r & 1) * 2] = v[0];
      cf[r / 2][(r & 1) * 2 + 1] = v[1];
    } else if constexpr (INPUT) {
      rf[r - 16] = *(LdsFrag)(uintptr_t)(rfrag[0] + slot * kSlot + (r - 16) * 2048);
    } else {
      constexpr int q = r - 16;
      const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(uintptr_t)(rfrag[q / 2] + slot * kSlot + (q & 1) * 2048)));
      rf[q / 2][(q & 1) * 2] = v[0];
      rf[q / 2][(q & 1) * 2 + 1] = v[1];
    }
  };

  // WEIGHT_8BIT: what this wave fetched of a step becomes values in the slot of its parity.  In three parts: read, convert, write.
  u32x4 code[2], value[2][2];
  uint32_t scale_byte[2];
  const uint32_t scale_at = scales + ((lane >> 4) * 8 + ((lane & 15) >> 1)) * 4;
  uint32_t value_at[2];
  if constexpr (EIGHT) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = wave * 8 + i * 4 + (lane >> 4), f = (t & 3) | ((t >> 1) & 4);
      value_at[i] = lds0 + t * 512 + ((lane & 15) ^ f) * 32;
    }
  }
  float scale_bits[2];
  auto read_codes = [&](auto SLOT, int i) {
    constexpr int slot = decltype(SLOT)::value;
    code[i] = *(LdsFrag)(uintptr_t)(codes + lane * 16 + slot * kCodeSlot + i * 1024);
    scale_byte[i] = *(const __attribute__((address_space(3))) uint32_t *)(uintptr_t)(scale_at + slot * kScaleSlot + i * 128);
  };
  auto write_values = [&](auto SLOT, int i, int h) {
    constexpr int slot = decltype(SLOT)::value;
    *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(value_at[i] + (slot % 2) * kSlot + h * 16) = value[i][h];
  };

  // Fill Q of the step in slot SLOT, by `load`(bytes, where: base and constant, offsets, buffer).  (Base and constant apart: 28 addresses would take as many registers.)
  auto fill_by = [&](auto SLOT, auto Q, auto &&load) {
    constexpr int slot = decltype(SLOT)::value, q = decltype(Q)::value, r = q - kColFills;
    if constexpr (r >= 0) load(std::false_type{}, rdst, integral_constant<int, slot * kSlot + (r < 0 ? 0 : r) * 1024>{}, roff[r < 0 ? 0 : r], rrsrc);
    else if constexpr (EIGHT && q == 2) load(std::true_type{}, scales, integral_constant<int, slot * kScaleSlot>{}, coff[2], srsrc);
    else if constexpr (EIGHT) load(std::false_type{}, codes, integral_constant<int, slot * kCodeSlot + q * 1024>{}, coff[q < 4 ? q : 0], crsrc);
    else load(std::false_type{}, cdst, integral_constant<int, slot * kSlot + q * 1024>{}, coff[q < 4 ? q : 0], crsrc);
  };
  auto fill = [&](auto SLOT, auto Q) {
    fill_by(SLOT, Q, [&](auto BYTE, uint32_t base, auto AT, uint32_t off, __amdgpu_buffer_rsrc_t rsrc) { load_to_lds<decltype(BYTE)::value, decltype(AT)::value>(base, off, rsrc); });
  };
  auto first_fills = [&]() {
    static_for<kSlots>([&](auto S) {
      next_buffers();
      static_for<kFills>([&](auto Q) { fill(S, Q); });
    });
    next_buffers();
  };

  // Clears what this wave fetched of a step that is not whole, behind its `rest` values.  (Lanes with nothing to clear write to a place of no use: a branch among the
  // lanes would cost the sums their registers.)
  const uint32_t nowhere = lds0 + lds_bytes(G) - 16;
  auto clear = [&](uint32_t at, bool there) { *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(there ? nowhere : at) = u32x4{0u, 0u, 0u, 0u}; };
  auto clear_columns = [&](int s) {
    const int lane = fresh_lane(), slot = s & (kSlots - 1);
    if constexpr (EIGHT) {
      for (int i = 0; i < 2; ++i) clear(codes + slot * kCodeSlot + i * 1024 + lane * 16, wave * 8 + i * 4 + (lane >> 4) < rest);
      *(__attribute__((address_space(3))) uint32_t *)(uintptr_t)(wave * 8 + (lane >> 3) < rest ? nowhere : scales + slot * kScaleSlot + lane * 4) = 0;
    } else {
      for (int i = 0; i < 4; ++i) clear(cdst + slot * kSlot + i * 1024 + lane * 16, wave * 8 + i * 2 + (lane >> 5) < rest);
    }
  };
  auto clear_rows = [&](int s) {
    const int lane = fresh_lane(), slot = s & (kSlots - 1);
    for (int i = 0; i < 4; ++i) {
      const int r = wave * 64 + i * 16 + (lane >> 2);
      clear(rdst + slot * kSlot + i * 1024 + lane * 16, INPUT ? ((lane & 3) ^ ((r >> 1) & 3)) * 8 < rest : wave * 8 + i * 2 + (lane >> 5) < rest);
    }
  };

  // What a step waits for: the next one's rows and columns; WEIGHT_8BIT: that one's rows and the codes of the one after it.
  constexpr int kOpen = EIGHT ? kFills + 4 : 2 * kFills;
  // Loads and stores leave the counter in their order, also when the loads go to LDS from cold memory and a single store to the caches comes after them (measured: 3 G
  // words behind 1 to 96 stores, none missing).  A tile's first fills are requested before the stores of the tile before it, so that the first kFresh steps need not wait
  // for those: kStores of them for 16 bits; twice as many for 32 bits, which with the fills are more than the counter holds: all fills are in before the first step.  (With queues the
  // first wave waits for all of them before its first step: see where it asks for the next tile.)
  constexpr int kFresh = EIGHT ? 2 : 3, kStores = 32, kMostCounted = 62;
  static_assert(kOpen + kFills + kStores <= kMostCounted && 2 * kStores >= kMostCounted, "waits that the counter holds");
  int behind = 0;  // stores behind the first fills, times kStores
  auto wait_step = [&](auto U, int s) {
    bool waited = false;
    if constexpr (decltype(U)::value < kFresh) {
      if (s == decltype(U)::value && behind != 0) {
        if (behind == 1) FLUXMI_VMCNT(kOpen + kStores);
        waited = true;
      }
    }
    if (!waited) FLUXMI_VMCNT(kOpen);
    if (s + 3 >= steps && rest < kStep) {
      if (s + 2 == steps) {
        clear_rows(s + 1);
        if (!EIGHT) clear_columns(s + 1);
      } else if (EIGHT && s + 3 == steps) {
        clear_columns(s + 2);
      }
      FLUXMI_LGKM0();
    }
  };

  // The part of a step's conversion that stands beside MFMA t of 64.
  auto conversion = [&](auto U, auto T) {
    constexpr int u = decltype(U)::value, t = decltype(T)::value;
    constexpr integral_constant<int, (u + 2) % kSlots> slot{};
    if constexpr (!EIGHT) return;
    else if constexpr (t == 1 || t == 3) read_codes(slot, t / 2);
    else if constexpr (t == 15 || t == 37) scale_bits[t / 37] = scale_of(scale_byte[t / 37]);
    else if constexpr (t >= 17 && t < 33 && t % 2 == 1) convert_pair<F16>(code[0], scale_bits[0], value[0], (t - 17) / 2);
    else if constexpr (t >= 39 && t < 55 && t % 2 == 1) convert_pair<F16>(code[1], scale_bits[1], value[1], (t - 39) / 2);
    else if constexpr (t == 33 || t == 35) write_values(slot, 0, (t - 33) / 2);
    else if constexpr (t == 55 || t == 57) write_values(slot, 1, (t - 55) / 2);
  };
  // Step s, in slot U = s % 4: its fragments are in (cf, rf), those of the next go to (cn, rn), and its slot is filled with the step four further on.
  auto step = [&](auto U, auto FIRST, int s, u32x4(&cf)[8], u32x4(&rf)[8], u32x4(&cn)[8], u32x4(&rn)[8]) {
    constexpr int u = decltype(U)::value;
    wait_step(U, s);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (FEW) {
      // (the reads and fills of eight MFMAs stand together before them, which costs whole tiles 7 to 10 %)
      static_for<8>([&](auto I) {
        constexpr int i = decltype(I)::value;
        static_for<kReads / 8>([&](auto R) { read_one(integral_constant<int, (u + 1) % kSlots>{}, integral_constant<int, i * (kReads / 8) + decltype(R)::value>{}, cn, rn); });
        if constexpr (i < kFills) fill(U, I);
        if constexpr (i == 7) next_buffers();
        __builtin_amdgcn_sched_barrier(0);
        row_block<F16, decltype(FIRST)::value>(acc[i], cf, rf[i], i, row_blocks);
        __builtin_amdgcn_sched_barrier(0);
      });
    } else static_for<64>([&](auto T) {
      constexpr int t = decltype(T)::value, q = t / 8;
      conversion(U, T);
      if constexpr (t < 2 * kReads && t % 2 == 0) read_one(integral_constant<int, (u + 1) % kSlots>{}, integral_constant<int, t / 2>{}, cn, rn);
      if constexpr (t == 62) next_buffers();
      if constexpr (t % 8 == 4 && q < kFills) {  // (MFMAs t and t + 1)
        fill_by(U, integral_constant<int, q>{}, [&](auto BYTE, uint32_t base, auto AT, uint32_t off, __amdgpu_buffer_rsrc_t rsrc) {
          mfma_and_load<F16, decltype(FIRST)::value, decltype(BYTE)::value, decltype(AT)::value>(acc[q][4], acc[q][5], cf[4], cf[5], rf[q], base, off, rsrc);
        });
      } else if constexpr (t % 8 != 5 || q >= kFills) {
        mfma<F16, decltype(FIRST)::value>(acc[q][t % 8], cf[t % 8], rf[q]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    FLUXMI_LGKM0();
    __builtin_amdgcn_sched_barrier(0);
  };

  Tile tile = !INPUT && args.queue != nullptr ? tile_of_queue(home, place) : tile_of_turn(0);
  int turn = 1;
  if (tile.rows == 0) return;
  begin_tile(tile);
  first_fills();
  for (;;) {
    if constexpr (EIGHT) {
      if (behind == 0) FLUXMI_VMCNT(2 * kFills);
      else if (behind == 1) FLUXMI_VMCNT(2 * kFills + kStores);
      else FLUXMI_VMCNT(kMostCounted);
      if (rest < kStep && steps <= 2) clear_columns(steps - 1), FLUXMI_LGKM0();
      static_for<2>([&](auto S) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          read_codes(S, i);
          const float scale = scale_of(scale_byte[i]);
#pragma unroll
          for (int pair = 0; pair < 8; ++pair) convert_pair<F16>(code[i], scale, value[i], pair);
          write_values(S, i, 0), write_values(S, i, 1);
        }
      });
    } else {
      if (behind == 0) FLUXMI_VMCNT(3 * kFills);
      else if (behind == 1) FLUXMI_VMCNT(3 * kFills + kStores);
      else FLUXMI_VMCNT(kMostCounted);
      if (rest < kStep && steps == 1) clear_columns(0);
    }
    if (rest < kStep && steps == 1) clear_rows(0);
    FLUXMI_LGKM0();
    __builtin_amdgcn_s_barrier();
    // The next tile's number, which is looked at when this one's sums are done.  The compiler waits for it here, though, and with it for what the first wave has requested before: this
    // tile's first fills and the last tile's stores; the other waves wait for it at the first step's barrier.
    int fetched = 0;
    if (!INPUT && args.queue != nullptr && threadIdx.x == 0) fetched = atomicAdd(args.queue + home * kQueueLine, 1);
    static_for<kReads>([&](auto R) { read_one(integral_constant<int, 0>{}, R, ca, ra); });
    FLUXMI_LGKM0();
    step(integral_constant<int, 0>{}, std::true_type{}, 0, ca, ra, cb, rb);
    int s = 1;
    for (; s + 4 <= steps; s += 4) {
      step(integral_constant<int, 1>{}, std::false_type{}, s, cb, rb, ca, ra);
      step(integral_constant<int, 2>{}, std::false_type{}, s + 1, ca, ra, cb, rb);
      step(integral_constant<int, 3>{}, std::false_type{}, s + 2, cb, rb, ca, ra);
      step(integral_constant<int, 0>{}, std::false_type{}, s + 3, ca, ra, cb, rb);
    }
    if (s < steps) {
      step(integral_constant<int, 1>{}, std::false_type{}, s, cb, rb, ca, ra);
      if (s + 1 < steps) {
        step(integral_constant<int, 2>{}, std::false_type{}, s + 1, ca, ra, cb, rb);
        if (s + 2 < steps) step(integral_constant<int, 3>{}, std::false_type{}, s + 2, cb, rb, ca, ra);
      }
    }
    Tile next{};
    if (!INPUT && args.queue != nullptr) {
      if (threadIdx.x == 0) *mail = fetched;
      FLUXMI_LGKM0();
      __builtin_amdgcn_s_barrier();  // nobody reads the slots any more
      next = tile_of_queue(home, (args.grid >> 3) + __builtin_amdgcn_readfirstlane(*mail));
      // The own queue is empty: the others'.
      for (int q = 1; q < 8 && next.rows == 0; ++q) {
        const int other = (home + q) & 7;
        __syncthreads();
        if (threadIdx.x == 0) *mail = atomicAdd(args.queue + other * kQueueLine, 1);
        __syncthreads();
        next = tile_of_queue(other, (args.grid >> 3) + __builtin_amdgcn_readfirstlane(*mail));
      }
    } else {
      if (turn < args.turns) next = tile_of_turn(turn++);
      __builtin_amdgcn_s_barrier();  // nobody reads the slots any more
    }
    if (next.rows > 0) {
      begin_tile(next);
      first_fills();
    }
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // the last sums are in their registers

    // ---- results: lane l has columns 4 (l / 16) .. + 3 of row l % 16 of a block.  Sixteen rows of 128 bytes at a time change lanes in the wave's window (chunk c of 16
    // bytes of row r at place c ^ (r / 2 % 8), off the other lanes' banks either way), so that eight neighbouring lanes store a whole line: stored from where
    // they are, neighbouring lanes' pieces lie in different rows, and a compute unit brings out a quarter as much. ----
    {
      const int l = fresh_lane(), r = l & 15, g = l >> 4;
      const uint32_t window = lds0 + windows_at(G) + wave * kWindow;
      const uint32_t from = window + (l >> 3) * 128 + ((l & 7) ^ ((l >> 4) & 7)) * 16;  // rows l / 8 and l / 8 + 8: the latter's place is another, 64 bytes from it
      // The buffer ends with the tile's rows; columns past its end are sent past the buffer's.  Every store is issued, so that they can be counted.
      const bool part = tile.part >= 0, f32 = part || a.out_f32, add = !part && a.accumulate;
      const int out_size = f32 ? 4 : 2;
      const uint32_t pitch = part ? kTile : a.k;
      uint8_t *const base = part ? reinterpret_cast<uint8_t *>(a.partial + static_cast<int64_t>(tile.slot) * kTile * kTile) : a.out + tile.out_row0 * a.k * out_size;
      const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(base, 0, static_cast<int>(static_cast<uint32_t>(tile.rows) * pitch * out_size), 0x00020000);
      const uint32_t row_at = static_cast<uint32_t>(wr * 16 + (l >> 3)) * pitch + (part ? 0 : tile.col0);
      // Results of group N are read before those of the one before it are stored.
      u32x4 v[2][2];
      auto read_back = [&](auto N) {
        constexpr int b = decltype(N)::value & 1;
        v[b][0] = *(LdsFrag)(uintptr_t)from;
        v[b][1] = *(LdsFrag)(uintptr_t)((from ^ 64) + 1024);
        __builtin_amdgcn_sched_barrier(0);
      };
      auto store_results = [&](auto LINES) {
        constexpr int policy = decltype(LINES)::value ? 2 : 0;  // non-temporal
        if (f32 || add) {
          auto put = [&](auto N) {
            constexpr int i = decltype(N)::value / 4, j = decltype(N)::value % 4 * 2;
  #pragma unroll
            for (int h = 0; h < 2; ++h)
              *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(window + r * 128 + ((h * 4 + g) ^ (r >> 1)) * 16) = __builtin_bit_cast(u32x4, sums_of(acc[i][j + h]));
            read_back(N);
          };
          put(integral_constant<int, 0>{});
          static_for<32>([&](auto N) {
            constexpr int n = decltype(N)::value, i = n / 4, j = n % 4 * 2;
            if constexpr (n < 31) put(integral_constant<int, (n < 31 ? n + 1 : 0)>{});
            const int c = wc * 128 + j * 16 + (l & 7) * 4;
  #pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t at = c < tile.cols ? (row_at + (i * 32 + h * 8) * pitch + c) * out_size : 0xfffffff0u;
              f32x4 x = __builtin_bit_cast(f32x4, v[n & 1][h]);
              if (!add) {
                __builtin_amdgcn_raw_buffer_store_b128(v[n & 1][h], out, at, 0, policy);
              } else if (f32) {
                x += __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(out, at, 0, 0));
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), out, at, 0, 0);
              } else {
                const u32x2 old = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(out, at, 0, 0));
  #pragma unroll
                for (int q = 0; q < 4; ++q) x[q] += unpack1<F16>(static_cast<uint16_t>(old[q / 2] >> (16 * (q & 1))));
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3])}, out, at, 0, 0);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          });
          behind = 2;
          if (add) {
            FLUXMI_VMCNT(0);
            behind = 0;
          }
        } else {
          auto put = [&](auto N) {
            constexpr int i = decltype(N)::value / 2, j = decltype(N)::value % 2 * 4;
  #pragma unroll
            for (int h = 0; h < 4; ++h) {
              const f32x4 x = sums_of(acc[i][j + h]);
              *(__attribute__((address_space(3))) u32x2 *)(uintptr_t)(window + r * 128 + ((h * 2 + (g >> 1)) ^ (r >> 1)) * 16 + (g & 1) * 8) =
                  u32x2{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3])};
            }
            read_back(N);
          };
          put(integral_constant<int, 0>{});
          static_for<16>([&](auto N) {
            constexpr int n = decltype(N)::value, i = n / 2, j = n % 2 * 4;
            if constexpr (n < 15) put(integral_constant<int, (n < 15 ? n + 1 : 0)>{});
            const int c = wc * 128 + j * 16 + (l & 7) * 8;
  #pragma unroll
            for (int h = 0; h < 2; ++h) __builtin_amdgcn_raw_buffer_store_b128(v[n & 1][h], out, c < tile.cols ? (row_at + (i * 32 + h * 8) * pitch + c) * 2 : 0xfffffff0u, 0, policy);
            __builtin_amdgcn_sched_barrier(0);
          });
          behind = 1;
        }
      };
      // Whole lines pass the caches by; parts of lines would come from memory again.  us, through / past the caches, weights of 64 experts to bf16 (fp32): 1408 x 2048, 128 rows
      // each 138 / 99 (182 / 141), 512 219 / 195 (291 / 231), 1024 347 / 357 (413 / 422); 1400 x 2040, whose rows begin off the lines, 161 / 196 (219 / 366), 256 / 208 (318 / 340),
      // 376 / 399 (455 / 524).
      if (!part && (a.k * out_size & 127) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 127) == 0) store_results(std::true_type{});
      else store_results(std::false_type{});
    }
    if (next.rows == 0) break;
    tile = next;
  }
  FLUXMI_VMCNT(0);  // no fill may come after the workgroup's end
#endif
}

// Empties the queues, and puts the experts in order.
__global__ __launch_bounds__(kMaxExperts) void grad_queue_kernel(const GradArgs a, int32_t *queue) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ int rows[kMaxExperts];
  if (threadIdx.x < 64) {
    int carry = 0;
    for (int e0 = 0; e0 < a.nexperts; e0 += 64) {
      const ExpertRows x = rows_of_lane(a, e0, carry);
      rows[e0 + threadIdx.x] = x.end - x.begin;
    }
  }
  if (threadIdx.x < 8) queue[threadIdx.x * kQueueLine] = 0;
  __syncthreads();
  const int e = threadIdx.x;
  if (e >= a.nexperts) return;
  const int mine = rows[e];
  int before = 0;
  for (int i = 0; i < a.nexperts; ++i) before += rows[i] > mine || (rows[i] == mine && i < e) ? 1 : 0;
  queue[kQueueExperts + before] = e;
#endif
}

// The parts of the last turn's tiles, added in their order: a workgroup has sixteen rows of a tile.
template <bool F16, Grad G>
__global__ __launch_bounds__(kThreads) void grad_tile_join_kernel(const TileArgs args) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool INPUT = G == Grad::INPUT;
  const GradArgs &a = args.a;
  const int tiles_k = (a.k + kTile - 1) / kTile, tiles_n = (a.n + kTile - 1) / kTile;
  int row_tiles = a.nexperts * tiles_n, all_rows = 0;
  if constexpr (INPUT) {
    row_tiles = 0;
    for (int e0 = 0; e0 < a.nexperts; e0 += 64) {
      const ExpertRows x = rows_of_lane(a, e0, all_rows);
      row_tiles += __builtin_amdgcn_readlane(wave_inclusive_scan((x.end - x.begin + kTile - 1) / kTile), 63);
    }
    row_tiles += (a.rows - all_rows + kTile - 1) / kTile;
  }
  const Turns turns = turns_of(row_tiles * tiles_k, args.grid, args.cutting);
  const int cut = blockIdx.x >> 4;
  if (cut >= turns.cut) return;
  const int item = turns.whole + cut, e = INPUT ? 0 : item / (tiles_n * tiles_k), local = INPUT ? item : item - e * tiles_n * tiles_k;
  const int group = local / (8 * tiles_k), in_group = local - group * 8 * tiles_k;
  const int high = (INPUT ? row_tiles : tiles_n) - group * 8, height = high < 8 ? high : 8;
  const int kt = in_group / height, rt = group * 8 + in_group - kt * height;
  int rows;
  int64_t out_row0;
  if constexpr (INPUT) {
    const RowTile t = row_tile<kTile>(a, rt);
    rows = t.rows;
    out_row0 = t.row0;
  } else {
    rows = a.n - rt * kTile;
    out_row0 = static_cast<int64_t>(e) * a.n + rt * kTile;
  }
  const int c = (threadIdx.x & 63) * 4, col = kt * kTile + c;
  if (col >= a.k) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (blockIdx.x & 15) * 16 + i * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int part = 0; part < turns.parts; ++part)
      v += *reinterpret_cast<const f32x4 *>(a.partial + (static_cast<int64_t>(part * turns.cut + cut) * kTile + r) * kTile + c);
    store4_whole<F16>(a, (out_row0 + r) * a.k + col, v);
  }
#endif
}

// Tiles of the result (INPUT: as many as there can be).
int64_t most_tiles(Grad g, int64_t nexperts, int64_t rows, int64_t n, int64_t k) {
  const int64_t tiles_k = (k + kTile - 1) / kTile, tiles_n = (n + kTile - 1) / kTile;
  return g == Grad::INPUT ? (rows / kTile + (rows < nexperts ? rows : nexperts) + 1) * tiles_k : nexperts * tiles_n * tiles_k;
}

Cutting cutting_of(Grad g, int64_t nexperts, int64_t rows, int64_t n) {
  const int64_t each = rows / (nexperts > 0 ? nexperts : 1), height = g == Grad::INPUT ? each : n;
  const int64_t steps = (g == Grad::INPUT ? n : each) / kStep;
  return {static_cast<int32_t>(steps < 1 << 20 ? steps : 1 << 20), static_cast<int32_t>(height < 16 ? 16 : (height > kTile ? kTile : height))};
}

// One workgroup to a compute unit: its tiles follow each other without a gap.
int grid_of(int64_t tiles) {
  const int cus = fluxmi_device_cu_count(), all = cus > 8 ? cus / 8 * 8 : 256;
  const int64_t want = (tiles * kMostParts + 7) / 8 * 8;
  return want < all ? static_cast<int>(want) : all;
}

}  // namespace

bool grad_tiles_take(Grad g, const GradArgs &a) {
  const auto on16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  if (a.n == 0 || a.nexperts == 0 || a.n % 8 != 0 || a.k % (g == Grad::WEIGHT_8BIT ? 16 : 8) != 0 || !on16(a.grad) || !on16(a.other) || !on16(a.out)) return false;
  if (most_tiles(g, a.nexperts, a.rows, a.n, a.k) >= 1 << 24) return false;
  // Offsets: 256 rows of G along, 32 rows across, 256 rows of the result.
  return a.n < 1 << 22 && a.k < 1 << 22;
}

// us, pieces of 128 x 128 / tiles.  Weights (experts, n x k, rows in all): 1, 1024 x 1024, 8192 41 / 55, 16384 62 / 59; 8, 512 x 512, 32768 41 / 52; 8, 1024 x 1024, 2048 15 / 15, 16384 56 / 51; 1, 1408 x 2048,
// 2048 39 / 45, 8192 92 / 67; 32, 1024 x 1024, 4096 34 / 22.  Input: 1, 512 x 512, 8192 16 / 25, 32768 38 / 26; 8, 1024 x 1024, 2048 26 / 33, 16384 63 / 36; 8, 1408 x 2048, 2048 34 / 45, 8192 73 / 45;
// 8, 2048 x 4096, 64 41 / 37; 8, 2048 x 128, 64 37 / 20; 32, 2048 x 4096, 64 123 / 96.
bool grad_tiles_are_faster(Grad g, int32_t nexperts, int64_t rows, int64_t n, int64_t k) {
  const double weights = static_cast<double>(nexperts) * n * k, flops = 2.0 * rows * n * k;
  if (g == Grad::INPUT) return flops >= 1.6e10 || weights >= 6e7 || n >= 2048;
  return flops >= 2.4e10 || most_tiles(g, nexperts, rows, n, k) >= 64;
}

// Several experts in four turns or more: a workgroup fetches its next tile when it has done with one.  The result has the same bits: a tile's sum is the same wherever
// it is computed.  us, queue / turns: 64 skewed experts 1400 x 2040 to fp32 602 / 735; equal ones, 8 of 14336 x 4096 1400 / 1401, 32 of 2048 x 7168 from 8 bits 1047 / 1060.
static bool by_queue(Grad g, int64_t nexperts, int64_t tiles, int grid) { return g != Grad::INPUT && nexperts > 1 && tiles >= 4 * static_cast<int64_t>(grid); }

size_t grad_tiles_workspace_bytes(Grad g, int32_t nexperts, int64_t rows, int64_t n, int64_t k) {
  const int64_t tiles = most_tiles(g, nexperts, rows, n, k);
  if (tiles == 0 || tiles >= 1 << 24 || !grad_tiles_are_faster(g, nexperts, rows, n, k)) return 0;
  const int grid = grid_of(tiles);
  if (by_queue(g, nexperts, tiles, grid)) return kQueueBytes;
  const Cutting c = cutting_of(g, nexperts, rows, n);
  // (the input's gradient has as many tiles as the row counts make, which are not known here: one may be all that is cut)
  if (turns_of(g == Grad::INPUT ? 1 : static_cast<int>(tiles), grid, c).cut == 0) return 0;
  return static_cast<size_t>(grid) * kTile * kTile * sizeof(float);  // (a part to each workgroup at most)
}

int launch_grad_tiles(Grad g, bool f16, const GradArgs &args, void *stream) {
  const GradArgs &a = args;
  const int64_t tiles_k = (a.k + kTile - 1) / kTile, tiles_n = (a.n + kTile - 1) / kTile, tiles = most_tiles(g, a.nexperts, a.rows, a.n, a.k);
  const int grid = grid_of(tiles);
  const bool queue = by_queue(g, a.nexperts, tiles, grid);
  const TileArgs t{a, cutting_of(g, a.nexperts, a.rows, a.n), grid, static_cast<int32_t>(tiles / grid + 1), divisor(tiles_n * tiles_k), divisor(8 * tiles_k), queue ? reinterpret_cast<int32_t *>(a.partial) : nullptr};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (queue) {
    grad_queue_kernel<<<1, kMaxExperts, 0, s>>>(a, t.queue);
    FLUXMI_HIP_CHECK(hipGetLastError());
  }
  const bool join = !queue && grad_tiles_workspace_bytes(g, a.nexperts, a.rows, a.n, a.k) > 0;
  auto launch = [&](auto F, auto K, auto FEW, std::atomic<uint64_t> &done) -> int {
    constexpr bool f = decltype(F)::value, few = decltype(FEW)::value;
    constexpr Grad k = decltype(K)::value;
    if (const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(grad_tile_kernel<f, k, few>), lds_bytes(k), done)) return rc;
    grad_tile_kernel<f, k, few><<<grid, kThreads, lds_bytes(k), s>>>(t);
    FLUXMI_HIP_CHECK(hipGetLastError());
    if (join) {
      // (at most half the workgroups have a tile that is cut)
      grad_tile_join_kernel<f, k == Grad::INPUT ? Grad::INPUT : Grad::WEIGHT><<<grid / 2 * 16, kThreads, 0, s>>>(t);
      FLUXMI_HIP_CHECK(hipGetLastError());
    }
    return FLUXMI_OK;
  };
  static std::atomic<uint64_t> done[8];
  const auto by_type = [&](auto K, auto FEW, int at) { return f16 ? launch(std::true_type{}, K, FEW, done[at]) : launch(std::false_type{}, K, FEW, done[at + 1]); };
  using std::integral_constant;
  // us, all row blocks -> those that there are: 8 experts 14336 x 4096, 74 rows in all 190 -> 176, 512 rows 195 -> 186, 4096 x 14336, 512 rows 210 -> 196, 32 experts 2048 x 7168,
  // 1024 rows 207 -> 191; 8 experts 4096 x 4096, 2048 rows 106 -> 109, 16384 rows 411 -> 454; 64 experts 1408 x 2048, 98304 rows 531 -> 570.
  if (g == Grad::INPUT && a.rows < static_cast<int64_t>(a.nexperts) * 160) return by_type(integral_constant<Grad, Grad::INPUT>{}, std::true_type{}, 0);
  if (g == Grad::INPUT) return by_type(integral_constant<Grad, Grad::INPUT>{}, std::false_type{}, 2);
  if (g == Grad::WEIGHT) return by_type(integral_constant<Grad, Grad::WEIGHT>{}, std::false_type{}, 4);
  return by_type(integral_constant<Grad, Grad::WEIGHT_8BIT>{}, std::false_type{}, 6);
}

}  // namespace fluxmi
