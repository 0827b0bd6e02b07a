// Gradients of the grouped product: what its kernels share.
#pragma once
#include "common.hpp"

namespace fluxmi {

constexpr int kMaxExperts = 1024;
constexpr int kGradMaxRows = 1 << 24;  // 64 counts of it still fit 32 bits

enum class Grad { INPUT, WEIGHT, WEIGHT_8BIT };  // WEIGHT_8BIT: the product's input is a checkpoint in 8 bits

struct GradArgs {
  const uint8_t *grad;     // [rows, n], 16 bits
  const uint8_t *other;    // INPUT: weight [nexperts, n, k]; otherwise the product's input [rows, k]: 16 bits, or e4m3 codes
  const uint8_t *scale;    // WEIGHT_8BIT: [rows, ceil(k / 32)]
  uint8_t *out;            // INPUT: [rows, k]; otherwise [nexperts, n, k]
  float *partial;          // parts of sums, where there is more than one
  const int32_t *splits;   // device [nexperts]
  int32_t nexperts, rows, n, k;
  int32_t out_f32, accumulate;
  int32_t parts;           // an expert's rows are summed in so many parts
};

namespace {

#if defined(__HIP_DEVICE_COMPILE__)

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 *LdsTr;

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
  else return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
}
template <bool F16>
__device__ __forceinline__ float unpack1(uint16_t v) {
  return F16 ? f16_bits_to_float(v) : bf16_bits_to_float(v);
}

// The rows of an expert.  Negative counts are 0; what lies past `rows` does not exist.
struct ExpertRows {
  int begin, end;
};
__device__ __forceinline__ ExpertRows rows_of_lane(const GradArgs &a, int e0, int &carry) {
  const int e = e0 + lane_id();
  int r = e < a.nexperts ? a.splits[e] : 0;
  r = r < 0 ? 0 : (r > a.rows ? a.rows : r);
  const int incl = wave_inclusive_scan(r);
  ExpertRows x = {carry + incl - r, carry + incl};
  if (x.begin > a.rows) x.begin = a.rows;
  if (x.end > a.rows) x.end = a.rows;
  carry = __builtin_amdgcn_readlane(x.end, 63);
  return x;
}
__device__ __forceinline__ ExpertRows rows_of_expert(const GradArgs &a, int e) {
  int carry = 0;
  for (int e0 = 0;; e0 += 64) {
    const ExpertRows x = rows_of_lane(a, e0, carry);
    if (e < e0 + 64) return {__builtin_amdgcn_readlane(x.begin, e - e0), __builtin_amdgcn_readlane(x.end, e - e0)};
  }
}

// Row tile `tile` of all experts' rows, cut into tiles of HEIGHT rows; behind the last expert come the rows that belong to none (e = nexperts).
struct RowTile {
  int e, row0, rows;  // rows = 0: there is no such tile
};
template <int HEIGHT>
__device__ __forceinline__ RowTile row_tile(const GradArgs &a, int tile) {
  int carry = 0, tiles = 0;
  for (int e0 = 0; e0 < a.nexperts; e0 += 64) {
    const ExpertRows x = rows_of_lane(a, e0, carry);
    const int mine = (x.end - x.begin + HEIGHT - 1) / HEIGHT, end = tiles + wave_inclusive_scan(mine);
    const uint64_t hit = __ballot(tile < end);
    if (hit != 0) {
      const int src = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      const int begin = __builtin_amdgcn_readlane(x.begin, src), last = __builtin_amdgcn_readlane(x.end, src);
      const int row0 = begin + (tile - (__builtin_amdgcn_readlane(end, src) - __builtin_amdgcn_readlane(mine, src))) * HEIGHT;
      return {e0 + src, row0, last - row0 < HEIGHT ? last - row0 : HEIGHT};
    }
    tiles = __builtin_amdgcn_readlane(end, 63);
  }
  const int64_t row0 = carry + static_cast<int64_t>(tile - tiles) * HEIGHT;
  if (row0 >= a.rows) return {a.nexperts, 0, 0};
  return {a.nexperts, static_cast<int>(row0), a.rows - static_cast<int>(row0) < HEIGHT ? a.rows - static_cast<int>(row0) : HEIGHT};
}

// Four neighbouring sums of a row to out[at ..], which starts on a multiple of four elements.
template <bool F16>
__device__ __forceinline__ void store4_whole(const GradArgs &a, int64_t at, f32x4 v) {
  if (a.out_f32) {
    float *p = reinterpret_cast<float *>(a.out) + at;
    if (a.accumulate) v += *reinterpret_cast<const f32x4 *>(p);
    *reinterpret_cast<f32x4 *>(p) = v;
    return;
  }
  uint16_t *p = reinterpret_cast<uint16_t *>(a.out) + at;
  if (a.accumulate) {
    const u32x2 old = *reinterpret_cast<const u32x2 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += unpack1<F16>(static_cast<uint16_t>(old[i / 2] >> (16 * (i & 1))));
  }
  *reinterpret_cast<u32x2 *>(p) = u32x2{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3])};
}
// The same for the first `count` of them, at any element unless `aligned`.
template <bool F16>
__device__ __forceinline__ void store4(const GradArgs &a, int64_t at, f32x4 v, int count, bool aligned) {
  if (count >= 4 && aligned) {
    store4_whole<F16>(a, at, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= count) continue;
    if (a.out_f32) {
      float *p = reinterpret_cast<float *>(a.out) + at + i;
      *p = a.accumulate ? *p + v[i] : v[i];
    } else {
      uint16_t *p = reinterpret_cast<uint16_t *>(a.out) + at + i;
      *p = static_cast<uint16_t>(pack2<F16>(a.accumulate ? v[i] + unpack1<F16>(*p) : v[i], 0.f));
    }
  }
}

#endif  // __HIP_DEVICE_COMPILE__

}  // namespace
}  // namespace fluxmi
