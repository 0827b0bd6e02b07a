// Rows of bf16, fp32 or fp16 in vectors of 16 bytes at any address; shared by the kernels that move and convert them.
#pragma once
#include <type_traits>

#include "common.hpp"

namespace fluxmi {
namespace {

enum class Row { BF16, F32, F16 };

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));  // at any address: one instruction on this hardware

template <bool NT = false>
__device__ __forceinline__ u32x4 load16(const uint8_t *p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
  else return *reinterpret_cast<const u32x4_any *>(p);
}
template <bool NT = false>
__device__ __forceinline__ void store16(uint8_t *p, u32x4 v) {
  if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any *>(p));
  else *reinterpret_cast<u32x4_any *>(p) = v;
}

template <Row T>
constexpr int kElt = T == Row::F32 ? 4 : 2;
template <Row T>
constexpr int kVec = 16 / kElt<T>;  // elements of a vector

template <Row T>
__device__ __forceinline__ void unpack(const u32x4 v, float (&x)[kVec<T>]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == Row::F32) {
      x[i] = __uint_as_float(v[i]);
    } else if constexpr (T == Row::F16) {
      x[2 * i] = f16_bits_to_float(static_cast<uint16_t>(v[i] & 0xffffu));
      x[2 * i + 1] = f16_bits_to_float(static_cast<uint16_t>(v[i] >> 16));
    } else {
      x[2 * i] = __uint_as_float(v[i] << 16);
      x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
}

typedef __bf16 bf16_pair __attribute__((ext_vector_type(2)));

// One rounding to the rows' type.
template <Row T>
__device__ __forceinline__ u32x4 pack(const float (&x)[kVec<T>]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == Row::F32) v[i] = __float_as_uint(x[i]);
    else if constexpr (T == Row::F16) v[i] = float_to_f16_bits(x[2 * i]) | static_cast<uint32_t>(float_to_f16_bits(x[2 * i + 1])) << 16;
    else v[i] = __builtin_bit_cast(uint32_t, bf16_pair{static_cast<__bf16>(x[2 * i]), static_cast<__bf16>(x[2 * i + 1])});  // one conversion instruction
  }
  return v;
}

// ---- host ----------------------------------------------------------------------------------------------------
inline int check_type(const char *who, int32_t type, Row *row) {
  FLUXMI_REQUIRE(type == FLUXMI_ROWS_BF16 || type == FLUXMI_ROWS_FP32 || type == FLUXMI_ROWS_FP16, FLUXMI_ERR_INVALID_ARG, "%s: unknown type %d", who, type);
  *row = type == FLUXMI_ROWS_BF16 ? Row::BF16 : type == FLUXMI_ROWS_FP32 ? Row::F32 : Row::F16;
  return FLUXMI_OK;
}

inline bool aligned_to(const void *p, Row t) { return (reinterpret_cast<uintptr_t>(p) & (t == Row::F32 ? 3u : 1u)) == 0; }

template <class F>
void by_type(Row t, F &&f) {
  if (t == Row::BF16) f(std::integral_constant<Row, Row::BF16>{});
  else if (t == Row::F32) f(std::integral_constant<Row, Row::F32>{});
  else f(std::integral_constant<Row, Row::F16>{});
}

}  // namespace
}  // namespace fluxmi
