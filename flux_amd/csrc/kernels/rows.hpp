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
