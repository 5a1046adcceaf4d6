// What the attention kernels that hold a query row across four lanes, or two, share:
// the row's maximum and sum, and how infinities and NaN in values are told and kept
// from rows that do not see them.
#pragma once

#include "chunk_traits.hpp"

namespace mvr {
namespace {

constexpr float kRescaleThreshold = 8.0f; // log2 units: P <= 2^8 between rescales

// 0 for a row without a key (its sum is 0: no exponential was added), else 1 / sum.
__device__ __forceinline__ float inverse_sum(float sum) { return __float_as_uint(sum) == 0 ? 0.f : 1.f / sum; }

typedef half_t half2v __attribute__((ext_vector_type(2)));

// Maximum and sum over the lanes l, l ^ 16, l ^ 32, l ^ 48, which hold one query row.
__device__ __forceinline__ float row_max(float v) {
  const uint32_t x = __float_as_uint(v);
  const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1])));
  const auto halves = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  const uint32_t x = __float_as_uint(v);
  const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const uint32_t y = __float_as_uint(__uint_as_float(rows[0]) + __uint_as_float(rows[1]));
  const auto halves = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
}

// Infinities and NaN are told by their bits, which are opaque to the optimiser
// here: where a file is compiled without regard for NaN, it would take such a
// test for one that only infinities pass.
__device__ __forceinline__ uint32_t opaque_bits(uint32_t x) {
  asm("" : "+v"(x));
  return x;
}
__device__ __forceinline__ bool non_finite_bits(half_t, uint32_t x) { return (x & 0x7c00u) == 0x7c00u; }
__device__ __forceinline__ bool non_finite_bits(float, uint32_t x) { return (x & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t bits_of(half_t v) { return opaque_bits(__builtin_bit_cast(uint16_t, v)); }
__device__ __forceinline__ uint32_t bits_of(float v) { return opaque_bits(__float_as_uint(v)); }
__device__ __forceinline__ half_t from_bits(half_t, uint32_t x) { return __builtin_bit_cast(half_t, (uint16_t)x); }
__device__ __forceinline__ float from_bits(float, uint32_t x) { return __uint_as_float(x); }

__device__ __forceinline__ bool any_non_finite(const half8& v) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 x = __builtin_bit_cast(u32x4, v);
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint32_t pair = opaque_bits(x[e]);
    bad |= (pair & 0x7c00u) == 0x7c00u || (pair & 0x7c000000u) == 0x7c000000u;
  }
  return bad;
}
__device__ __forceinline__ bool any_non_finite(const float4v& v) {
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; e++) bad |= non_finite_bits(v[e], bits_of(v[e]));
  return bad;
}

template <typename T>
__device__ __forceinline__ T finite_or_zero(T v) {
  const uint32_t x = bits_of(v);
  return from_bits(v, non_finite_bits(v, x) ? 0 : x);
}

// An infinity or a NaN itself, 0 for a finite value.
template <typename T>
__device__ __forceinline__ float non_finite_part(T v) {
  const uint32_t x = bits_of(v);
  return (float)from_bits(v, non_finite_bits(v, x) ? x : 0);
}

} // namespace
} // namespace mvr
