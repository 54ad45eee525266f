// A lane's share of a row of scores, in the attentions whose lanes hold one row each (a lane and the one 32 away:
// a 32 x 32 product's columns): packing, sums of packed weights, and what passes between the two halves.
#pragma once

#include "nt_common.h"

namespace nt {
namespace lane_rows {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf162_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, f16_t>::value)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{lo, hi}, half2_t));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{lo, hi}, bf162_t));
}

// The magnitude bits of infinity in the 16-bit types: above it lie the NaN.
template <typename T>
constexpr uint32_t inf_bits = std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u;
template <typename T>
constexpr uint32_t one_bits = std::is_same<T, f16_t>::value ? 0x3c00u : 0x3f80u;

// x of lane l ^ 32, and the larger of the two.  (v_permlane32_swap of two copies of x leaves the
// low half's values in the first and the high half's in the second, in both halves; the VALU
// write of its operands needs wait states before it.)
__device__ __forceinline__ void both_halves(float x, float& lo, float& hi) {
  lo = x;
  hi = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
}
__device__ __forceinline__ float max_halves(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float other_half(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return (threadIdx.x & 32) ? lo : hi;
}
// acc plus the two packed values of w, in fp32.
template <typename T>
__device__ __forceinline__ float add2(uint32_t w, float acc) {
  const uint32_t one2 = one_bits<T> | one_bits<T> << 16;
  if constexpr (std::is_same<T, f16_t>::value)
    acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, w), __builtin_bit_cast(half2_t, one2), acc, false);
  else
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf162_t, w), __builtin_bit_cast(bf162_t, one2), acc, false);
  return acc;
}

// Eight packed values with zeros for the infinities and NaN.
template <typename T>
__device__ __forceinline__ u32x4 finite8(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = ((w[i] & 0x7fffu) < inf_bits<T> ? w[i] & 0xffffu : 0u) |
           (((w[i] >> 16) & 0x7fffu) < inf_bits<T> ? w[i] & 0xffff0000u : 0u);
  return w;
}

}  // namespace lane_rows
}  // namespace nt
