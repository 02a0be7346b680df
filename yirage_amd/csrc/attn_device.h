// Device helpers shared by the attention kernels.
#pragma once
#include "yr_common.h"

namespace yr {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;  // running-max slack (log2 units)

// P is rounded to 16 bits for the second product, the row sum is not: half a step of
// each weight, against the result's own half step (fp32 products would take 8 times
// the matrix instructions).  f16's normal range ends at
// 2^-14: weights carry a factor 2^7 there (cancelled by the row sum, at most
// 2^15 with the lazy maximum's slack of 2^8), so a weight loses bits only below
// 2^-21 of the largest and vanishes below 2^-32.
template <int DT>
constexpr float kPBias = DT == DT_F16 ? 7.f : 0.f;

// An exponent is one fma, score log2 e / sqrt(D) less the running maximum, a rounded
// number: the largest comes out as that rounding, a 16th at most up to here.  From
// 2^24 on it may be 1 and more, and P, up to 2^15 with its factor and slack, would leave
// f16's range, from 2^31 on fp32's; so beyond this the product is rounded like the
// maximum before they are subtracted (777 rows of 16 pages of 64: 1 % for the branch).
constexpr float kFarScore = 0x1p20f;
__device__ __forceinline__ float far_exponent(float score, float scale, float m) {
  float x = score * scale;
  asm volatile("" : "+v"(x));  // (no fma)
  return fabsf(m) > kFarScore ? x - m : fmaf(score, scale, -m);
}

// 4 consecutive 16-bit elements from LDS, transposed across each 16-lane group
// (an address-space cast, not a trip through an integer: the compiler keeps
// track of the LDS object and does not wait for direct loads into others)
__device__ __forceinline__ uint2 lds_tr4(const uint16_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)p));
}

// max over lanes l and l ^ 16 (l ^ 32): a permlane swap of the value with
// itself hands each 16-lane row its partner row, in registers (no LDS trip)
__device__ __forceinline__ float max_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 16 bytes per lane from global memory straight into LDS: lane l's data
// lands at lds_base + 16 l (lds_base wave-uniform)
__device__ __forceinline__ void lds_load16(const uint16_t* g, uint16_t* lds_base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(g),
                                   reinterpret_cast<__attribute__((address_space(3))) void*>(
                                       reinterpret_cast<__attribute__((address_space(3))) char*>(
                                           reinterpret_cast<uintptr_t>(lds_base))),
                                   16, 0, 0);
}

// 4 bytes (or 1, zero-extended) per lane: lane l's land at lds_base + 4 l bytes
__device__ __forceinline__ void lds_load4(const void* g, uint32_t* lds_base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(g),
                                   reinterpret_cast<__attribute__((address_space(3))) void*>(
                                       reinterpret_cast<__attribute__((address_space(3))) char*>(
                                           reinterpret_cast<uintptr_t>(lds_base))),
                                   4, 0, 0);
}
__device__ __forceinline__ void lds_load1(const void* g, uint32_t* lds_base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(g),
                                   reinterpret_cast<__attribute__((address_space(3))) void*>(
                                       reinterpret_cast<__attribute__((address_space(3))) char*>(
                                           reinterpret_cast<uintptr_t>(lds_base))),
                                   1, 0, 0);
}

}  // namespace yr
