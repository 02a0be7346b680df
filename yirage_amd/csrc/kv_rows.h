// A head's row of a new token as the operators that append to a paged cache hold it:
// D / 16 lanes, 8 elements of each half a lane, so a rotated pair sits in one lane.
#pragma once
#include "ragged.h"

namespace yr {

// What is written is not read again here: stored past the caches.
__device__ __forceinline__ void stg16_stream(uint16_t* p, uint4 v) {
  __builtin_nontemporal_store(__builtin_bit_cast(yr_u32x4, v), (YR_G yr_u32x4*)p);
}
template <int DT>
__device__ __forceinline__ void unpack8(uint4 v, float* x) {
  x[0] = lo16<DT>(v.x); x[1] = hi16<DT>(v.x); x[2] = lo16<DT>(v.y); x[3] = hi16<DT>(v.y);
  x[4] = lo16<DT>(v.z); x[5] = hi16<DT>(v.z); x[6] = lo16<DT>(v.w); x[7] = hi16<DT>(v.w);
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7]));
}

// 8 table entries at `at`
template <int DT, bool F32>
__device__ __forceinline__ void table8(const void* t, size_t at, float* x) {
  if constexpr (F32) {
    const uint4 a = ldg16((const float*)t + at), b = ldg16((const float*)t + at + 4);
    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
  } else {
    unpack8<DT>(ldg16((const uint16_t*)t + at), x);
  }
}

// One lane's angles at position p.
template <int DT, int D, bool F32>
__device__ __forceinline__ void angles(const void* cos_table, const void* sin_table, int p, int l, float* c, float* s) {
  const size_t at = (size_t)p * D + 8 * l;
  table8<DT, F32>(cos_table, at, c);
  table8<DT, F32>(cos_table, at + D / 2, c + 8);
  table8<DT, F32>(sin_table, at, s);
  table8<DT, F32>(sin_table, at + D / 2, s + 8);
}

// One lane's 16 elements of a row, normalised by the weights w and rotated.
template <int D>
__device__ __forceinline__ void norm_rotate(bool norm, bool rotate, float eps, const float* w, const float* c,
                                            const float* s, float* x) {
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = 1; o < D / 16; o <<= 1) ss += __shfl_xor(ss, o, kWave);
    const float f = 1.f / sqrtf(ss * (1.f / D) + eps);
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = x[i] * f * w[i];
  }
  if (rotate) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float u = x[i], t = x[i + 8];
      x[i] = u * c[i] - t * s[i];
      x[i + 8] = t * c[i + 8] + u * s[i + 8];
    }
  }
}
// The same from 16 bits to 16 bits, with one rounding.
template <int DT, int D>
__device__ __forceinline__ void norm_rotate(bool norm, bool rotate, float eps, const float* w, const float* c,
                                            const float* s, uint4 lo, uint4 hi, uint4* out) {
  float x[16];
  unpack8<DT>(lo, x);
  unpack8<DT>(hi, x + 8);
  norm_rotate<D>(norm, rotate, eps, w, c, s, x);
  out[0] = pack8<DT>(x);
  out[1] = pack8<DT>(x + 8);
}

}  // namespace yr
