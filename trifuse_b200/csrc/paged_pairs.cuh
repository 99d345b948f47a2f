// Packed fp32 pairs of the append kernels: arithmetic, and conversion from and
// to eight 16-bit values.
#pragma once

#include "common.cuh"

namespace tf {

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}
// Eight values as four packed pairs, and back with one rounding (by the paired
// conversions: value by value they took half of the kernel's instructions).
__device__ __forceinline__ float2 pair_of(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t word_of(float2 f, __half) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t word_of(float2 f, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack4(const uint4& v, float2* f) {
  f[0] = pair_of(v.x, T());
  f[1] = pair_of(v.y, T());
  f[2] = pair_of(v.z, T());
  f[3] = pair_of(v.w, T());
}
template <typename T>
__device__ __forceinline__ uint4 pack4(const float2* f) {
  return make_uint4(word_of(f[0], T()), word_of(f[1], T()), word_of(f[2], T()), word_of(f[3], T()));
}

}  // namespace tf
