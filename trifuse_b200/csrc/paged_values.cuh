// Values of masked keys.  A masked key has weight 0, but 0 * inf and 0 * NaN
// are NaN, so a value that is not finite would reach the rows that must not see
// its key wherever a tile's product takes in both.  Tiles with such rows are
// therefore looked through before their product: values that are not finite,
// of keys that some row of the tile does not see, become zeros in shared
// memory, and are added again to the rows that do see them (whose result they
// decide alone: a sum with an infinity or a NaN in it).
#pragma once

#include <math.h>

#include "common.cuh"

namespace tf {

// Eight values: acc + 0 * v in packed halves, NaN from the first one that is
// not finite on.
__device__ __forceinline__ __half2 fold_finite(const uint4& v, __half2 acc) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const __half2 zero = __float2half2_rn(0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __hfma2(h[i], zero, acc);
  return acc;
}
__device__ __forceinline__ __nv_bfloat162 fold_finite(const uint4& v, __nv_bfloat162 acc) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __hfma2(h[i], zero, acc);
  return acc;
}

template <typename C>
struct PairOf;
template <>
struct PairOf<__half> {
  using type = __half2;
  static constexpr uint32_t kExponent = 0x7c00u;
};
template <>
struct PairOf<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static constexpr uint32_t kExponent = 0x7f80u;
};

// Weights P = 2^(s - m) go to the second product in the cache's 16-bit type.  f16
// ends at 2^-24: against a row's maximum, 60000 weights just below 2^-25 would
// all vanish, 0.2 per cent of the row beside one key that outweighs the rest.
// So for f16 the reference m lies kLift (log2 units) below the maximum, and P
// uses the type's upper range as well; sums and outputs carry the same factor,
// which the quotient drops.  bf16 reaches as far as fp32.  (Not for maxima so
// large that the difference would round, up to a P past 65504.)
constexpr float kLift = 7.f;
constexpr float kFar = 1048576.f;  // 2^20: fp32's steps are an eighth there

template <typename C>
__device__ __forceinline__ float lifted(float maximum) {
  if constexpr (PairOf<C>::kExponent != 0x7c00u) return maximum;
  return maximum - (fabsf(maximum) < kFar ? kLift : 0.f);
}

template <typename C>
__device__ __forceinline__ bool not_finite(C v) {
  const uint32_t w = *reinterpret_cast<const uint16_t*>(&v);
  return (w & PairOf<C>::kExponent) == PairOf<C>::kExponent;
}

// Whether n chunks of 16 bytes in shared memory are finite throughout; a
// warp's lanes share them and the answer.
template <typename C>
__device__ __forceinline__ bool all_finite(const uint8_t* chunks, int n, int lane) {
  typename PairOf<C>::type acc[2];
  *reinterpret_cast<uint2*>(acc) = make_uint2(0u, 0u);
  const uint4* at = reinterpret_cast<const uint4*>(chunks);
  int i = lane;
#pragma unroll 1
  for (; i + 7 * 32 < n; i += 8 * 32) {
    uint4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at[i + 32 * j];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j & 1] = fold_finite(v[j], acc[j & 1]);
  }
#pragma unroll 1
  for (; i < n; i += 32) acc[0] = fold_finite(at[i], acc[0]);
  // 0 or -0 in both halves of both.
  const uint2 w = *reinterpret_cast<const uint2*>(acc);
  return __all_sync(0xffffffffu, ((w.x | w.y) & 0x7fff7fffu) == 0u);
}

// Zeros in place of those that are not finite.
template <typename C>
__device__ __forceinline__ void clear_not_finite(uint8_t* chunks, int n, int lane) {
#pragma unroll 1
  for (int i = lane; i < n; i += 32) {
    uint4* at = reinterpret_cast<uint4*>(chunks) + i;
    uint4 v = *at;
    C* c = reinterpret_cast<C*>(&v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (not_finite(c[j])) *reinterpret_cast<uint16_t*>(&c[j]) = 0;
    *at = v;
  }
}

// Queries of bf16 for products in f16, which ends at 65504 and below 2^-14 has
// steps of 2^-24: a row with larger values, or with none of kSmallQuery or more,
// goes to the product times a power of two that brings its largest value to 2^15,
// and its scores get the inverse back with the scale (exact both ways; what is
// 2^-39 of the row's largest may be rounded).  A caller's scale, or an 8-bit
// cache's, can make ordinary scores of such rows.  Other rows are converted as
// they are: their values are off by at most 2^-25, which is 2^-21 of the largest.
//
// The largest magnitude, as bf16 bits, of two packed values.
__device__ __forceinline__ uint32_t magnitude(uint32_t w, uint32_t most) {
  return max(most, max(w & 0x7fffu, w >> 16 & 0x7fffu));
}
constexpr int kSmallQuery = 127 - 4;  // exponent of 2^-4 in bf16
__device__ __forceinline__ bool outside_f16(uint32_t most) {
  return (int)(most >> 7) > 127 + 15 || (most != 0u && (int)(most >> 7) < kSmallQuery);
}
// The power by which a row of that magnitude must be divided (0: by none), not
// below `least` (power_floor).
__device__ __forceinline__ int beyond_f16(uint32_t most, int least) {
  return outside_f16(most) ? max((int)(most >> 7) - (127 + 15), least) : 0;
}
// The least power whose product with the scale is a normal number; 2^120 makes
// f16 numbers of all bf16 ones that are smaller than 2^-105 (multiples of 2^-133).
inline int power_floor(float scale_log2) {
  int exponent;
  frexpf(scale_log2, &exponent);
  const int least = -125 - exponent;
  return least < -120 ? -120 : least > 0 ? 0 : least;
}
// 2^n, n in [-126, 127].
__device__ __forceinline__ float power2(int n) { return __uint_as_float((uint32_t)(127 + n) << 23); }

}  // namespace tf
