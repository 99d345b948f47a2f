// Codes of an 8-bit cache: the storage types I8 and E4M3, narrowing and widening,
// the reference of value scales, and what both attention kernels fetch codes with.
// Both types widen to f16 without rounding (integers up to 127; e4m3 has 4 bits of
// precision and magnitudes from 2^-9 to 448).
#pragma once

#include <cuda.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "paged_pairs.cuh"
#include "tc_ptx.cuh"

namespace tf {

struct I8 {
  uint8_t bits;
};
struct E4M3 {
  uint8_t bits;
};

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }

template <typename S>
struct Code;

// Division by a block's scale, given with its rounded reciprocal: the quotient
// once improved by its remainder, so that a value that lies halfway between two
// codes is not moved off it (16-bit values over a scale of few bits often do).
// A scale that has no reciprocal gives zeros.
struct Divisor {
  float2 by, inverse;
  __device__ __forceinline__ explicit Divisor(float scale) {
    const float r = scale > 0.f && scale < INFINITY ? __fdiv_rn(1.f, scale) : 0.f;
    by = make_float2(-scale, -scale);
    inverse = make_float2(r, r);
  }
  __device__ __forceinline__ float2 operator()(float2 x) const {
    const float2 y = mul2(x, inverse);
    return fma2(fma2(y, by, x), inverse, y);
  }
};

// 2^x down to 2^-149.
__device__ __forceinline__ float exp2_far(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The reference r of value scales: a power of two at or above those that are finite
// (2^-126 .. 2^126; beyond that, near them).  Ratios s_v / r down to 2^-61 are worked
// with as they are; below that (or at zero, which has no logarithm) scales count as
// far apart.  So they do below 2^-13 where scores are so far out (kFar) that a row's
// reference cannot take in log2(s_v / r): the ratio itself then has to leave a weight
// f16's 11 bits.
constexpr float kLeastRef = 1.17549435e-38f, kLeastInverse = 8.50705917e37f;  // 2^-126, 2^126
constexpr float kLeastRatio = 4.33680869e-19f;                                // 2^-61
constexpr float kFarRatio = 1.220703125e-4f;                                  // 2^-13
__device__ __forceinline__ float power_above(float v) {
  return __uint_as_float(min((__float_as_uint(v) + 0x7fffffu) & 0x7f800000u, 0x7e800000u));
}
__device__ __forceinline__ float inverse_of(float power) { return __uint_as_float(0x7f000000u - __float_as_uint(power)); }
__device__ __forceinline__ float exponent_of(float power) { return (float)((int)(__float_as_uint(power) >> 23) - 127); }
__device__ __forceinline__ bool far_apart(float lowest, float ref) { return lowest < ref * kLeastRatio || lowest == 0.f; }

template <>
struct Code<I8> {
  static constexpr tf_dtype kDtype = TF_DTYPE_I8;
  static constexpr float kLargest = 127.f;
  // A byte c + 128 under 0x64 is the f16 number 1024 + 128 + c.
  __device__ __forceinline__ static uint32_t lift(uint32_t biased, uint32_t select) {
    return half2_bits(__hsub2(bits_half2(__byte_perm(biased, 0x64646464u, select)), bits_half2(0x64806480u)));
  }
  // Four codes -> f16 pairs (0, 1) and (2, 3).
  __device__ __forceinline__ static void widen(uint32_t w, uint32_t& a, uint32_t& b) {
    const uint32_t u = w ^ 0x80808080u;
    a = lift(u, 0x4140);
    b = lift(u, 0x4342);
  }
  // Four codes -> f16 pairs (0, 2) and (1, 3).
  __device__ __forceinline__ static void widen_cross(uint32_t w, uint32_t& a, uint32_t& b) {
    const uint32_t u = w ^ 0x80808080u;
    a = lift(u, 0x4240);
    b = lift(u, 0x4341);
  }
  // Four values within 127.5 -> codes, the first in the lowest byte.  Added to
  // 1.5 * 2^23 a number is rounded to the nearest integer, whose lowest byte is the
  // code.
  __device__ __forceinline__ static uint32_t narrow(float2 x, float2 y) {
    const float2 one = make_float2(1.f, 1.f), magic = make_float2(12582912.f, 12582912.f);
    x = fma2(x, one, magic);
    y = fma2(y, one, magic);
    const uint32_t lo = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
};

template <>
struct Code<E4M3> {
  static constexpr tf_dtype kDtype = TF_DTYPE_E4M3;
  static constexpr float kLargest = 448.f;
  __device__ __forceinline__ static void widen(uint32_t w, uint32_t& a, uint32_t& b) {
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "mov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
  }
  __device__ __forceinline__ static void widen_cross(uint32_t w, uint32_t& a, uint32_t& b) {
    widen(__byte_perm(w, 0, 0x3120), a, b);
  }
  __device__ __forceinline__ static uint32_t narrow(float2 x, float2 y) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
    return __byte_perm(lo, hi, 0x5410);
  }
};

// `row` .. of a page of codes, all columns.
__device__ __forceinline__ void tma_codes(void* dst, const CUtensorMap* map, int row, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          tc::smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(page), "r"(tc::smem_addr(bar))
      : "memory");
}
// One value, or zero, into shared memory; the barrier's phase waits for the
// copies that a thread has begun before it arrives.
__device__ __forceinline__ void copy_value(float* dst, const float* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(tc::smem_addr(dst)), "l"(src), "r"(real ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void arrive_with_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_addr(bar)) : "memory");
}

}  // namespace tf
