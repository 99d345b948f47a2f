// New tokens into a paged key/value cache: full-width RMSNorm of q and k,
// rotation by halves, append.
//
//   q, k:  x' = x * rsqrt(mean(x^2) + eps) * w   over the row's whole width
//   pair (a, b) = (x'[d], x'[d + D/2]) of a head, angle t = pos * theta^(-2d/D):
//          (a cos t - b sin t, a sin t + b cos t)
//   v:     copied
//
// What bounds it: each value is read once and written once; the only other
// traffic is the norm weights, from L2.  A unit is one row's q, k or v part,
// taken by as many warps as hold it in registers at 32 values a thread, so
// that a row is read once for the norm and the rotation alike, and its loads
// are all in flight while the angles are computed.  A thread holds 8 values of
// a head's first half together with their rotation partners in the second, and
// works on packed fp32 pairs: with the partners in another lane the shuffles
// and selects took 190 instructions for 8 values, and issue was the limit.
//
// The angle is reduced in double precision (t / 2 pi, less its nearest whole
// number) before the fp32 sine and cosine: in fp32 a position of 10^5 would
// leave it off by up to 6e-3 radians.  The block's threads share the D/2
// angles of each of its rows through shared memory: one sine and cosine for
// each thread where every thread would else compute eight.
//
// fp32 throughout, one rounding at the end: the rotated k is rounded straight
// to the cache's type.
//
// Measured, L2 flushed: 16384 rows of 16 + 2 x 16 heads of 128 with norms and
// rotation 82 us, 4.9 TB/s (without either 70: the latency of a block's one
// pass, not the arithmetic, is what is left); 64 rows 3.9 us in a warm L2.  At
// most 64 registers a thread: 82 us, without the cap 86 to 90; blocks of 4
// warps where a row's parts fit them: 84 us, of 8 86, of 16 96; the norm
// weights fetched before the sum is known: 84 -> 82; 64 values a thread instead
// of 32: 92 against 88.
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "paged.h"

namespace tf {

namespace {

constexpr int kPairs = 2;  // pairs of 16-byte chunks (a head's halves) a thread holds

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

struct AppendParams {
  const void* qkv;
  int64_t qkv_stride;
  int64_t rows;
  int heads, kv_heads;
  const __half* q_norm;
  const __half* k_norm;
  float eps;
  const int32_t* positions;
  const int32_t* requests;
  tf_page_table table;
  void* k;
  void* v;
  int64_t pages, page_stride;
  int page_size, page_shift;
  void* q_out;
  unsigned q_blocks, k_blocks;  // blocks of the q units, then of the k units, then of the v units
  int q_shift, kv_shift;        // log2 of the warps of a unit
  int rotate;
  double turns[64];             // theta^(-2d/D) / (2 pi)
};

template <typename T, typename C, int D>
__global__ void __launch_bounds__(512, 2) paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kHalfChunks = D / 16;  // chunks of half a head
  __shared__ float rot[2][16][D / 2];  // cos and sin for each of the block's rows
  __shared__ float total[16];          // warp sums of squares
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = blockIdx.x < p.q_blocks ? 0 : blockIdx.x < p.q_blocks + p.k_blocks ? 1 : 2;
  const unsigned block = blockIdx.x - (part == 0 ? 0u : part == 1 ? p.q_blocks : p.q_blocks + p.k_blocks);
  const int shift = part == 0 ? p.q_shift : p.kv_shift;
  const int warps = 1 << shift;  // of a unit
  const int heads = part == 0 ? p.heads : p.kv_heads;
  const int units = (int)(blockDim.x >> 5) >> shift;  // rows of this block
  const int unit = warp >> shift;
  const int64_t row = (int64_t)block * units + unit;
  const bool live = row < p.rows;
  // This thread's pairs: first-half chunk `at` of heads head0, head0 + step.
  const int index = (warp & (warps - 1)) * 32 + lane;
  const int at = index % kHalfChunks, head0 = index / kHalfChunks, step = 32 * warps / kHalfChunks;

  const T* src = static_cast<const T*>(p.qkv) + (live ? row : 0) * p.qkv_stride +
                 (int64_t)(part == 0 ? 0 : part == 1 ? p.heads : p.heads + p.kv_heads) * D + 8 * at;
  uint4 raw[kPairs][2];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int h = head0 + step * i;
    const bool mine = live && h < heads;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      raw[i][j] = mine ? ld_stream_v4(src + h * D + j * (D / 2)) : make_uint4(0, 0, 0, 0);
  }
  // Where the row goes.  A row whose slot does not exist is not stored.
  C* dst = nullptr;
  if (part != 0 && live) {
    const int pos = p.positions[row], req = p.requests[row];
    const int column = pos >> p.page_shift;
    if (pos >= 0 && req >= 0 && req < p.table.requests && column < p.table.columns) {
      const int64_t page = p.table.ids[req * p.table.stride + column];
      if (page >= 0 && page < p.pages)
        dst = static_cast<C*>(part == 1 ? p.k : p.v) + page * p.page_stride + (int64_t)(pos & (p.page_size - 1)) * D;
    }
  }
  const __half* norm = part == 0 ? p.q_norm : part == 1 ? p.k_norm : nullptr;
  const bool rotate = p.rotate && part < 2;
  uint4 weight[kPairs][2];  // on their way during the angles and the sum
  if (norm) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (head0 + step * i < heads) weight[i][j] = ld_v4(norm + (head0 + step * i) * D + j * (D / 2) + 8 * at);
  }
  if (rotate) {
    for (int i = tid; i < units * (D / 2); i += (int)blockDim.x) {
      const int64_t r = (int64_t)block * units + i / (D / 2);
      if (r < p.rows) {
        const double t = (double)p.positions[r] * p.turns[i % (D / 2)];
        float sn, cs;
        sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
        rot[0][i / (D / 2)][i % (D / 2)] = cs;
        rot[1][i / (D / 2)][i % (D / 2)] = sn;
      }
    }
  }
  if (norm) {
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float2 f[4];
        unpack4<T>(raw[i][j], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum = fma2(f[k], f[k], sum);
      }
    const float all = warp_sum_butterfly(sum.x + sum.y);
    if (lane == 0) total[warp] = all;
  }
  if (norm || rotate) __syncthreads();
  float2 scale = make_float2(1.f, 1.f);
  if (norm) {
    float sum = 0.f;
    for (int w = 0; w < warps; ++w) sum += total[unit * warps + w];
    scale.x = scale.y = rms_scale(sum, heads * D, p.eps);
  }
  float2 cs[4], sn[4];
  if (rotate) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      cs[k] = *reinterpret_cast<const float2*>(&rot[0][unit][8 * at + 2 * k]);
      sn[k] = *reinterpret_cast<const float2*>(&rot[1][unit][8 * at + 2 * k]);
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int h = head0 + step * i;
    if (!live || h >= heads) continue;
    float2 f[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unpack4<T>(raw[i][j], f[j]);
      if (norm) {
        float2 w[4];
        unpack4<__half>(weight[i][j], w);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[j][k] = mul2(mul2(f[j][k], scale), w[k]);
      }
    }
    if (rotate) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 a = f[0][k], b = f[1][k];
        const float2 minus = make_float2(-sn[k].x, -sn[k].y);
        f[0][k] = fma2(a, cs[k], mul2(b, minus));
        f[1][k] = fma2(a, sn[k], mul2(b, cs[k]));
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (part == 0)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + (row * heads + h) * D + j * (D / 2) + 8 * at) =
            pack4<T>(f[j]);
      else if (dst)
        *reinterpret_cast<uint4*>(dst + (int64_t)h * p.page_size * D + j * (D / 2) + 8 * at) = pack4<C>(f[j]);
    }
  }
}

// log2 of the warps (1 to 16) that hold `width` values at kPairs pairs of
// chunks a thread.
int unit_shift(int width) {
  int s = 0;
  while ((32 << s) * kPairs * 16 < width) ++s;
  return s;
}

}  // namespace

tf_status launch_paged_append(const AppendArgs& a, cudaStream_t s) {
  if (a.rows == 0) return TF_OK;
  const int D = a.kv.head_dim;
  AppendParams p;
  memset(&p, 0, sizeof(p));
  p.qkv = a.qkv;
  p.qkv_stride = a.qkv_stride;
  p.rows = a.rows;
  p.heads = a.heads;
  p.kv_heads = a.kv.kv_heads;
  p.q_norm = static_cast<const __half*>(a.q_norm);
  p.k_norm = static_cast<const __half*>(a.k_norm);
  p.eps = a.eps;
  p.positions = a.positions;
  p.requests = a.requests;
  p.table = a.table;
  p.k = a.kv.k;
  p.v = a.kv.v;
  p.pages = a.kv.pages;
  p.page_stride = a.kv.page_stride;
  p.page_size = a.kv.page_size;
  p.q_out = a.q_out;
  p.rotate = a.theta != 0.f;
  if (p.rotate) {
    // One power, then products: 63 roundings of 2^-53 stay far below fp32.
    const double step = pow((double)a.theta, -2.0 / D);
    double f = 0.15915494309189535;  // 1 / (2 pi)
    for (int d = 0; d < D / 2; ++d, f *= step) p.turns[d] = f;
  }
  while ((1 << p.page_shift) < a.kv.page_size) ++p.page_shift;
  p.q_shift = unit_shift(a.heads * D);
  p.kv_shift = unit_shift(a.kv.kv_heads * D);
  const int warps = p.q_shift > 2 ? 1 << p.q_shift : 4;  // per block
  const int q_rows = warps >> p.q_shift, kv_rows = warps >> p.kv_shift;
  const int64_t qb = (a.rows + q_rows - 1) / q_rows;
  const int64_t kb = (a.rows + kv_rows - 1) / kv_rows;
  if (qb + 2 * kb > 2147483647LL) return set_error(TF_ERR_UNSUPPORTED, "paged_append: too many rows");
  p.q_blocks = (unsigned)qb;
  p.k_blocks = (unsigned)kb;
  const unsigned grid = (unsigned)(qb + 2 * kb);
#define TF_APPEND(T, C)                                                        \
  do {                                                                         \
    if (D == 128)                                                              \
      paged_append_kernel<T, C, 128><<<grid, 32 * warps, 0, s>>>(p);           \
    else                                                                       \
      paged_append_kernel<T, C, 64><<<grid, 32 * warps, 0, s>>>(p);            \
    return check_launch("paged_append");                                       \
  } while (0)
  if (a.act == TF_DTYPE_F16) TF_APPEND(__half, __half);
  if (a.kv.dtype == TF_DTYPE_F16) TF_APPEND(__nv_bfloat16, __half);
  TF_APPEND(__nv_bfloat16, __nv_bfloat16);
#undef TF_APPEND
}

}  // namespace tf
