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
// are all in flight while the angles are computed.  Chunk c (8 values) of a
// head and its rotation partner c ^ (D/16) sit in lanes of the same warp.
//
// The angle is reduced in double precision (t / 2 pi, less its nearest whole
// number) before the fp32 sine and cosine: in fp32 a position of 10^5 would
// leave it off by up to 6e-3 radians.  The block's threads share the D/2
// angles of each of its rows through shared memory: one sine and cosine for
// each thread where every thread would else compute eight.
//
// fp32 throughout, one rounding at the end: the rotated k is rounded straight
// to the cache's type.
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "paged.h"

namespace tf {

namespace {

constexpr int kChunks = 4;  // 16-byte chunks a thread holds

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
  int page_size;
  void* q_out;
  unsigned q_blocks, k_blocks;  // blocks of the q units, then of the k units, then of the v units
  int q_warps, kv_warps;        // warps of a unit
  int rotate;
  double turns[64];             // theta^(-2d/D) / (2 pi)
};

template <typename T, typename C, int D>
__global__ void __launch_bounds__(512) paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kHeadChunks = D / 8;
  __shared__ float2 rot[16][D / 2];  // (cos, sin) for each of the block's rows
  __shared__ float total[16];        // warp sums of squares
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = blockIdx.x < p.q_blocks ? 0 : blockIdx.x < p.q_blocks + p.k_blocks ? 1 : 2;
  const unsigned block = blockIdx.x - (part == 0 ? 0u : part == 1 ? p.q_blocks : p.q_blocks + p.k_blocks);
  const int warps = part == 0 ? p.q_warps : p.kv_warps;
  const int heads = part == 0 ? p.heads : p.kv_heads;
  const int units = (int)(blockDim.x >> 5) / warps;  // rows of this block
  const int unit = warp / warps;
  const int64_t row = (int64_t)block * units + unit;
  const bool live = row < p.rows;
  const int W = heads * D;
  const int c0 = (warp % warps) * 32 + lane;  // this thread's chunks: c0 + 32 * warps * i

  const T* src = static_cast<const T*>(p.qkv) + (live ? row : 0) * p.qkv_stride +
                 (int64_t)(part == 0 ? 0 : part == 1 ? p.heads : p.heads + p.kv_heads) * D;
  uint4 raw[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = c0 + 32 * warps * i;
    raw[i] = live && 8 * c < W ? ld_stream_v4(src + 8 * c) : make_uint4(0, 0, 0, 0);
  }
  const __half* norm = part == 0 ? p.q_norm : part == 1 ? p.k_norm : nullptr;
  const bool rotate = p.rotate && part < 2;
  if (rotate) {
    for (int i = tid; i < units * (D / 2); i += (int)blockDim.x) {
      const int64_t r = (int64_t)block * units + i / (D / 2);
      if (r < p.rows) {
        const double t = (double)p.positions[r] * p.turns[i % (D / 2)];
        float sn, cs;
        sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
        rot[i / (D / 2)][i % (D / 2)] = make_float2(cs, sn);
      }
    }
  }
  float scale = 1.f;
  if (norm) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float f[8];
      unpack8<T>(raw[i], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(f[j], f[j], sum);
    }
    sum = warp_sum_butterfly(sum);
    if (lane == 0) total[warp] = sum;
  }
  __syncthreads();
  if (norm) {
    float sum = 0.f;
    for (int w = 0; w < warps; ++w) sum += total[unit * warps + w];
    scale = rms_scale(sum, W, p.eps);
  }
  // Where the row goes.  A row whose slot does not exist is not stored.
  T* q_row = nullptr;
  C* dst = nullptr;
  if (part == 0) {
    q_row = static_cast<T*>(p.q_out) + row * W;
  } else if (live) {
    const int pos = p.positions[row], req = p.requests[row];
    const int column = pos / p.page_size;
    if (pos >= 0 && req >= 0 && req < p.table.requests && column < p.table.columns) {
      const int64_t page = p.table.ids[req * p.table.stride + column];
      if (page >= 0 && page < p.pages)
        dst = static_cast<C*>(part == 1 ? p.k : p.v) + page * p.page_stride + (int64_t)(pos % p.page_size) * D;
    }
  }
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = c0 + 32 * warps * i;
    const bool mine = live && 8 * c < W;
    float f[8];
    unpack8<T>(raw[i], f);
    if (norm) {
      float w[8];
      unpack8<__half>(mine ? ld_v4(norm + 8 * c) : make_uint4(0, 0, 0, 0), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * scale * w[j];
    }
    if (rotate) {
      const bool first = (c % kHeadChunks) < kHeadChunks / 2;
      const float2* cs = &rot[unit][(c % (kHeadChunks / 2)) * 8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float other = __shfl_xor_sync(0xffffffffu, f[j], kHeadChunks / 2);
        const float2 r = cs[j];
        f[j] = first ? f[j] * r.x - other * r.y : other * r.y + f[j] * r.x;
      }
    }
    if (!mine) continue;
    if (part == 0) {
      *reinterpret_cast<uint4*>(q_row + 8 * c) = pack8<T>(f);
    } else if (dst) {
      const int h = c / kHeadChunks, d0 = (c % kHeadChunks) * 8;
      *reinterpret_cast<uint4*>(dst + (int64_t)h * p.page_size * D + d0) = pack8<C>(f);
    }
  }
}

// Warps that hold `width` values at kChunks chunks a thread: 1, 2, 4, 8 or 16.
int unit_warps(int width) {
  int w = 1;
  while (w * 32 * kChunks * 8 < width) w *= 2;
  return w;
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
  p.q_warps = unit_warps(a.heads * D);
  p.kv_warps = unit_warps(a.kv.kv_heads * D);
  const int warps = p.q_warps > 8 ? p.q_warps : 8;  // per block
  const int64_t qb = (a.rows + warps / p.q_warps - 1) / (warps / p.q_warps);
  const int64_t kb = (a.rows + warps / p.kv_warps - 1) / (warps / p.kv_warps);
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
