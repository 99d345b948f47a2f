// Codes of an 8-bit cache to f16 numbers, for requests with many rows: the
// tensor-core kernel reads a tile once for every 256 of them.
//
// A block takes one page of one key head, keys and values: reads a byte a code,
// writes two (without rounding), and lays the scales out by head and block, as
// they are read.  Slots past the request's length become zeros, and so do pages
// that do not exist.  What bounds it: these bytes.
//
// Measured: 16384 tokens of 8 key heads of 128 (101 MB) 20 us of a call; 8 x 2048
// tokens of 16 heads (201 MB) 35.
#include "common.cuh"
#include "paged.h"
#include "paged_codes.cuh"

namespace tf {

namespace {

constexpr int kThreads = 256;

struct WidenParams {
  const uint8_t* codes[2];
  const float* scales[2];
  uint8_t* to[2];
  float* to_scales[2];
  int64_t pages, page_stride, scale_stride, blocks;
  tf_page_table table;
  int kv_heads, page_size, head_dim;
  const WidenedRequest* list;
  int requests;
};

// One whole 32-byte sector.
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
               "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

template <typename S>
__global__ void __launch_bounds__(kThreads) paged_widen_kernel(const __grid_constant__ WidenParams p) {
  const int page = blockIdx.x, head = blockIdx.y;
  // The last request that begins at or before the page.
  int lo = 0, hi = p.requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.list[mid].first_page <= page)
      lo = mid;
    else
      hi = mid;
  }
  const WidenedRequest r = p.list[lo];
  const int column = page - r.first_page;
  int64_t id = column < p.table.columns ? p.table.ids[r.request * p.table.stride + column] : -1;
  if (id >= p.pages) id = -1;
  const int have = id < 0 ? 0 : min(p.page_size, r.kv_len - column * p.page_size);  // tokens
  const int row = p.head_dim / 16;                                                  // vectors of a token
  const int vectors = p.page_size * row;
  const int64_t from = id * p.page_stride + (int64_t)head * p.page_size * p.head_dim;
  const int64_t to = ((int64_t)page * p.kv_heads + head) * p.page_size * p.head_dim * 2;
  // Four vectors of a thread are under way at a time.
  constexpr int kBatch = 4;
  for (int i0 = threadIdx.x; i0 < 2 * vectors; i0 += kBatch * kThreads) {
    uint4 w[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * kThreads, side = i >= vectors, at = side ? i - vectors : i;
      w[k] = make_uint4(0, 0, 0, 0);
      if (i < 2 * vectors && at / row < have) w[k] = ld_stream_v4(p.codes[side] + from + 16 * at);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * kThreads, side = i >= vectors, at = side ? i - vectors : i;
      if (i >= 2 * vectors) break;
      uint4 a, b;
      Code<S>::widen(w[k].x, a.x, a.y);
      Code<S>::widen(w[k].y, a.z, a.w);
      Code<S>::widen(w[k].z, b.x, b.y);
      Code<S>::widen(w[k].w, b.z, b.w);
      store32(p.to[side] + to + 32 * at, a, b);
    }
  }
  const int blocks = p.page_size / kScaleTokens;
  if (threadIdx.x < 2 * blocks) {
    const int side = threadIdx.x >= blocks, b = threadIdx.x % blocks;
    float scale = 0.f;
    if (b * kScaleTokens < have) scale = p.scales[side][id * p.scale_stride + head * blocks + b];
    p.to_scales[side][head * p.blocks + (int64_t)page * blocks + b] = scale;
  }
}

}  // namespace

tf_status launch_paged_widen(const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  if (plan.widened_pages == 0) return TF_OK;
  const WidenedPages w(a);
  WidenParams p{};
  p.codes[0] = static_cast<const uint8_t*>(a.kv.k);
  p.codes[1] = static_cast<const uint8_t*>(a.kv.v);
  p.scales[0] = a.scales.k;
  p.scales[1] = a.scales.v;
  p.to[0] = static_cast<uint8_t*>(w.kv.k);
  p.to[1] = static_cast<uint8_t*>(w.kv.v);
  p.to_scales[0] = w.k_scales;
  p.to_scales[1] = w.v_scales;
  p.pages = a.kv.pages;
  p.page_stride = a.kv.page_stride;
  p.scale_stride = a.scales.page_stride;
  p.blocks = w.blocks;
  p.table = a.table;
  p.kv_heads = plan.kv_heads;
  p.page_size = plan.page_size;
  p.head_dim = plan.head_dim;
  p.list = w.list;
  p.requests = plan.widened_requests;
  if (plan.widened_pages > 2147483647LL) return set_error(TF_ERR_UNSUPPORTED, "paged_attention: too many pages");
  const dim3 grid((unsigned)plan.widened_pages, (unsigned)plan.kv_heads);
  if (a.kv.dtype == TF_DTYPE_I8)
    paged_widen_kernel<I8><<<grid, kThreads, 0, s>>>(p);
  else
    paged_widen_kernel<E4M3><<<grid, kThreads, 0, s>>>(p);
  return check_launch("paged_widen");
}

}  // namespace tf
