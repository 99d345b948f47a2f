// Copies of pages inside caches: dst page of a pair = src page, in every layer
// and every array of a call (codes and scales, keys and values together).
//
// What bounds it: each byte is read once and written once.  A block copies up
// to 16 KB of one page of one layer, four 16-byte vectors a thread, all loaded
// before the first is stored; eight such blocks on an SM keep 128 KB in flight.
// Pages below 4 KB (scales) go a warp each.  The pairs travel with the launch,
// so a call uploads nothing, waits for nothing and can be captured.
//
// Measured: 301 pages of 128 KB in 8 layers, keys and values (1.26 GB moved) 190 us,
// 6.65 TB/s; 3 pages of 32 KB in 16 layers 3.1 us.
#include <string.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "common.cuh"
#include "internal.h"

namespace tf {

namespace {

constexpr int kThreads = 256;
constexpr int kVectors = 4;                           // of a thread
constexpr int kChunk = kThreads * kVectors * 16;      // bytes of a block
constexpr int kSmallPage = 4096;                      // up to here a warp copies a page
constexpr int kMaxArrays = TF_MAX_COPY_ARRAYS;

struct CopyArray {
  char* base;
  int64_t layer_stride, page_stride, page_bytes;
  int64_t first;   // block of the grid
  int64_t chunks;  // blocks of a page; 0: a warp a page
  int width;       // bytes of an access
};

template <int N>
struct CopyParams {
  CopyArray arrays[kMaxArrays];
  int count;
  int layers;
  int pairs;
  int32_t src[N], dst[N];
};

template <typename V>
__device__ __forceinline__ void copy_span(char* to, const char* from, int64_t bytes, int at, int step) {
  V* d = reinterpret_cast<V*>(to);
  const V* s = reinterpret_cast<const V*>(from);
  const int64_t n = bytes / (int64_t)sizeof(V);
  for (int64_t i = at; i < n; i += kVectors * step) {
    V v[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
      if (i + k * step < n) v[k] = __ldcs(s + i + k * step);
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
      if (i + k * step < n) __stcs(d + i + k * step, v[k]);
  }
}
__device__ __forceinline__ void copy_span(char* to, const char* from, int64_t bytes, int at, int step, int width) {
  if (width == 16)
    copy_span<uint4>(to, from, bytes, at, step);
  else if (width == 4)
    copy_span<uint32_t>(to, from, bytes, at, step);
  else
    copy_span<uint8_t>(to, from, bytes, at, step);
}

template <int N>
__global__ void __launch_bounds__(kThreads) paged_copy_kernel(const __grid_constant__ CopyParams<N> p) {
  int a = 0;
  while (a + 1 < p.count && blockIdx.x >= p.arrays[a + 1].first) ++a;
  const CopyArray& array = p.arrays[a];
  const int64_t block = blockIdx.x - array.first;
  int64_t item = block, from = 0, bytes = array.page_bytes;  // item = layer * pairs + pair
  int at = threadIdx.x, step = kThreads;
  if (array.chunks) {
    item = block / array.chunks;
    from = block % array.chunks * kChunk;
    bytes = min(array.page_bytes - from, (int64_t)kChunk);
  } else {
    item = block * (kThreads / 32) + (threadIdx.x >> 5);
    if (item >= (int64_t)p.layers * p.pairs) return;
    at = threadIdx.x & 31;
    step = 32;
  }
  const int64_t layer = item / p.pairs;
  const int pair = (int)(item % p.pairs);
  char* base = array.base + layer * array.layer_stride + from;
  copy_span(base + p.dst[pair] * array.page_stride, base + p.src[pair] * array.page_stride, bytes, at, step,
            array.width);
}

template <int N>
tf_status launch(const tf_copy_array* arrays, int count, int layers, const std::vector<int32_t>& src,
                 const std::vector<int32_t>& dst, size_t from, cudaStream_t s) {
  static CopyParams<N> zero;
  CopyParams<N> p = zero;
  p.count = count;
  p.layers = layers;
  p.pairs = (int)std::min<size_t>(N, src.size() - from);
  memcpy(p.src, src.data() + from, p.pairs * sizeof(int32_t));
  memcpy(p.dst, dst.data() + from, p.pairs * sizeof(int32_t));
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    const tf_copy_array& t = arrays[i];
    const uint64_t bits = reinterpret_cast<uintptr_t>(t.base) | (uint64_t)t.layer_stride | (uint64_t)t.page_stride |
                          (uint64_t)t.page_bytes;
    CopyArray& o = p.arrays[i];
    o = {static_cast<char*>(t.base), t.layer_stride, t.page_stride, t.page_bytes, blocks, 0,
         bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1};
    const int64_t items = (int64_t)layers * p.pairs;
    if (t.page_bytes > kSmallPage) {
      o.chunks = (t.page_bytes + kChunk - 1) / kChunk;
      blocks += items * o.chunks;
    } else {
      blocks += (items + kThreads / 32 - 1) / (kThreads / 32);
    }
  }
  if (blocks > 2147483647LL) return set_error(TF_ERR_UNSUPPORTED, "paged_copy: too much for one call");
  paged_copy_kernel<N><<<(unsigned)blocks, kThreads, 0, s>>>(p);
  return check_launch("paged_copy");
}

}  // namespace

tf_status launch_paged_copy(const tf_copy_array* arrays, int count, int layers, int64_t pages, const int32_t* src,
                            const int32_t* dst, int64_t pairs, cudaStream_t s) {
  std::vector<int32_t> from, to;
  try {
    for (int64_t i = 0; i < pairs; ++i) {
      if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
        return set_error(TF_ERR_INVALID_ARGUMENT, "paged_copy: pair %lld (%d to %d) outside the %lld pages",
                         (long long)i, src[i], dst[i], (long long)pages);
      if (src[i] == dst[i]) continue;
      from.push_back(src[i]);
      to.push_back(dst[i]);
    }
    // No page may be written twice, or written and read: the copies run in any order.
    std::vector<int32_t> written(to), read(from);
    std::sort(written.begin(), written.end());
    std::sort(read.begin(), read.end());
    const auto twice = std::adjacent_find(written.begin(), written.end());
    if (twice != written.end())
      return set_error(TF_ERR_INVALID_ARGUMENT, "paged_copy: page %d is written twice", *twice);
    for (size_t i = 0, j = 0; i < written.size(); ++i) {
      while (j < read.size() && read[j] < written[i]) ++j;
      if (j < read.size() && read[j] == written[i])
        return set_error(TF_ERR_INVALID_ARGUMENT, "paged_copy: page %d is read and written", written[i]);
    }
  } catch (const std::exception&) {
    return set_error(TF_ERR_OUT_OF_MEMORY, "paged_copy: out of host memory");
  }
  if (layers == 0 || count == 0) return TF_OK;
  // Few pairs with a small launch, many with as many as a launch takes along.
  constexpr int kFew = 32, kMany = 480;
  for (size_t at = 0; at < from.size(); at += kMany)
    TF_TRY(from.size() <= kFew ? launch<kFew>(arrays, count, layers, from, to, at, s)
                               : launch<kMany>(arrays, count, layers, from, to, at, s));
  return TF_OK;
}

}  // namespace tf
