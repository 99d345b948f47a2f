// Paged attention for few packed rows per key head (single tokens, grouped
// heads, short drafts): a memory-bound stream over the pages.
//
// out = softmax(q K^T * scale) V by one pass over the keys with a running
// maximum m and sum l per row: a tile of scores s gives
//   m' = max(m, max s),  O = O * 2^(m - m') + 2^(s - m') V,  l likewise,
// in log2 units (scale * log2(e) folded into the scores' FMA).
//
// What bounds it: every key and value is read once (512 bytes per token and
// key head at head_dim 128), so HBM is the bound and the products only have to
// keep out of the way.  mma.sync m16n8k16 serves them from registers: a tcgen05
// tile has 128 rows of which at most 16 would be filled.  Its products are slow
// here (some 32 clocks each), so keys take the 16-row side and the queries the
// 8-column side:
//   S^T = K Q^T,  O^T = V^T P^T      (K, V^T by ldmatrix, P^T by movmatrix)
// Up to 8 packed rows then need half the products of 16 (kernel variants for
// one and two 8-row groups), and 32 keys take less time than their bytes.
//
// One block of four warps per SM walks its segments (paged.h).  The warps take
// the segment's 32-key tiles in turn and never wait for one another inside a
// segment: each has a ring of its own that lane-parallel TMA copies keep full
// across segment boundaries (48 KB per warp in flight, 192 KB per SM; the
// bandwidth-delay product needs about 45 KB per SM).  At a segment's end the
// four warps' (m, l, O) are joined through shared memory, and the pieces of a
// cut item through global memory by the last block to arrive.
//
// P is rounded to the cache's 16-bit type for the second product (its relative
// error is the type's, the same size as the output's own rounding, in f16 down
// to 2^-21 of the row's largest, paged_values.cuh); scores, m, l and O stay fp32.
//
// An 8-bit cache (storage S = I8 or E4M3, C = f16) runs through the same code with
// 12 warps (8 for 16 rows), since its tiles are half the bytes and the same
// products.  Codes become f16 on the way from shared memory to the products,
// exactly, and a block's scales (16 tokens = one 16-key half of the products) go to
// the scores and to the weights: S = (K Q^T) s_k, P' = 2^(S - m + log2(s_v / r)),
// l += (r / s_v) sum P', O += P' V.  r is a power of two at or above the value
// scales that the warp has met; where it grows, m falls by as much.  m is the
// maximum of S + log2(s_v / r), so the largest share of an output is a P' of 2^7 and
// not rounded, and the weights use f16's range whatever the scales.
//   Once a warp has met scales more than 2^61 apart (or zero; 2^13 where scores are
// far out), r / s_v no longer serves: keys with a tiny scale may hold all of a row's weight, or none of it beside
// a large one that counts, or one that the row does not see.  From there on l sums
// 2^(S - mu), mu the scores' own maximum, and m = mu + kappa is kept in two parts.
//
// Measured: 64 decodes of 4096 tokens, 16 heads, pages of 64: 311 us, 6.9 TB/s;
// 37 ragged decodes of up to 32768 tokens, 8 key heads, pages of 16: 279 us, 6.0
// TB/s (277 with the products taken out: 4 KB pages set that); one decode of 600
// tokens 7.2 us, of one token 4.0.  Codes: the same 64 decodes 175 us (e4m3; 6.1
// TB/s), the ragged ones 158 (int8; 124 with the arithmetic taken out), 600 tokens
// 8.4 or 8.2 (e4m3), one token 6; 64 decodes of 1024 tokens 65 and 62 (a segment
// is three tiles a warp there, and the warps meet at its end).  With m the scores'
// maximum the ragged ones took 149, and f16 outputs over few keys were off by up to
// 1.9 times their own rounding (now 1.2).  Joins and references that hold any scales
// cost 1 per cent of the long ones, half a microsecond of the short ones.
#pragma once

#include <cuda.h>
#include <math.h>
#include <string.h>

#include <type_traits>

#include "common.cuh"
#include "paged.h"
#include "paged_codes.cuh"
#include "paged_values.cuh"
#include "tc_ptx.cuh"

namespace tf {

namespace {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowBytes = 128;                        // one swizzled row: 64 values

// S: what the pages hold; the products' type C, or codes.
template <int D, int NT, typename C, typename S>
struct Shape {
  static constexpr bool kCoded = !std::is_same<S, C>::value;
  static constexpr int kWarps = !kCoded ? 4 : NT == 1 ? 12 : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRow = kCoded ? D : kRowBytes;             // bytes of a row in shared memory
  static constexpr int kHalves = kCoded ? 1 : D / 64;             // column parts that lie apart
  static constexpr int kTile = kHalves * kSplitKeys * kRow;       // bytes of a tile's keys (and of its values)
  static constexpr int kStages = kCoded ? 256 / D : 384 / D;      // 48 KB per warp, of codes 16
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kJoin = kCoded ? 64 : D;       // columns that are joined at a time
  static constexpr int kJoinRows = kCoded ? 8 * NT : kSplitRows;
  static constexpr int kPitch = kJoin + 4;            // joined outputs: rows 4 words apart in the banks
  static constexpr int kOffJoin = kWarps * kRing;
  static constexpr int kOffStat = kOffJoin + kWarps * kJoinRows * kPitch * 4;
  static constexpr int kStat = kSplitRows * (kCoded ? 3 : 2);  // a row's m and l, of codes also r
  static constexpr int kOffScale = kOffStat + kWarps * kStat * 4;  // [warp][stage] k, k, v, v
  static constexpr int kOffBar = kOffScale + (kCoded ? kWarps * kStages * 16 : 0);
  static constexpr int kSmem = kOffBar + kWarps * kStages * 8 + 16 + 1024;  // + alignment slack
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

struct SplitParams {
  CUtensorMap tm_k, tm_v;
  const void* q;
  int64_t q_stride;
  const int32_t* ids;
  int64_t ids_stride;
  int32_t columns;
  int32_t page_size;
  int32_t page_shift;
  int32_t box_rows, box_shift;  // min(page_size, kSplitKeys)
  int32_t group;     // query heads per key head
  int32_t heads;
  const PagedSegment* segments;
  const int32_t* starts;
  int* counters;
  float* stat;  // [part][2][16]: m, l
  float* part;  // [part][16][D] (of codes divided by l)
  void* out;
  float scale_log2;
  int least_power;  // power_floor of the scale
  int* err;
  const long long* wait_cycles;
  const float* k_scales;  // of codes
  const float* v_scales;
  int64_t scale_stride;
  int64_t pages;
};

// Waits for a phase of one of the warp's own copies, at most `limit` cycles.
__device__ __forceinline__ bool wait_copy(uint64_t* bar, uint32_t parity, long long limit) {
  const uint32_t suspend = limit < 2000000000LL ? 0u : kSuspendNs;  // a shortened limit polls
  if (mbar_try(bar, parity, suspend)) return true;
  const long long t0 = clock64();
  while (clock64() - t0 < limit)
    if (mbar_try(bar, parity, suspend)) return true;
  return false;
}

// `row` .. of a page, all columns: [64-column half][box row][128 bytes].
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int row, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(0), "r"(page), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// The 8x8 matrix of 16-bit values across the warp, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename C>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename C>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const C a = from_f<C>(lo), b = from_f<C>(hi);
  uint32_t u;
  if constexpr (sizeof(C) == 2) {
    const uint16_t x = *reinterpret_cast<const uint16_t*>(&a), y = *reinterpret_cast<const uint16_t*>(&b);
    u = (uint32_t)x | ((uint32_t)y << 16);
  }
  return u;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// max that keeps a NaN, so a row with a NaN score ends as NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Of the lanes that share a row of the products.
__device__ __forceinline__ float rows_max(float v) {
  v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return max_nan(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

// Weight of a part with maximum m against the joined maximum M: an empty part
// (m = -inf) weighs nothing, also where every part is empty.
__device__ __forceinline__ float part_weight(float m, float M) { return m == -INFINITY ? 0.f : exp2_fast(m - M); }

// The same times the part's sum, where a part's outputs are kept divided by it (an
// 8-bit cache, whose values may lie anywhere in fp32's range): down to 2^-149, for
// a small weight may stand before a large value.
__device__ __forceinline__ float part_share(float m, float M, float sum) {
  const float f = exp2_far(m - M);  // (before the choice, which then is no branch)
  return m == -INFINITY ? 0.f : f * sum;
}
// A power of two that brings up to 2^kParts shares of at most `most` each (a sum,
// below 2^110) to a total below one, and its inverse.
template <int kParts>
__device__ __forceinline__ float share_unit(float most) {
  return __uint_as_float((253u - kParts << 23) - (__float_as_uint(fmaxf(most, 0.f)) & 0x7f800000u));
}
template <int kParts>
__device__ __forceinline__ float share_unit_inverse(float most) {
  return __uint_as_float((1u + kParts << 23) + (__float_as_uint(fmaxf(most, 0.f)) & 0x7f800000u));
}

// The pieces of a segment's rows joined, in piece order within each of the groups
// of threads that share them; each piece's outputs are divided by its sum.  work:
// parts * 16 floats of shared memory, and at least four a thread.  Called by the
// whole block; ends with a barrier.
constexpr int kFewParts = 8;
template <typename T, int D, int kThreads>
__device__ __forceinline__ void merge_many(const SplitParams& p, const PagedSegment& sg, float* work) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int r = warp; r < sg.rows; r += kThreads / 32) {
    const float* stat = p.stat + (int64_t)sg.part0 * 32 + r;
    float M = -INFINITY, sum = 0.f;
    for (int k = lane; k < sg.parts; k += 32) M = max_nan(M, __ldcg(stat + (int64_t)k * 32));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, off));
    for (int k = lane; k < sg.parts; k += 32) {
      const float f = part_share(__ldcg(stat + (int64_t)k * 32), M, __ldcg(stat + (int64_t)k * 32 + 16));
      sum += f;
      work[k * kSplitRows + r] = f;
    }
    sum = warp_sum_butterfly(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int k = lane; k < sg.parts; k += 32) work[k * kSplitRows + r] *= inv;
  }
  __syncthreads();
  // Four values a thread; threads i, i + n, i + 2 n, ... take every g-th piece.
  const int n = sg.rows * (D / 4), groups = max(1, min(kThreads / n, 8));
  for (int i0 = 0; i0 < n; i0 += kThreads) {  // one round but for many rows
    const int i = groups > 1 ? tid % n : i0 + tid, group = groups > 1 ? tid / n : 0;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool mine = i < n && group < groups;
    const int r = mine ? i / (D / 4) : 0, d = i % (D / 4) * 4;
    if (mine) {
      const float* from = p.part + ((int64_t)sg.part0 * kSplitRows + r) * D + d;
#pragma unroll 4
      for (int k = group; k < sg.parts; k += groups) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(from + (int64_t)k * kSplitRows * D));
        const float f = work[k * kSplitRows + r];
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
    }
    if (groups > 1) {  // the weights' place is free now
      __syncthreads();
      float4* out = reinterpret_cast<float4*>(work);
      if (mine && group > 0) out[(group - 1) * n + i] = acc;
      __syncthreads();
      if (mine && group == 0)
        for (int g = 1; g < groups; ++g) {
          const float4 v = out[(g - 1) * n + i];
          acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
        }
    }
    if (mine && group == 0) {
      const int pr = sg.row0 + r;
      T* orow = static_cast<T*>(p.out) + ((int64_t)(sg.q_row + pr / p.group) * p.heads + sg.kv_head * p.group +
                                          pr % p.group) * D + d;
      alignas(8) const T v[4] = {from_f<T>(acc.x), from_f<T>(acc.y), from_f<T>(acc.z), from_f<T>(acc.w)};
      *reinterpret_cast<uint2*>(orow) = *reinterpret_cast<const uint2*>(v);
    }
  }
  __syncthreads();
}

// A warp's position in its block's work: tile `tile` of segment `seg`.
struct Cursor {
  int seg, end, tile, tile1;
  int request, kv_head, kv_len;
  __device__ __forceinline__ void load(const PagedSegment* s, int warp) {
    const PagedSegment& g = s[seg];
    tile = g.tile0 + warp;
    tile1 = g.tile1;
    request = g.request;
    kv_head = g.kv_head;
    kv_len = g.kv_len;
  }
  // Moves to the next tile that exists; false at the end of the block's work.
  __device__ __forceinline__ bool settle(const PagedSegment* s, int warp) {
    while (tile >= tile1) {
      if (++seg >= end) return false;
      load(s, warp);
    }
    return true;
  }
};

template <typename T, typename C, int D, int NT, typename St>  // NT: groups of 8 packed rows
__global__ void __launch_bounds__(Shape<D, NT, C, St>::kThreads, 1)
    paged_split_kernel(const __grid_constant__ SplitParams p) {
  using S = Shape<D, NT, C, St>;
  constexpr bool kCoded = S::kCoded;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kStat = S::kStat;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = base + warp * S::kRing;
  float* join = reinterpret_cast<float*>(base + S::kOffJoin);
  float* stat = reinterpret_cast<float*>(base + S::kOffStat);  // [warp][kStat / 16][16]
  float* scales = reinterpret_cast<float*>(base + S::kOffScale) + warp * S::kStages * 4;
  float* kappa = stat + warp * kStat + 32;  // of the warp's rows, until its results are joined
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kOffBar) + warp * S::kStages;
  int* last_s = reinterpret_cast<int*>(base + S::kOffBar + kWarps * S::kStages * 8);

  // A tensor-core kernel of the same call may start where blocks have left.
  asm volatile("griddepcontrol.launch_dependents;");
  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&bars[i], kCoded ? 33 : 1);  // of codes: each lane's scales
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();

  const int seg0 = p.starts[blockIdx.x], seg_end = p.starts[blockIdx.x + 1];
  Cursor in;  // next tile to fetch
  in.seg = seg0;
  in.end = seg_end;
  bool more = seg0 < seg_end;
  if (more) {
    in.load(p.segments, warp);
    more = in.settle(p.segments, warp);
  }
  int fetched = 0, used = 0;
  // Box of this lane in a tile: which page's part, keys or values.  The page id of
  // the next tile is looked up a tile ahead.
  const int box = lane >> 1, is_v = lane & 1;
  // Of codes, box = 16-key half of the tile as far as the scales go.
  const int half_bytes = p.box_rows * S::kRow, box_bytes = half_bytes * S::kHalves;
  int page = -1;
  auto look_up = [&]() {
    if (kCoded && lane >= 4) return;
    const int column = (in.tile * kSplitKeys + box * (kCoded ? kScaleTokens : p.box_rows)) >> p.page_shift;
    page = column < p.columns ? __ldg(p.ids + in.request * p.ids_stride + column) : -1;
  };
  if (more) look_up();

  // Fetches one tile into the ring's next slot: lanes 2 i, 2 i + 1 copy the keys
  // and the values of box i of the tile's existing pages.
  auto fetch = [&]() {
    const int slot = fetched % S::kStages;
    uint8_t* dst = ring + slot * 2 * S::kTile;
    const int key0 = in.tile * kSplitKeys;
    const int left = in.kv_len - key0;
    const int want = left < kSplitKeys ? left : kSplitKeys;
    const int boxes = (want + p.box_rows - 1) / p.box_rows;  // pages (or parts of one) that exist
    if (lane == 0) mbar_expect_tx(&bars[slot], (uint32_t)(boxes * box_bytes * 2));
    __syncwarp();
    if (box < boxes) {
      const int row = in.kv_head * p.page_size + ((key0 + box * p.box_rows) & (p.page_size - 1));
      if constexpr (kCoded)
        tma_codes(dst + is_v * S::kTile + box * box_bytes, is_v ? &p.tm_v : &p.tm_k, row, page, &bars[slot]);
      else
        tma_page(dst + is_v * S::kTile + box * box_bytes, is_v ? &p.tm_v : &p.tm_k, row, page, &bars[slot]);
    }
    if constexpr (kCoded) {
      if (lane < 4) {
        const int key = key0 + box * kScaleTokens;
        const bool real = key < in.kv_len && page >= 0 && page < p.pages;
        const float* from = is_v ? p.v_scales : p.k_scales;
        if (real)
          from += page * p.scale_stride + in.kv_head * (p.page_size / kScaleTokens) +
                  (key & (p.page_size - 1)) / kScaleTokens;
        copy_value(scales + slot * 4 + 2 * is_v + box, from, real);
      }
      arrive_with_copies(&bars[slot]);
    }
    ++fetched;
    in.tile += kWarps;
    more = in.settle(p.segments, warp);
    if (more) look_up();
  };
  for (int i = 0; i < S::kStages && more; ++i) fetch();

  const int g = lane >> 2, c2 = (lane & 3) * 2;  // MMA fragment row (or column) and column pair
  const long long limit_cycles = *p.wait_cycles;
  // Offset of key r in a tile, and those of the keys that this lane's ldmatrix
  // addresses name.
  auto key_at = [&](int r) {
    return kCoded ? r * S::kRow : (r >> p.box_shift) * box_bytes + (r & (p.box_rows - 1)) * S::kRow;
  };
  // Of codes, the lane's 16-byte chunk lane / 16 of row lane % 16 (128- or 64-byte
  // swizzle); chunk + k, k even, lies at the address ^ 16 k, and 16 rows on the
  // swizzle is the same.
  const uint32_t code_at = (lane & 15) * D + ((lane >> 4 ^ (D == 128 ? lane & 7 : lane >> 1 & 3)) << 4);
  int k_at[2], v_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    k_at[h] = key_at(16 * h + (lane & 15));
    v_at[h] = key_at(16 * h + (lane & 7) + ((lane >> 4) << 3));
  }
  bool ok = true;
  for (int seg = seg0; seg < seg_end; ++seg) {
    const PagedSegment sg = p.segments[seg];
    // Queries as the B operand: packed row 8 t + g.
    uint32_t qb[D / 16][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int pr = sg.row0 + min(8 * t + g, sg.rows - 1);
      const T* qr = static_cast<const T*>(p.q) + (sg.q_row + pr / p.group) * p.q_stride +
                    (int64_t)(sg.kv_head * p.group + pr % p.group) * D;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          qb[k][t][j] = *reinterpret_cast<const uint32_t*>(qr + 16 * k + (kCoded ? 2 * c2 + 2 * j : 8 * j + c2));
    }
    float scale[NT][2];  // of the scores of rows 8 t + c2, + 1
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      scale[t][0] = scale[t][1] = p.scale_log2;
      if constexpr (Act<T>::kDtype != Act<C>::kDtype) {
        uint32_t most = 0;  // of row 8 t + g, whose values four lanes share
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) most = magnitude(qb[k][t][j], most);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int over = beyond_f16(most, p.least_power);
        const float down = power2(-over);
#pragma unroll
        for (int i = 0; i < 2; ++i) scale[t][i] *= power2(__shfl_sync(0xffffffffu, over, 4 * (c2 + i)));
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const T* v = reinterpret_cast<const T*>(&qb[k][t][j]);
            qb[k][t][j] = pack2<C>(to_f(v[0]) * down, to_f(v[1]) * down);
          }
      }
    }
    int limit[NT][2];  // last key that rows 8 t + c2, + 1 see
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        limit[t][i] = sg.kv_len - sg.new_len + (sg.row0 + min(8 * t + c2 + i, sg.rows - 1)) / p.group;
    const int first_limit = sg.kv_len - sg.new_len + sg.row0 / p.group;  // what the first row sees
    // O^T: dims 16 d + g, + 8 (of codes 16 d + 2 g, + 1), rows 8 t + c2, + 1
    float o[D / 16][NT][4];
    float ref = kLeastRef, ref_inverse = kLeastInverse;  // r, of codes
    float lowest = INFINITY;  // value scale so far
    bool wide = false;        // scales so far apart that l has a reference of its own
    float fall = 0.f;         // log2(r of the tile before / r)
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][t][j] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) m[t][i] = -INFINITY, l[t][i] = 0.f;

    // Of codes two loops: the second from the first tile on with which scales lie far
    // apart (in one loop that rare path cost 2 per cent of the time).
    int tile = sg.tile0 + warp;
#pragma unroll
    for (int apart = 0; apart < (kCoded ? 2 : 1); ++apart) {
    if (apart == 1) {
      if (__builtin_expect(!wide, 1)) break;
      if (lane < 16) kappa[lane] = 0.f;
      __syncwarp();
    }
    for (; tile < sg.tile1 && ok; tile += kWarps) {
      const int slot = used % S::kStages;
      ok = __all_sync(0xffffffffu, wait_copy(&bars[slot], (uint32_t)((used / S::kStages) & 1), limit_cycles));
      if (!ok) {
        if (lane == 0) atomicCAS(p.err, 0, 71);
        break;
      }
      const uint32_t ks = smem_addr(ring + slot * 2 * S::kTile), vs = ks + S::kTile;
      const int key0 = tile * kSplitKeys;
      // Scores S^T: keys 16 h + g, + 8, rows 8 t + c2, + 1.
      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[h][t][j] = 0.f;
      float k_scale[2] = {1.f, 1.f};
      float offset[2], back[2];  // log2(s_v / r), r / s_v
      bool odd = false;     // a value scale is not finite
      bool spread = false;  // scales too far apart for scores far out
      if constexpr (kCoded) {
        const float4 four = *reinterpret_cast<const float4*>(scales + slot * 4);
        k_scale[0] = four.x;
        k_scale[1] = four.y;
        float v[2] = {four.z, four.w}, some[2];
        const auto grow = [&](float most) {
          if (!(most > ref)) return;
          const float next = power_above(most);
          fall += exponent_of(ref) - exponent_of(next);
          ref = next;
          ref_inverse = inverse_of(next);
        };
        // (Of a block past the request's length the scale is zero.)
        const float larger = fmaxf(v[0], v[1]);
        if (larger < INFINITY) grow(larger);
        some[0] = v[0] * ref_inverse;
        some[1] = v[1] * ref_inverse;
        const float low = fminf(fminf(some[0], some[1]), lowest * ref_inverse);
        if (__builtin_expect(!(low >= kFarRatio && max_nan(some[0], some[1]) <= 1.f), 0)) {
          bool real[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            real[h] = key0 + kScaleTokens * h < sg.kv_len && v[h] < INFINITY;
            odd |= key0 + kScaleTokens * h < sg.kv_len && !real[h];
            if (real[h]) grow(v[h]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!real[h]) v[h] = ref;  // any will do
            some[h] = v[h] * ref_inverse;
          }
          const float least = fminf(lowest, fminf(v[0], v[1]));
          if (apart == 0 && far_apart(least, ref)) {
            wide = true;
            break;
          }
          spread = least < ref * kFarRatio;
        }
        lowest = fminf(lowest, fminf(v[0], v[1]));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          offset[h] = apart ? log2f(v[h]) - exponent_of(ref) : __log2f(some[h]);
          back[h] = __fdividef(1.f, some[h]);
        }
        // Bytes 4 c .. 4 c + 3 of a lane's row are taken as columns 2 c, 2 c + 1, 2 c + 8
        // and 2 c + 9 of the product, as the queries are.
#pragma unroll
        for (int k = 0; k < D / 16; k += 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
            ldsm4((ks + code_at ^ k << 4) + 16 * h * D, w);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t a[4];
              Code<St>::widen(w[2 * j], a[0], a[2]);
              Code<St>::widen(w[2 * j + 1], a[1], a[3]);
#pragma unroll
              for (int t = 0; t < NT; ++t) mma16816<C>(s[h][t], a, qb[k + j][t][0], qb[k + j][t][1]);
            }
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a[4];
            const int chunk = (2 * k + (lane >> 4)) & 7;
            ldsm4(ks + (k >> 2) * half_bytes + k_at[h] + ((chunk ^ (lane & 7)) << 4), a);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma16816<C>(s[h][t], a, qb[k][t][0], qb[k][t][1]);
          }
        }
      }
      if (kCoded && apart == 0 && __builtin_expect(spread, 0)) {
        bool far = false;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) far |= fabsf(s[h][t][j] * (scale[t][j & 1] * k_scale[h])) >= kFar;
        if (__any_sync(0xffffffffu, far)) {
          wide = true;
          break;
        }
      }
      const bool ragged = key0 + kSplitKeys - 1 > first_limit;
      uint32_t pb[2][NT][2];  // P^T as the B operand
      float keep[NT][2];
      bool moved = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float sub[2];
        if (apart) {
          // P' = 2^((s - mu) + log2(s_v / r) - kappa), mu the scores' maximum (in m), kappa
          // that of the shares beside it; l has mu for its reference.
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 8 * t + c2 + i;
            float own = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = i; j < 4; j += 2) {
                float v = s[h][t][j] * (scale[t][i] * k_scale[h]);
                if (ragged && key0 + 16 * h + g + 4 * (j - i) > limit[t][i]) v = -INFINITY;
                s[h][t][j] = v;
                own = max_nan(own, v);
              }
            own = rows_max(own);
            const float mu = max_nan(m[t][i], own), from = mu == -INFINITY ? 0.f : mu;
            l[t][i] *= part_weight(m[t][i], from);
            float most = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = i; j < 4; j += 2) {
                const float v = s[h][t][j];
                // The NaN of a key or of inf - inf stays; a hidden key is none.
                const float d = v - from;
                l[t][i] += exp2_fast(d);
                s[h][t][j] = d + offset[h];
                most = max_nan(most, s[h][t][j]);
                if (odd && v != -INFINITY && !(fabsf(scales[slot * 4 + 2 + h]) < INFINITY))
                  l[t][i] = __uint_as_float(0x7fc00000u);
              }
            most = rows_max(most) - kLift;
            const float stands = kappa[r] + fall + (m[t][i] - from), next = max_nan(stands, most);
            __syncwarp();
            if (g == 0) kappa[r] = next;
            __syncwarp();
            sub[i] = next == -INFINITY ? 0.f : next;
            keep[t][i] = stands == -INFINITY ? 1.f : exp2_fast(stands - sub[i]);  // nothing stands in O yet
            moved |= keep[t][i] != 1.f;
            m[t][i] = mu;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            pb[h][t][0] = transpose8(pack2<C>(exp2_fast(s[h][t][0] - sub[0]), exp2_fast(s[h][t][1] - sub[1])));
            pb[h][t][1] = transpose8(pack2<C>(exp2_fast(s[h][t][2] - sub[0]), exp2_fast(s[h][t][3] - sub[1])));
          }
          continue;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float most = -INFINITY;
#pragma unroll
            for (int j = i; j < 4; j += 2) {
              float v = s[h][t][j] * (kCoded ? scale[t][i] * k_scale[h] : scale[t][i]);
              if (ragged && key0 + 16 * h + g + 4 * (j - i) > limit[t][i]) v = -INFINITY;
              s[h][t][j] = v;
              most = max_nan(most, v);
            }
            // (Far out the sum's rounding would lie between m and the scores.)
            if constexpr (kCoded) most += fabsf(most) < kFar ? offset[h] : 0.f;
            mx = max_nan(mx, most);
          }
          mx = rows_max(mx);
          // What m stands for falls with r, of codes.
          const float mn = max_nan(kCoded ? m[t][i] + fall : m[t][i], lifted<C>(mx));
          // Rows that have seen no key yet keep m = -inf and add nothing.
          sub[i] = mn == -INFINITY ? 0.f : mn;
          keep[t][i] = exp2_fast(kCoded ? (m[t][i] - sub[i]) + fall : m[t][i] - sub[i]);
          moved |= keep[t][i] != 1.f;
          if (kCoded && __builtin_expect(fall != 0.f, 0))
            l[t][i] *= exp2_fast(m[t][i] - sub[i]);  // 2^61 at most: else the scales are far apart
          else
            l[t][i] *= keep[t][i];
          m[t][i] = mn;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kCoded) {
              e[j] = exp2_fast((s[h][t][j] - sub[j & 1]) + offset[h]);
            } else {
              e[j] = exp2_fast(s[h][t][j] - sub[j & 1]);
              l[t][j & 1] += e[j];
            }
          }
          if constexpr (kCoded) {
#pragma unroll
            for (int i = 0; i < 2; ++i) l[t][i] = fmaf(e[i] + e[i + 2], back[h], l[t][i]);
            if (odd) {  // the rows that see a key of such a block are NaN
              const float v = scales[slot * 4 + 2 + h];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (!(fabsf(v) < INFINITY) && s[h][t][j] != -INFINITY) l[t][j & 1] = __uint_as_float(0x7fc00000u);
            }
          }
          pb[h][t][0] = transpose8(pack2<C>(e[0], e[1]));
          pb[h][t][1] = transpose8(pack2<C>(e[2], e[3]));
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[d][t][j] *= keep[t][j & 1];
      }
      const int have = sg.kv_len - key0;
      if (kCoded) {
        // Integer codes are finite, whatever lies there.
        if (!std::is_same<St, I8>::value && have < kSplitKeys) {
          uint8_t* v = ring + slot * 2 * S::kTile + S::kTile;
          for (int i = have * (D / 16) + lane; i < kSplitKeys * (D / 16); i += 32)
            *reinterpret_cast<uint4*>(v + 16 * i) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
      } else if (have < kSplitKeys) {
        // Slots past the request's length hold anything, NaN included: 0 * NaN
        // would reach the outputs, so their values become zeros.
        uint8_t* v = ring + slot * 2 * S::kTile + S::kTile;
        for (int i = have * 8 + lane; i < kSplitKeys * 8; i += 32)
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
            *reinterpret_cast<uint4*>(v + key_at(i >> 3) + h * half_bytes + 16 * (i & 7)) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      // Keys that some row does not see, with values that are not finite.
      const int hidden = max(first_limit + 1 - key0, 0), hidden_end = min(have, kSplitKeys);
      bool cleared = false;
      if (!kCoded && hidden < hidden_end) {
        uint8_t* v = ring + slot * 2 * S::kTile + S::kTile;
        // A box's keys of one column half lie side by side.
        for (int key = hidden; key < hidden_end;) {
          const int next = min((key | (p.box_rows - 1)) + 1, hidden_end);
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
            cleared |= !all_finite<C>(v + key_at(key) + h * half_bytes, (next - key) * 8, lane);
          key = next;
        }
        if (cleared) {
#pragma unroll 1
          for (int key = hidden; key < hidden_end; ++key)
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int dim = (16 * d + 8 * half + g) & 63;
                const C c = *reinterpret_cast<const C*>(v + key_at(key) + (d >> 2) * half_bytes +
                                                        (((dim >> 3) ^ (key & 7)) << 4) + 2 * (dim & 7));
                if (!not_finite(c)) continue;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                  for (int i = 0; i < 2; ++i)
                    if (key0 + key <= limit[t][i]) o[d][t][2 * half + i] += to_f(c);
              }
          __syncwarp();
          for (int key = hidden; key < hidden_end; ++key)
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h) clear_not_finite<C>(v + key_at(key) + h * half_bytes, 8, lane);
          __syncwarp();
        }
      }
      if constexpr (kCoded) {
        // A transposed pair of bytes holds two dims of one key: the even dims take
        // the product's first eight rows, the odd ones the rest.
#pragma unroll
        for (int d = 0; d < D / 16; d += 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
            ldsm4_t((vs + code_at ^ d << 4) + 16 * h * D, w);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t a[4];
              Code<St>::widen_cross(w[2 * j], a[0], a[1]);
              Code<St>::widen_cross(w[2 * j + 1], a[2], a[3]);
#pragma unroll
              for (int t = 0; t < NT; ++t) mma16816<C>(o[d + j][t], a, pb[h][t][0], pb[h][t][1]);
            }
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a[4];
            const int chunk = (2 * d + ((lane >> 3) & 1)) & 7;
            ldsm4_t(vs + (d >> 2) * half_bytes + v_at[h] + ((chunk ^ (lane & 7)) << 4), a);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma16816<C>(o[d][t], a, pb[h][t][0], pb[h][t][1]);
          }
        }
      }
      // Every lane's shared loads fed an MMA above, so they have returned: the
      // slot may be refilled.  Zeros written above precede the copy.
      if (have < kSplitKeys || cleared) fence_proxy_async();
      __syncwarp();
      ++used;
      if (more) fetch();
      fall = 0.f;
    }
    }

    // Join the warps' results.
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 4);
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 8);
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 16);
        const int r = 8 * t + c2 + i;
        float gain = ref;  // of codes: what O is to be multiplied with
        if (kCoded && wide) {
          gain = exp2_far(kappa[r] + exponent_of(ref));
          __syncwarp();  // it takes kappa's place
        }
        if (g == 0) {
          stat[warp * kStat + r] = m[t][i];
          stat[warp * kStat + 16 + r] = l[t][i];
          if (kCoded) stat[warp * kStat + 32 + r] = gain;
        }
      }
#pragma unroll
    for (int pass = 0; pass < D / S::kJoin; ++pass) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float* row = join + (warp * S::kJoinRows + 8 * t + c2 + i) * S::kPitch;
#pragma unroll
          for (int d = 0; d < S::kJoin / 16; ++d) {
            row[16 * d + (kCoded ? 2 * g : g)] = o[pass * (S::kJoin / 16) + d][t][i];
            row[16 * d + (kCoded ? 2 * g + 1 : g + 8)] = o[pass * (S::kJoin / 16) + d][t][i + 2];
          }
        }
      __syncthreads();
      for (int i = tid; i < sg.rows * S::kJoin; i += kThreads) {
        const int r = i / S::kJoin, at = i % S::kJoin, d = pass * S::kJoin + at;
        float M = stat[r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) M = max_nan(M, stat[w * kStat + r]);
        float acc = 0.f, sum = 0.f, most = 0.f;
        if constexpr (kCoded) {
#pragma unroll
          for (int w = 0; w < kWarps; ++w) most = fmaxf(most, stat[w * kStat + 16 + r]);
          const float unit = share_unit<4>(most);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            // O has the sum's size, so a large gain goes with the unit, a small one apart from
            // it: nothing on the way lies outside fp32's range that does not in the end.
            const float f = part_share(stat[w * kStat + r], M, 1.f), gain = stat[w * kStat + 32 + r];
            acc = fmaf(join[(w * S::kJoinRows + r) * S::kPitch + at] * (unit * fmaxf(gain, 1.f)), f * fminf(gain, 1.f), acc);
            sum = fmaf(f, stat[w * kStat + 16 + r] * unit, sum);
          }
          acc = sum == 0.f ? 0.f : acc / sum;
        } else {
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float f = part_weight(stat[w * kStat + r], M);
            acc = fmaf(f, join[(w * S::kJoinRows + r) * S::kPitch + at], acc);
            sum = fmaf(f, stat[w * kStat + 16 + r], sum);
          }
        }
        if (sg.part < 0) {
          const int pr = sg.row0 + r;
          T* orow = static_cast<T*>(p.out) + ((int64_t)(sg.q_row + pr / p.group) * p.heads + sg.kv_head * p.group +
                                              pr % p.group) * D;
          orow[d] = from_f<T>(kCoded ? acc : sum == 0.f ? 0.f : acc / sum);
        } else {
          p.part[((int64_t)sg.part * kSplitRows + r) * D + d] = acc;
          if (d == 0) {
            p.stat[(int64_t)sg.part * 32 + r] = M;
            p.stat[(int64_t)sg.part * 32 + 16 + r] = kCoded ? sum * share_unit_inverse<4>(most) : sum;
          }
        }
      }
      __syncthreads();
    }
    if (sg.part >= 0) {
      // The last piece of these rows to finish merges all of them, in order.
      if (tid == 0) {
        __threadfence();
        const int seen = atomicAdd(&p.counters[sg.counter], 1);
        const int last = seen == sg.parts - 1;
        if (last) p.counters[sg.counter] = 0;  // as the next call expects it
        *last_s = last;
      }
      __syncthreads();
      const bool last = *last_s != 0;
      __syncthreads();
      if (!last) continue;
      __threadfence();
      if constexpr (kCoded) {
        // Many pieces: their weights first, a warp a row, then groups of threads that
        // share the pieces (one long request, 148 pieces: 65 -> 27 us).
        constexpr int kRoom = kWarps * S::kJoinRows * S::kPitch;
        static_assert(kRoom >= 4 * kThreads, "the groups' outputs");
        if (sg.parts > kFewParts && sg.parts * kSplitRows <= kRoom) {
          merge_many<T, D, kThreads>(p, sg, join);
          continue;
        }
      }
      for (int i = tid; i < sg.rows * D; i += kThreads) {
        const int r = i / D, d = i % D;
        float M = -INFINITY, most = 0.f;
        for (int k = 0; k < sg.parts; ++k) {
          const float* st = &p.stat[(int64_t)(sg.part0 + k) * 32 + r];
          M = max_nan(M, __ldcg(st));
          if (kCoded) most = fmaxf(most, __ldcg(st + 16));
        }
        const float unit = share_unit<8>(most);
        float acc = 0.f, sum = 0.f;
        for (int k = 0; k < sg.parts; ++k) {
          const int64_t at = sg.part0 + k;
          const float m = __ldcg(&p.stat[at * 32 + r]), own = __ldcg(&p.stat[at * 32 + 16 + r]);
          const float f = kCoded ? part_share(m, M, own * unit) : part_weight(m, M);
          acc = fmaf(f, __ldcg(&p.part[(at * kSplitRows + r) * D + d]), acc);
          sum = kCoded ? sum + f : fmaf(f, own, sum);
        }
        const int pr = sg.row0 + r;
        T* orow = static_cast<T*>(p.out) + ((int64_t)(sg.q_row + pr / p.group) * p.heads + sg.kv_head * p.group +
                                            pr % p.group) * D;
        orow[d] = from_f<T>(sum == 0.f ? 0.f : acc / sum);
      }
    }
  }
  // After an expired wait copies may still be in flight: they land before the
  // block's shared memory goes to another (they always complete).
  for (; used < fetched; ++used)
    wait_copy(&bars[used % S::kStages], (uint32_t)((used / S::kStages) & 1), 2000000000LL);
}

template <typename T, typename C, int D, int NT, typename St>
tf_status launch(const SplitParams& p, int blocks, cudaStream_t s) {
  using S = Shape<D, NT, C, St>;
  static PerDeviceOnce attr;
  int dev = 0;
  if (attr.needed(&dev)) {
    TF_CUDA(cudaFuncSetAttribute(paged_split_kernel<T, C, D, NT, St>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 S::kSmem));
    attr.mark(dev);
  }
  paged_split_kernel<T, C, D, NT, St><<<blocks, S::kThreads, S::kSmem, s>>>(p);
  return check_launch("paged_split");
}

// What all launches fill in alike.
tf_status split_params(const PagedArgs& a, SplitParams* out) {
  const tf_paged_plan& plan = *a.plan;
  SplitParams& p = *out;
  memset(&p, 0, sizeof(p));
  p.box_rows = a.kv.page_size < kSplitKeys ? a.kv.page_size : kSplitKeys;
  while ((1 << p.box_shift) < p.box_rows) ++p.box_shift;
  p.q = a.q;
  p.q_stride = a.q_stride;
  p.ids = a.table.ids;
  p.ids_stride = a.table.stride;
  p.columns = a.table.columns;
  p.page_size = a.kv.page_size;
  while ((1 << p.page_shift) < a.kv.page_size) ++p.page_shift;
  p.group = plan.heads / plan.kv_heads;
  p.heads = plan.heads;
  p.segments = reinterpret_cast<const PagedSegment*>(a.plan_table + plan.split_segments_offset);
  p.starts = reinterpret_cast<const int32_t*>(a.plan_table + plan.split_starts_offset);
  p.counters = reinterpret_cast<int*>(a.plan_table);
  p.stat = reinterpret_cast<float*>(a.workspace);
  p.part = p.stat + (int64_t)plan.split_parts * 2 * kSplitRows;
  p.out = a.out;
  p.scale_log2 = a.scale * kLog2e;
  p.least_power = power_floor(p.scale_log2);
  TF_TRY(tc_flags(&p.err, const_cast<long long**>(&p.wait_cycles)));
  return TF_OK;
}

template <typename T, typename C, typename St>
tf_status launch_rows(const SplitParams& p, const tf_paged_plan& plan, cudaStream_t s) {
  // Half the products where no request has more than 8 packed rows.
  if (plan.split_rows <= 8)
    return plan.head_dim == 128 ? launch<T, C, 128, 1, St>(p, plan.split_blocks, s)
                                : launch<T, C, 64, 1, St>(p, plan.split_blocks, s);
  return plan.head_dim == 128 ? launch<T, C, 128, 2, St>(p, plan.split_blocks, s)
                              : launch<T, C, 64, 2, St>(p, plan.split_blocks, s);
}

}  // namespace

}  // namespace tf
