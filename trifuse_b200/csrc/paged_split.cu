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
// Measured: 64 decodes of 4096 tokens, 16 heads, pages of 64: 311 us, 6.9 TB/s;
// 37 ragged decodes of up to 32768 tokens, 8 key heads, pages of 16: 279 us, 6.0
// TB/s (277 with the products taken out: 4 KB pages set that); one decode of 600
// tokens 7.2 us, of one token 4.0.
#include <cuda.h>
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "paged.h"
#include "paged_values.cuh"
#include "tc_ptx.cuh"

namespace tf {

namespace {

using namespace tc;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowBytes = 128;                        // one swizzled row: 64 values

template <int D>
struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kSplitKeys * kRowBytes;  // bytes of a tile's keys (and of its values)
  static constexpr int kStages = 384 / D;             // 48 KB per warp
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kPitch = D + 4;                // joined outputs: rows 4 words apart in the banks
  static constexpr int kOffJoin = kWarps * kRing;
  static constexpr int kOffStat = kOffJoin + kWarps * kSplitRows * kPitch * 4;
  static constexpr int kOffBar = kOffStat + kWarps * kSplitRows * 2 * 4;
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
  float* part;  // [part][16][D]
  void* out;
  float scale_log2;
  int* err;
  const long long* wait_cycles;
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

// Weight of a part with maximum m against the joined maximum M: an empty part
// (m = -inf) weighs nothing, also where every part is empty.
__device__ __forceinline__ float part_weight(float m, float M) { return m == -INFINITY ? 0.f : exp2_fast(m - M); }

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

template <typename T, typename C, int D, int NT>  // NT: groups of 8 packed rows
__global__ void __launch_bounds__(kThreads, 1) paged_split_kernel(const __grid_constant__ SplitParams p) {
  using S = Shape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = base + warp * S::kRing;
  float* join = reinterpret_cast<float*>(base + S::kOffJoin);
  float* stat = reinterpret_cast<float*>(base + S::kOffStat);  // [warp][2][16]
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kOffBar) + warp * S::kStages;
  int* last_s = reinterpret_cast<int*>(base + S::kOffBar + kWarps * S::kStages * 8);

  // A tensor-core kernel of the same call may start where blocks have left.
  asm volatile("griddepcontrol.launch_dependents;");
  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&bars[i], 1);
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
  // Box of this lane in a tile: which page's part, keys or values.  The page id of the next tile is looked up a tile ahead.
  const int box = lane >> 1, is_v = lane & 1;
  const int half_bytes = p.box_rows * kRowBytes, box_bytes = half_bytes * S::kHalves;
  int page = -1;
  auto look_up = [&]() {
    const int column = (in.tile * kSplitKeys + box * p.box_rows) >> p.page_shift;
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
      tma_page(dst + is_v * S::kTile + box * box_bytes, is_v ? &p.tm_v : &p.tm_k, row, page, &bars[slot]);
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
  auto key_at = [&](int r) { return (r >> p.box_shift) * box_bytes + (r & (p.box_rows - 1)) * kRowBytes; };
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
          qb[k][t][j] = *reinterpret_cast<const uint32_t*>(qr + 16 * k + 8 * j + c2);
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
        const int over = beyond_f16(most);
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
    float o[D / 16][NT][4];  // O^T: dims 16 d + g, + 8, rows 8 t + c2, + 1
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

    for (int tile = sg.tile0 + warp; tile < sg.tile1 && ok; tile += kWarps) {
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
      const bool ragged = key0 + kSplitKeys - 1 > first_limit;
      uint32_t pb[2][NT][2];  // P^T as the B operand
      float keep[NT][2];
      bool moved = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float sub[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = i; j < 4; j += 2) {
              float v = s[h][t][j] * scale[t][i];
              if (ragged && key0 + 16 * h + g + 4 * (j - i) > limit[t][i]) v = -INFINITY;
              s[h][t][j] = v;
              mx = max_nan(mx, v);
            }
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = max_nan(m[t][i], lifted<C>(mx));
          // Rows that have seen no key yet keep m = -inf and add nothing.
          sub[i] = mn == -INFINITY ? 0.f : mn;
          keep[t][i] = exp2_fast(m[t][i] - sub[i]);
          moved |= keep[t][i] != 1.f;
          m[t][i] = mn;
          l[t][i] *= keep[t][i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            e[j] = exp2_fast(s[h][t][j] - sub[j & 1]);
            l[t][j & 1] += e[j];
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
      if (have < kSplitKeys) {
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
      if (hidden < hidden_end) {
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
      // Every lane's shared loads fed an MMA above, so they have returned: the
      // slot may be refilled.  Zeros written above precede the copy.
      if (have < kSplitKeys || cleared) fence_proxy_async();
      __syncwarp();
      ++used;
      if (more) fetch();
    }

    // Join the four warps' results.
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 4);
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 8);
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 16);
        const int r = 8 * t + c2 + i;
        if (g == 0) {
          stat[warp * 32 + r] = m[t][i];
          stat[warp * 32 + 16 + r] = l[t][i];
        }
        float* row = join + (warp * kSplitRows + r) * S::kPitch;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          row[16 * d + g] = o[d][t][i];
          row[16 * d + g + 8] = o[d][t][i + 2];
        }
      }
    __syncthreads();
    for (int i = tid; i < sg.rows * D; i += kThreads) {
      const int r = i / D, d = i % D;
      float M = stat[r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) M = max_nan(M, stat[w * 32 + r]);
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = part_weight(stat[w * 32 + r], M);
        acc = fmaf(f, join[(w * kSplitRows + r) * S::kPitch + d], acc);
        sum = fmaf(f, stat[w * 32 + 16 + r], sum);
      }
      if (sg.part < 0) {
        const int pr = sg.row0 + r;
        T* orow = static_cast<T*>(p.out) + ((int64_t)(sg.q_row + pr / p.group) * p.heads + sg.kv_head * p.group +
                                            pr % p.group) * D;
        orow[d] = from_f<T>(sum == 0.f ? 0.f : acc / sum);
      } else {
        p.part[((int64_t)sg.part * kSplitRows + r) * D + d] = acc;
        if (d == 0) {
          p.stat[(int64_t)sg.part * 32 + r] = M;
          p.stat[(int64_t)sg.part * 32 + 16 + r] = sum;
        }
      }
    }
    __syncthreads();
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
      for (int i = tid; i < sg.rows * D; i += kThreads) {
        const int r = i / D, d = i % D;
        float M = -INFINITY;
        for (int k = 0; k < sg.parts; ++k) M = max_nan(M, __ldcg(&p.stat[(int64_t)(sg.part0 + k) * 32 + r]));
        float acc = 0.f, sum = 0.f;
        for (int k = 0; k < sg.parts; ++k) {
          const int64_t at = sg.part0 + k;
          const float f = part_weight(__ldcg(&p.stat[at * 32 + r]), M);
          acc = fmaf(f, __ldcg(&p.part[(at * kSplitRows + r) * D + d]), acc);
          sum = fmaf(f, __ldcg(&p.stat[at * 32 + 16 + r]), sum);
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

template <typename T, typename C, int D, int NT>
tf_status launch(const SplitParams& p, int blocks, cudaStream_t s) {
  static PerDeviceOnce attr;
  int dev = 0;
  if (attr.needed(&dev)) {
    TF_CUDA(cudaFuncSetAttribute(paged_split_kernel<T, C, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 Shape<D>::kSmem));
    attr.mark(dev);
  }
  paged_split_kernel<T, C, D, NT><<<blocks, kThreads, Shape<D>::kSmem, s>>>(p);
  return check_launch("paged_split");
}

template <typename T, typename C>
tf_status launch_rows(const SplitParams& p, const tf_paged_plan& plan, cudaStream_t s) {
  // Half the products where no request has more than 8 packed rows.
  if (plan.split_rows <= 8)
    return plan.head_dim == 128 ? launch<T, C, 128, 1>(p, plan.split_blocks, s)
                                : launch<T, C, 64, 1>(p, plan.split_blocks, s);
  return plan.head_dim == 128 ? launch<T, C, 128, 2>(p, plan.split_blocks, s)
                              : launch<T, C, 64, 2>(p, plan.split_blocks, s);
}

// cuTensorMapEncodeTiled, fetched from the driver at run time.
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

}  // namespace

tf_status make_page_map(void* map, const void* base, const tf_paged_kv& kv, int box_rows, int box_columns) {
  const cuuint64_t dims[4] = {64, (cuuint64_t)kv.kv_heads * kv.page_size, (cuuint64_t)kv.head_dim / 64,
                              (cuuint64_t)kv.pages};
  const cuuint64_t strides[3] = {(cuuint64_t)kv.head_dim * 2, 128, (cuuint64_t)kv.page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_columns / 64, 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  const EncodeFn encode = encode_fn();
  if (!encode) return set_error(TF_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const CUresult r = encode(
      static_cast<CUtensorMap*>(map),
      kv.dtype == TF_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
      const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(TF_ERR_CUDA, "paged attention: tensor map (%d)", (int)r);
  return TF_OK;
}

tf_status launch_paged_split(const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  if (plan.split_blocks == 0) return TF_OK;
  SplitParams p;
  memset(&p, 0, sizeof(p));
  p.box_rows = a.kv.page_size < kSplitKeys ? a.kv.page_size : kSplitKeys;
  while ((1 << p.box_shift) < p.box_rows) ++p.box_shift;
  TF_TRY(make_page_map(&p.tm_k, a.kv.k, a.kv, p.box_rows, a.kv.head_dim));
  TF_TRY(make_page_map(&p.tm_v, a.kv.v, a.kv, p.box_rows, a.kv.head_dim));
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
  TF_TRY(tc_flags(&p.err, const_cast<long long**>(&p.wait_cycles)));
  if (a.act == TF_DTYPE_F16) return launch_rows<__half, __half>(p, plan, s);
  if (a.kv.dtype == TF_DTYPE_F16) return launch_rows<__nv_bfloat16, __half>(p, plan, s);
  return launch_rows<__nv_bfloat16, __nv_bfloat16>(p, plan, s);
}

}  // namespace tf
