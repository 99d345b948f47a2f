// Paged attention for many packed rows per key head (prompt chunks, whole
// prompts) on the sm_100a tensor cores: tcgen05 with scores, weights and
// outputs in tensor memory, keys and values by TMA from the pages.
//
// out = softmax(q K^T * scale) V over 128-key tiles with a running maximum m
// and sum l per row; per tile s = q K^T, P = 2^(s * scale * log2 e - m),
// O += P V, l += sum P.  The maximum is refreshed lazily: a row keeps the m it
// used until a tile raises it by more than 7 (log2 units), so P <= 2^7 (in f16
// 2^14: m lies 7 below the maximum, paged_values.cuh) and O is rescaled only on
// such tiles; O / l is the same quotient.
//
// What bounds it: 4 D flops per (row, key) pair on the tensor cores, and one
// exponential per pair on a unit that gives 16 a clock and SM, which is just
// as long (128 x 128 pairs: 1024 clocks of either at D = 128).  Hence
//   * a block holds two halves of 128 rows, each with a softmax warpgroup of
//     its own (thread = row), so one half's products run while the other's
//     exponentials do;
//   * one block per SM walks the segments of the plan (paged.h) and the roles
//     run ahead across them: the next segment's queries and first scores are
//     computed while this one's outputs are written.
// Requests of at most 128 packed rows run the same code with one half a block
// and two blocks an SM: with half B empty, the chain scores - softmax -
// products of half A alone would set the pace, at half of what the pages'
// memory gives (24 requests of 35 rows over 8011 keys: 42 us with
// two halves a block, 36 with one).
//
// Roles (two halves: 384 threads, registers move from the third warpgroup to
// the softmax; one half: 192 threads):
//   warps 0-3, 4-7  softmax of half A, B: read S from tensor memory, mask, write
//              P in 16 bits over S's first columns; after a segment's last
//              scores copy the next segment's queries into shared memory
//              (whole rows by a warp, converted where the cache's type
//              differs), then read O and write out (or the piece's partial
//              result).  A warp of its own for the queries took 9000 clocks a
//              half, most of a short segment.
//   MMA warps   of half A, B: one elected lane issues, tile by tile,
//              O += P V; S = Q K' with K' the next tile.  MMAs of one thread
//              execute in issue order, so a next S may be issued over a P that
//              the product before it still reads, and its completion implies
//              that product's.  A warp each, because the waits between the
//              products (some 150 clocks even when they are met) would leave
//              the tensor cores idle: with the softmax taken out a tile of both
//              halves took 3214 clocks with one warp for both and 2260 with two
//              (2048 at the peak rate).  The halves take turns issuing (baton),
//              which keeps one's softmax beside the other's products; without
//              it both ran in step, 4090 clocks a tile against 3500.  Neither
//              passes it a second time before the other has seen the first.
//   loader     page ids and TMA of the K and V tiles (128-byte
//              swizzle) into one ring of tiles, K and V in turn.
// Tensor memory columns: O_A [0, 128), O_B [128, 256), S_A [256, 384), S_B
// (one half: O [0, 128), S [128, 256)).
//
// P is rounded to the cache's 16-bit type, relative 2^-11 (f16, down to 2^-21 of
// the row's largest) or 2^-8 (bf16), the size of the output's own rounding; l
// sums the unrounded values.
// Every wait is bounded; an expired one records an error code (tf_device_error)
// and all roles stop.
//
// Measured: 2048 tokens after 14336 (32 query and 8 key heads of 128) 424 us,
// 1.22 PFLOP/s (444 us under a profiler: tensor pipe 64% at the 1.58 GHz that the
// power cap leaves); 8 prompts of 2048 tokens (16 heads) 163 us, 0.84 PFLOP/s
// (segments of 9 tiles on average, whose ends cost 5600 clocks each; 4 us of it
// for looking the causal edge's values through, paged_values.cuh), 182 us with
// bf16 queries over an f16 cache.
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

constexpr int kHalf = 128;  // rows of a half = TMEM lanes
constexpr uint32_t kColO = 0;  // half x's columns: O at kColO + 128 x, S after the halves' O
constexpr float kLog2e = 1.4426950408889634f;
// Log2 units that a row's maximum may rise by before O is rescaled (with 8 a sum
// near 2^28, where fp32 has steps of 16, would round up to twice as much).
constexpr float kRescale = 7.f;
constexpr int kColBytes = kTileKeys * 128;  // 64 columns of a tile: 128 rows of 128 bytes

// A block of H halves: two of them one to an SM, or one half two to an SM.
template <int D, int H>
struct Shape {
  static constexpr int kTile = D / 64 * kColBytes;  // bytes of 128 rows or keys
  static constexpr int kSlots = (H == 2 ? 160 : 64) * 1024 / kTile - (H == 2 && D == 64 ? 2 : 0);  // ring of K and V
  static constexpr int kOffRing = H * kTile;        // after the halves' queries
  static constexpr int kOffBar = kOffRing + kSlots * kTile;
  static constexpr int kSmem = kOffBar + 512 + 1024;  // + barriers + alignment slack
  static_assert(kSmem <= 227 * 1024 / (3 - H) - (2 - H) * 1024, "shared memory of an SM");
  // Warps: softmax 0 .. 4 H - 1, then the halves' MMA warps, then the loader
  // (with two halves one more fills the third warpgroup).
  static constexpr int kMmaWarp = 4 * H, kLoadWarp = 5 * H;
  static constexpr int kThreads = H == 2 ? 384 : 192;
  static constexpr uint32_t kColumns = 256 * H, kColS = 128 * H;
  static constexpr int kRows = kHalf * H;
};

struct TileParams {
  CUtensorMap tm_k, tm_v;
  const void* q;
  int64_t q_stride;
  const int32_t* ids;
  int64_t ids_stride;
  int32_t columns;
  int32_t page_size, page_shift;
  int32_t box_rows;  // min(page_size, kTileKeys)
  int32_t group, heads;
  const void* v;  // the value pages, for values that are not finite
  int64_t pages, page_stride;
  const PagedSegment* segments;
  const int32_t* starts;
  float* stat;  // [part][2][rows of a block]: m, l
  float* part;  // [part][D / 4][rows of a block][4]: a warp's rows side by side
  void* out;
  float scale_log2;
  int* err;
  const long long* wait_cycles;
};

struct Control {
  volatile int abort;
  volatile int cleared;  // the block has cleared values that are not finite
  long long limit;
};

// The first try is all that a met wait costs.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Control* c, int* err, int code) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  const long long limit = c->limit;
  while (!mbar_try(bar, parity)) {
    if (c->abort) return false;
    if (clock64() - t0 > limit) {
      atomicCAS(err, 0, code);
      c->abort = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, Control* c, int* err, int code) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, c, err, code));
}
// The block's own copies and MMAs always complete: fixed limit, abort ignored.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity, int* err) {
  if (mbar_try(bar, parity)) return;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity))
    if (clock64() - t0 > 2000000000LL) {
      atomicCAS(err, 0, 89);
      return;
    }
}

// 64 columns (of half `half`) of `row` .. of a page.
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int row, int half, int page,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(half), "r"(page), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// 32 columns, valid only after tmem_wait of the same registers.
__device__ __forceinline__ void tmem_ld32_begin(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
// Waits for every load begun; the registers pass through, so no use of them
// can be scheduled before it.
__device__ __forceinline__ void tmem_wait32(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                 "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                 "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
                 "+f"(v[29]), "+f"(v[30]), "+f"(v[31])::"memory");
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <typename C>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One whole 32-byte sector (a thread's rows are apart, so 16-byte stores would
// touch every sector twice).
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
               "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// A segment as the roles see it: the tiles that each half meets.
template <int H>
struct View {
  int count[H];  // tiles of half A, B, from tile0
  int tiles;     // the larger: tiles that are loaded
  __device__ __forceinline__ View(const PagedSegment& g, int group) {
    tiles = 0;
#pragma unroll
    for (int x = 0; x < H; ++x) {
      count[x] = 0;
      if (kHalf * x >= g.rows) continue;
      const int last_row = g.row0 + min(kHalf * x + kHalf, g.rows) - 1;
      const int last = g.kv_len - g.new_len + last_row / group;  // last key that the half's last row sees
      const int nt = last < 0 ? 0 : last / kTileKeys + 1;
      count[x] = max(0, min(nt, g.tile1) - g.tile0);
      tiles = max(tiles, count[x]);
    }
  }
};

// Adds to a row's stored result (or piece of one, `pitch` rows apart) the
// values that are not finite, of the keys that it sees: a product may have had
// zeros in their place.  Such keys lie past what the segment's first row sees.
template <typename T, typename C, int D>
__device__ __forceinline__ void add_cleared(const TileParams& p, const PagedSegment& g, int limit, T* out, float* part,
                                         int pitch) {
  const int begin = max(g.kv_len - g.new_len + g.row0 / p.group + 1, g.tile0 * kTileKeys);
  const int end = min(min(limit + 1, g.kv_len), g.tile1 * kTileKeys);
  for (int key = begin; key < end; ++key) {
    const int column = key >> p.page_shift;
    const int64_t page = column < p.columns ? p.ids[g.request * p.ids_stride + column] : -1;
    if (page < 0 || page >= p.pages) continue;
    const C* v = static_cast<const C*>(p.v) + page * p.page_stride +
                 (int64_t)(g.kv_head * p.page_size + (key & (p.page_size - 1))) * D;
    for (int c = 0; c < D; c += 8) {
      const uint4 eight = ld_v4(v + c);
      const C* value = reinterpret_cast<const C*>(&eight);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (not_finite(value[k])) {
          if (out)
            out[c + k] = from_f<T>(to_f(out[c + k]) + to_f(value[k]));
          else
            part[(c + k) / 4 * 4 * pitch + (c + k) % 4] += to_f(value[k]);
        }
    }
  }
}

template <typename T, typename C, int D, int H>
__global__ void __launch_bounds__(Shape<D, H>::kThreads, 3 - H)
    paged_tile_kernel(const __grid_constant__ TileParams p) {
  using S = Shape<D, H>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kOffBar);
  uint64_t* q_full = bars;       // [2] 128 threads: the half's query rows are written
  uint64_t* s_full = bars + 2;   // [2] MMA: scores of a tile
  uint64_t* p_full = bars + 4;   // [2][2] 128 threads: a part of P written (before the first, O rescaled)
  uint64_t* o_full = bars + 8;   // [2] MMA, and the warp that issues it: a segment's last product
  uint64_t* o_free = bars + 10;  // [2] 128 threads: O read
  uint64_t* kv_full = bars + 12;             // [slots] TMA
  uint64_t* kv_empty = kv_full + S::kSlots;  // [slots] each half: its products of the tile done
  uint64_t* done = kv_empty + S::kSlots;     // [2] MMA: all products of a half
  uint64_t* baton = done + 2;                // [2] the other half's products of a tile are issued
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(baton + 2);
  Control* ctl = reinterpret_cast<Control*>(baton + 3);
  static_assert((12 + 2 * S::kSlots + 5) * 8 + sizeof(Control) <= 512, "barrier block");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* err = p.err;
  if (tid == 0) {
    for (int x = 0; x < H; ++x) {
      mbar_init(&q_full[x], kHalf);
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[2 * x], kHalf);
      mbar_init(&p_full[2 * x + 1], kHalf);
      mbar_init(&o_full[x], 2);
      mbar_init(&o_free[x], kHalf);
      mbar_init(&done[x], 1);
      mbar_init(&baton[x], 1);
    }
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], H);
    }
    ctl->abort = 0;
    ctl->cleared = 0;
    ctl->limit = *p.wait_cycles;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == S::kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(S::kColumns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (warp == S::kLoadWarp && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&p.tm_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&p.tm_v)) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int seg0 = p.starts[blockIdx.x], seg1 = p.starts[blockIdx.x + 1];

  if (warp >= S::kMmaWarp) {
    // 384 threads x 168 registers = 2 x 128 x 208 + 128 x 88.
    if constexpr (H == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == S::kLoadWarp) {
      int n = 0;  // tiles fetched (K and V each count)
      bool ok = true;
      for (int seg = seg0; seg < seg1 && ok; ++seg) {
        const PagedSegment g = p.segments[seg];
        const View<H> view(g, p.group);
        const int32_t* ids = p.ids + g.request * p.ids_stride;
        const int box_bytes = p.box_rows * 128;
        for (int j = 0; j < view.tiles && ok; ++j) {
          const int key0 = (g.tile0 + j) * kTileKeys;
          const int left = g.kv_len - key0;
          const int boxes = ((left < kTileKeys ? left : kTileKeys) + p.box_rows - 1) / p.box_rows;
          // Lane i fetches box i (at most 16 of the tile's pages).
          int page = -1, row = 0;
          if (lane < boxes) {
            const int key = key0 + lane * p.box_rows, column = key >> p.page_shift;
            if (column < p.columns) page = __ldg(ids + column);
            row = g.kv_head * p.page_size + (key & (p.page_size - 1));
          }
#pragma unroll
          for (int v = 0; v < 2; ++v, ++n) {
            const int slot = n % S::kSlots, turn = n / S::kSlots;
            if (turn > 0 && !(ok = wait_warp(&kv_empty[slot], (uint32_t)((turn - 1) & 1), ctl, err, 81))) break;
            if (lane == 0) mbar_expect_tx(&kv_full[slot], (uint32_t)(boxes * box_bytes * (D / 64)));
            __syncwarp();
            if (lane < boxes) {
              uint8_t* dst = base + S::kOffRing + slot * S::kTile + lane * box_bytes;
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
                tma_page(dst + h * kColBytes, v ? &p.tm_v : &p.tm_k, row, h, page, &kv_full[slot]);
            }
          }
        }
      }
      // Copies in flight land before the block exits.
      for (int i = n > S::kSlots ? n - S::kSlots : 0; i < n; ++i)
        drain(&kv_full[i % S::kSlots], (uint32_t)((i / S::kSlots) & 1), err);
    } else if (warp < S::kLoadWarp) {
      // ---- products of half x.
      const int x = warp - S::kMmaWarp;
      const uint32_t leader = elect_one();
      const uint32_t fmt = Act<C>::kDtype == TF_DTYPE_BF16 ? (1u << 7) | (1u << 10) : 0u;  // A and B are bf16
      const uint32_t id_qk = idesc_f16(kHalf, kTileKeys) | fmt;
      const uint32_t id_pv = idesc_f16(kHalf, D) | (1u << 16) | fmt;  // B (V) MN-major
      const uint32_t t_o = tmem + kColO + 128 * x, t_s = tmem + S::kColS + 128 * x;
      const uint32_t qa = smem_addr(base + x * S::kTile);
      int n = 0;  // ring position
      uint32_t q_turn = 0, p_turn = 0, o_turn = 0, baton_turn = 0;
      bool ok = true;
      auto landed = [&](int at) {  // tile `at` of the ring is there
        return wait_warp(&kv_full[at % S::kSlots], (uint32_t)((at / S::kSlots) & 1), ctl, err, 82);
      };
      auto scores = [&](int at) {
        const int slot = at % S::kSlots;
        const uint32_t ka = smem_addr(base + S::kOffRing + slot * S::kTile);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          const uint32_t off = (uint32_t)((s >> 2) * kColBytes + (s & 3) * 32);
          mma_f16(leader, t_s, sw128_desc(qa + off), sw128_desc(ka + off), id_qk, s > 0 ? 1u : 0u);
        }
        mma_commit(leader, &s_full[x]);
        mma_commit(leader, &kv_empty[slot]);
      };
      for (int seg = seg0; seg < seg1 && ok; ++seg) {
        const PagedSegment g = p.segments[seg];
        const View<H> view(g, p.group);
        const int count = view.count[x];
        if (count > 0) {
          if (!(ok = landed(n) && wait_warp(&q_full[x], q_turn & 1, ctl, err, 83))) break;
          ++q_turn;
          tc_fence_after();
          scores(n);
        }
        // First key, from the segment's first, that not all rows of the half see.
        const int hidden0 = g.kv_len - g.new_len + (g.row0 + kHalf * x) / p.group + 1 - g.tile0 * kTileKeys;
        const int both = H == 2 ? min(count, view.count[(1 - x) & (H - 1)]) : 0;  // tiles that both halves meet
        for (int j = 0; j < count && ok; ++j) {
          // Ring: K of tile j at n, V of tile j, K of tile j + 1.
          const bool more = j + 1 < count;
          if (!(ok = landed(n + 1) && (!more || landed(n + 2)))) break;
          const int vs = (n + 1) % S::kSlots;
          uint8_t* vt = base + S::kOffRing + vs * S::kTile;
          const int have = g.kv_len - (g.tile0 + j) * kTileKeys;
          if (have < kTileKeys) {
            // Slots past the request's length hold anything, NaN included:
            // 0 * NaN would reach the outputs, so their values become zeros
            // (by both halves' warps, each before its own products).
            for (int i = have * 8 + lane; i < kTileKeys * 8; i += 32)
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
                *reinterpret_cast<uint4*>(vt + h * kColBytes + 16 * i) = make_uint4(0, 0, 0, 0);
            fence_proxy_async();
            __syncwarp();
          }
          // Keys that some row of the half does not see, with values that are
          // not finite (the other half may read them cleared as well).
          const int hidden = max(hidden0 - j * kTileKeys, 0);
          const int chunks = (min(have, kTileKeys) - hidden) * 8;  // of a column half
          if (chunks > 0) {
            uint8_t* first = vt + hidden * 128;
            bool finite = true;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) finite &= all_finite<C>(first + h * kColBytes, chunks, lane);
            if (!finite) {
              if (lane == 0) ctl->cleared = 1;
              __threadfence_block();
#pragma unroll
              for (int h = 0; h < D / 64; ++h) clear_not_finite<C>(first + h * kColBytes, chunks, lane);
              fence_proxy_async();
              __syncwarp();
            }
          }
          // O still holds the half's last segment until it has been read.
          if (j == 0 && o_turn++ > 0 && !(ok = wait_warp(&o_free[x], o_turn & 1, ctl, err, 86))) break;
          const uint32_t va = smem_addr(vt);
          if (j < both) {
            // Half A waits for B's turn before its own, but for the block's first.
            if ((x == 1 || baton_turn > 0) &&
                !(ok = wait_warp(&baton[x], (baton_turn - (1 - x)) & 1, ctl, err, 87)))
              break;
            ++baton_turn;
            // At a segment's end half B says that it has seen A's: without a word
            // A would pass the baton again in the next segment, and B, held up
            // by its outputs, would miss a phase and wait for good.
            if (x == 1 && j + 1 == both && lane == 0) mbar_arrive(&baton[0]);
          }
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            if (!(ok = wait_warp(&p_full[2 * x + part], p_turn & 1, ctl, err, 85))) break;
            tc_fence_after();
#pragma unroll
            for (int s = 4 * part; s < 4 * part + 4; ++s)
              mma_f16_ts(leader, t_o, t_s + 8 * s, sw128_mn_desc(va + s * 2048, kColBytes, 1024), id_pv,
                         (j > 0 || s > 0) ? 1u : 0u);
          }
          if (!ok) break;
          ++p_turn;
          mma_commit(leader, &kv_empty[vs]);
          if (more) {
            scores(n + 2);
          } else {
            mma_commit(leader, &o_full[x]);
            if (lane == 0) mbar_arrive(&o_full[x]);
          }
          if (lane == 0 && (x == 0 ? j < both : j + 1 < both)) mbar_arrive(&baton[1 - x]);
          n += 2;
        }
        // Tiles that only the other half meets: released once they are there,
        // so this warp never runs a turn of the ring ahead.
        for (int j = count; j < view.tiles && ok; ++j)
          for (int v = 0; v < 2 && ok; ++v, ++n)
            if ((ok = landed(n)) && lane == 0) mbar_arrive(&kv_empty[n % S::kSlots]);
      }
      // Every MMA issued here completes before tensor memory is released.
      mma_commit(leader, &done[x]);
      drain(&done[x], 0, err);
    }
  } else {
    if constexpr (H == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax of half x: thread r owns row r = TMEM lane r.
    const int x = warp >> 2;
    const int r = tid - kHalf * x;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_o = lane_base + kColO + 128 * x, t_s = lane_base + S::kColS + 128 * x;
    uint32_t s_turn = 0, o_turn = 0;
    bool ok = true;
    // Copies the query rows of the half's next segment with tiles, from
    // segment `seg` on, into the K-major 128-byte swizzle: row i of each
    // 64-column half at i * 128, 16-byte chunk c at (c ^ (i & 7)) * 16.  A warp
    // copies its 32 rows whole rows at a time; rows past the segment's become
    // zeros.  Leaves what the own row's scores are to be multiplied with.
    float boost = 1.f;
    auto copy_queries = [&](int seg) {
      constexpr int kChunks = D / 8, kRowsAt = 32 / kChunks;  // chunks of a row, rows per pass
      for (; seg < seg1; ++seg) {
        const PagedSegment g = p.segments[seg];
        if (View<H>(g, p.group).count[x] == 0) continue;
        const int pr = g.row0 + min(kHalf * x + r, g.rows - 1);
        const T* own = static_cast<const T*>(p.q) + (int64_t)(g.q_row + pr / p.group) * p.q_stride +
                       (int64_t)(g.kv_head * p.group + pr % p.group) * D;
        const int c = lane % kChunks;
        uint8_t* to = base + x * S::kTile + (c >> 3) * kColBytes;
        constexpr int kBatch = 8;  // rows' loads in flight
        static_assert(32 / kRowsAt % kBatch == 0, "batches");
        boost = 1.f;
#pragma unroll 1
        for (int i0 = 0; i0 < 32 / kRowsAt; i0 += kBatch) {
          uint4 values[kBatch];
          uint32_t most[kBatch], all = 0;
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int from = (i0 + b) * kRowsAt + lane / kChunks;  // lane whose row this is
            const T* q = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(own), from)) + 8 * c;
            const int row = (warp & 3) * 32 + from;
            const bool real = kHalf * x + row < g.rows;
            if constexpr (Act<T>::kDtype == Act<C>::kDtype) {
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                               smem_addr(to + row * 128 + (((c & 7) ^ (row & 7)) << 4))),
                           "l"(q), "r"(real ? 16 : 0)
                           : "memory");
            } else {
              values[b] = real ? ld_v4(q) : make_uint4(0, 0, 0, 0);
            }
          }
          if constexpr (Act<T>::kDtype != Act<C>::kDtype) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              const uint4 v = values[b];
              most[b] = magnitude(v.w, magnitude(v.z, magnitude(v.y, magnitude(v.x, 0))));
              all = max(all, most[b]);
            }
            const bool wide = __any_sync(0xffffffffu, beyond_f16(all) > 0);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              float f[8];
              unpack8<T>(values[b], f);
              if (wide) {
#pragma unroll
                for (int off = 1; off < kChunks; off <<= 1) most[b] = max(most[b], __shfl_xor_sync(0xffffffffu, most[b], off));
                const int over = beyond_f16(most[b]);
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] *= power2(-over);
                const int mine = __shfl_sync(0xffffffffu, over, lane % kRowsAt * kChunks);
                if (lane / kRowsAt == i0 + b) boost = power2(mine);
              }
              const int row = (warp & 3) * 32 + (i0 + b) * kRowsAt + lane / kChunks;
              *reinterpret_cast<uint4*>(to + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = pack8<C>(f);
            }
          }
        }
        if constexpr (Act<T>::kDtype == Act<C>::kDtype) asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async();
        mbar_arrive(&q_full[x]);
        return;
      }
    };
    copy_queries(seg0);
    for (int seg = seg0; seg < seg1 && ok; ++seg) {
      const PagedSegment g = p.segments[seg];
      if (kHalf * x >= g.rows) continue;
      const View<H> view(g, p.group);
      const int count = view.count[x];
      // Threads past the rows follow the last one; what they make is dropped.
      const int pr = g.row0 + min(kHalf * x + r, g.rows - 1);
      const int token = pr / p.group;
      const int limit = g.kv_len - g.new_len + token;  // last key the row sees
      const int first_limit = g.kv_len - g.new_len + (g.row0 + kHalf * x) / p.group;
      const float scale = Act<T>::kDtype == Act<C>::kDtype ? p.scale_log2 : p.scale_log2 * boost;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < count; ++j) {
        if (!(ok = wait_warp(&s_full[x], s_turn & 1, ctl, err, 90))) break;
        ++s_turn;
        tc_fence_after();
        float sc[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32_begin(t_s + c, sc + c);
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_wait32(sc + c);
        const int key0 = (g.tile0 + j) * kTileKeys;
        if (key0 + kTileKeys - 1 > first_limit) {
          const int lim = limit - key0;  // later columns are masked
#pragma unroll
          for (int c = 0; c < 128; ++c) sc[c] = c > lim ? -INFINITY : sc[c];
        }
        // The maximum of the raw scores (the scale is positive), NaN kept.
        float mp[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mp[i] = max_nan(sc[2 * i], sc[2 * i + 1]);
#pragma unroll
        for (int c = 16; c < 128; c += 16)
#pragma unroll
          for (int i = 0; i < 8; ++i) mp[i] = max_nan(mp[i], sc[c + 2 * i], sc[c + 2 * i + 1]);
        float mx = max_nan(max_nan(mp[0], mp[1], mp[2]), max_nan(mp[3], mp[4], mp[5]), max_nan(mp[6], mp[7])) *
                   scale;
        if (mx == INFINITY) mx = __uint_as_float(0x7fc00000u);  // inf - inf: the row is NaN
        // Far out the product with the scale is rounded by more than the
        // exponential bears: there each score takes the maximum's rounding.
        float unit = scale;
        if (__any_sync(0xffffffffu, fabsf(mx) > kFar)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) sc[c] *= scale;
          unit = 1.f;
        }
        float factor = 1.f;
        mx = lifted<C>(mx);
        if (!(mx <= m + kRescale)) {  // also for NaN, and for the first key seen
          mx = max_nan(m, mx);  // a NaN stays
          factor = fast_exp2(m - mx);
          m = mx;
          l *= factor;
        }
        // This tile's scores were issued after the last tile's product: O is
        // stable, and P may overlay S.  (The vote is taken on the first tile too:
        // it brings the warp together for the stores of P.)
        if (__any_sync(0xffffffffu, factor != 1.f) && j > 0) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32];
            tmem_ld32(t_o + c, o);
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(o[i] * factor);
            tmem_st16(t_o + c, w);
            tmem_st16(t_o + c + 16, w + 16);
          }
        }
        // Exponent arguments and sums on packed pairs.  P goes out in two
        // parts of 64 keys, so the product of the first runs while the
        // second's exponentials do.
        const float sub = m == -INFINITY ? 0.f : -m;
        const uint64_t sl2 = f2_pack(unit, unit), nm = f2_pack(sub, sub);
        uint64_t sp[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sp[i] = 0ull;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int k0 = 64 * half + 2 * c;
            float a, b;
            f2_unpack(f2_fma(f2_pack(sc[k0], sc[k0 + 1]), sl2, nm), a, b);
            a = fast_exp2(a);
            b = fast_exp2(b);
            sp[c & 3] = f2_add(sp[c & 3], f2_pack(a, b));
            pk[c] = pack2<C>(a, b);
          }
          tmem_st16(t_s + 32 * half, pk);
          tmem_st16(t_s + 32 * half + 16, pk + 16);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&p_full[2 * x + half]);
        }
        float s0, s1;
        f2_unpack(f2_add(f2_add(sp[0], sp[1]), f2_add(sp[2], sp[3])), s0, s1);
        l += s0 + s1;
      }
      if (!ok) break;
      const int row = kHalf * x + r;
      const bool mine = row < g.rows;
      if (count > 0) {
        copy_queries(seg + 1);  // the last scores are done, so the rows' place is free
        if (!(ok = wait_warp(&o_full[x], o_turn & 1, ctl, err, 91))) break;
        ++o_turn;
        tc_fence_after();
      }
      const bool cleared = ctl->cleared != 0;
      // A row that has seen no key above -inf gives zeros.
      const float inv = m == -INFINITY ? 0.f : 1.f / l;
      T* orow = static_cast<T*>(p.out) +
                ((int64_t)(g.q_row + token) * p.heads + g.kv_head * p.group + pr % p.group) * D;
      float* prow = p.part + (int64_t)g.part * S::kRows * D + row * 4;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (count > 0) {
          tmem_ld32(t_o + c, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (mine && g.part < 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            float f[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) f[k] = m == -INFINITY ? 0.f : o[i + k] * inv;
            store32(orow + c + i, pack8<T>(f), pack8<T>(f + 8));
          }
        } else if (mine) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(prow + (c + i) * S::kRows) =
                make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
        __syncwarp();  // the next load takes the whole warp, also where the rows end inside it
      }
      if (cleared) {
        if (mine && m != -INFINITY)
          add_cleared<T, C, D>(p, g, limit, g.part < 0 ? orow : nullptr, prow, S::kRows);
        __syncwarp();
      }
      if (mine && g.part >= 0) {
        p.stat[(int64_t)g.part * 2 * S::kRows + row] = m;
        p.stat[(int64_t)g.part * 2 * S::kRows + S::kRows + row] = l;
      }
      if (count > 0) {
        tc_fence_before();
        mbar_arrive(&o_free[x]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // This kernel may have begun while the few-rows kernel before it still ran
  // (it needs none of its results); what follows counts on both.
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == S::kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns));
}

// Joins the pieces of cut row blocks, in piece order.  A warp takes 32 rows
// and 4 columns, so the pieces' outputs arrive 512 bytes at a time.
constexpr int kMergeWarps = 8;

template <typename T, int D, int R>
__global__ void __launch_bounds__(32 * kMergeWarps)
    paged_merge_kernel(const PagedSegment* items, const float* stat, const float* part, int group, int heads,
                       T* out) {
  const PagedSegment g = items[blockIdx.z];
  const int row = blockIdx.x * 32 + (threadIdx.x & 31);
  const int c = blockIdx.y * kMergeWarps + (threadIdx.x >> 5);  // columns 4 c ..
  if (row >= g.rows) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the pieces are written
  const float* st = stat + (int64_t)g.part0 * 2 * R + row;
  const float* o = part + (int64_t)g.part0 * R * D + (c * R + row) * 4;
  float M = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < g.parts; ++i) M = max_nan(M, st[(int64_t)i * 2 * R]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < g.parts; ++i) {
    const float m = st[(int64_t)i * 2 * R];
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - M);  // an empty piece holds zeros
    const float4 v = *reinterpret_cast<const float4*>(o + (int64_t)i * R * D);
    sum = fmaf(f, st[(int64_t)i * 2 * R + R], sum);
    acc.x = fmaf(f, v.x, acc.x);
    acc.y = fmaf(f, v.y, acc.y);
    acc.z = fmaf(f, v.z, acc.z);
    acc.w = fmaf(f, v.w, acc.w);
  }
  const float inv = M == -INFINITY ? 0.f : 1.f / sum;
  const int pr = g.row0 + row;
  T* to = out + ((int64_t)(g.q_row + pr / group) * heads + g.kv_head * group + pr % group) * D + 4 * c;
  alignas(8) const T v[4] = {from_f<T>(acc.x * inv), from_f<T>(acc.y * inv), from_f<T>(acc.z * inv), from_f<T>(acc.w * inv)};
  *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(v);
}

// The work of one kind of block in a plan.
struct Work {
  int64_t segments, starts, merges;  // offsets in the table
  int32_t blocks, parts, cuts;
  float* stat;
};

template <typename T, typename C, int D, int H>
tf_status launch(TileParams p, const Work& w, const char* table, bool early, cudaStream_t s) {
  using S = Shape<D, H>;
  if (w.blocks == 0) return TF_OK;
  static PerDeviceOnce attr;
  int dev = 0;
  if (attr.needed(&dev)) {
    TF_CUDA(cudaFuncSetAttribute(paged_tile_kernel<T, C, D, H>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 S::kSmem));
    attr.mark(dev);
  }
  p.segments = reinterpret_cast<const PagedSegment*>(table + w.segments);
  p.starts = reinterpret_cast<const int32_t*>(table + w.starts);
  p.stat = w.stat;
  p.part = p.stat + (int64_t)w.parts * 2 * S::kRows;
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)w.blocks);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cfg.attrs = &overlap;
  cfg.numAttrs = early ? 1 : 0;
  TF_CUDA(cudaLaunchKernelEx(&cfg, paged_tile_kernel<T, C, D, H>, p));
  TF_TRY(check_launch("paged_tile"));
  if (w.cuts == 0) return TF_OK;
  // grid.z is below 65536: at most one cut item per block.
  const dim3 grid(S::kRows / 32, D / 4 / kMergeWarps, (unsigned)w.cuts);
  // The merge is launched while the pieces' last blocks still run and waits on
  // the device for them.
  cfg = cudaLaunchConfig_t{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.stream = s;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  TF_CUDA(cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, D, S::kRows>,
                             reinterpret_cast<const PagedSegment*>(table + w.merges), (const float*)p.stat,
                             (const float*)p.part, p.group, p.heads, static_cast<T*>(p.out)));
  return check_launch("paged_merge");
}

template <typename T, typename C, int D>
tf_status launch_both(const TileParams& p, const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  float* stat = reinterpret_cast<float*>(a.workspace + split_workspace_bytes(plan));
  const Work tile = {plan.tile_segments_offset, plan.tile_starts_offset, plan.tile_merges_offset,
                     plan.tile_blocks, plan.tile_parts, plan.tile_merges, stat};
  const Work half = {plan.half_segments_offset, plan.half_starts_offset, plan.half_merges_offset,
                     plan.half_blocks, plan.half_parts, plan.half_merges,
                     stat + (int64_t)plan.tile_parts * kTileRows * (2 + D)};
  // The first kernel after the few-rows kernel starts on the SMs that it leaves.
  const bool after_split = plan.split_blocks > 0;
  TF_TRY((launch<T, C, D, 2>(p, tile, a.plan_table, after_split, s)));
  return launch<T, C, D, 1>(p, half, a.plan_table, after_split && plan.tile_blocks == 0, s);
}

}  // namespace

tf_status launch_paged_tile(const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  if (plan.tile_blocks == 0 && plan.half_blocks == 0) return TF_OK;
  TileParams p;
  memset(&p, 0, sizeof(p));
  p.box_rows = a.kv.page_size < kTileKeys ? a.kv.page_size : kTileKeys;
  TF_TRY(make_page_map(&p.tm_k, a.kv.k, a.kv, p.box_rows, 64));
  TF_TRY(make_page_map(&p.tm_v, a.kv.v, a.kv, p.box_rows, 64));
  p.q = a.q;
  p.q_stride = a.q_stride;
  p.ids = a.table.ids;
  p.ids_stride = a.table.stride;
  p.columns = a.table.columns;
  p.page_size = a.kv.page_size;
  while ((1 << p.page_shift) < a.kv.page_size) ++p.page_shift;
  p.group = plan.heads / plan.kv_heads;
  p.heads = plan.heads;
  p.v = a.kv.v;
  p.pages = a.kv.pages;
  p.page_stride = a.kv.page_stride;
  p.out = a.out;
  p.scale_log2 = a.scale * kLog2e;
  TF_TRY(tc_flags(&p.err, const_cast<long long**>(&p.wait_cycles)));
#define TF_TILE(T, C) return plan.head_dim == 128 ? launch_both<T, C, 128>(p, a, s) : launch_both<T, C, 64>(p, a, s)
  if (a.act == TF_DTYPE_F16) TF_TILE(__half, __half);
  if (a.kv.dtype == TF_DTYPE_F16) TF_TILE(__nv_bfloat16, __half);
  TF_TILE(__nv_bfloat16, __nv_bfloat16);
#undef TF_TILE
}

}  // namespace tf
