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
// An 8-bit cache (C = f16): codes widen to f16 exactly, and the scales of a
// tile's 16-token blocks go to the softmax: s_k into the factor of the exponent's
// argument and of the block's maximum, and s_v / r into the weights as a summand
// log2(s_v / r) of the argument, which the row's sum takes out again block by
// block: P' = 2^(s s_k - m + log2(s_v / r)), l += (r / s_v) sum P', O += P' V.
// m is the maximum of s s_k + log2(s_v / r): the largest share of an output is a
// P' of 2^7 and not rounded in the tile that sets m, which counts where few keys do
// (f16 outputs are off by 1.1 to 1.3 times their own rounding; with m the scores'
// maximum 1.4 to 1.6, and 2048 of 16384 took 3% less).
// That costs a few instructions a block, none a score, and rounds nothing but P'.
// r is a power of two at or above the segment's value scales (one half: those so
// far; where it grows, m falls by as much).  Where they lie more than 2^61 apart
// (or are zero), r / s_v no longer serves: keys with a tiny scale may hold all of a
// row's weight, or none of it beside a large one that counts, or one that the row
// does not see.  (Where scores are far out, from 2^13 on.)  Then l sums 2^(s s_k - m) itself, m is the scores' own maximum, and
// O stands at 2^(m + kappa), kappa the largest (s s_k - m) + log2(s_v / r): twice the
// exponentials, on such segments (one half: from such a tile on).
//   Two halves (storage Widened): the requests' codes are widened by a kernel of
// their own first (paged_widen.cu), for the tensor cores are the limit and a
// tile is read by many row blocks.  (Widened in this kernel by a warpgroup more,
// 2048 tokens of 16384 took 702 us; shared memory then carries 96 KB more a tile
// beside the products' 192, and without that work it were 568.)
//   One half (storage I8 or E4M3): two warps more widen the tiles on their way,
// from a small ring of codes that TMA fills into the ring that the products read.
//
// Every wait is bounded; an expired one records an error code (tf_device_error)
// and all roles stop.
//
// Measured: 2048 tokens after 14336 (32 query and 8 key heads of 128) 424 us,
// 1.22 PFLOP/s (444 us under a profiler: tensor pipe 64% at the 1.58 GHz that the
// power cap leaves); 8 prompts of 2048 tokens (16 heads) 163 us, 0.84 PFLOP/s
// (segments of 9 tiles on average, whose ends cost 5600 clocks each; 4 us of it
// for looking the causal edge's values through, paged_values.cuh), 182 us with
// bf16 queries over an f16 cache.  Over int8 codes (bf16 queries) the first takes
// 539 us, widening included, where f16 keys and values take 443; the prompts 252 to
// 262 against 182, with f16 queries 230 against 166; 35 rows each of 24 requests (8
// heads of 128, 8011 tokens, one half) 188 to 197 against 142 to 150.
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

constexpr int kHalf = 128;  // rows of a half = TMEM lanes
constexpr uint32_t kColO = 0;  // half x's columns: O at kColO + 128 x, S after the halves' O
constexpr float kLog2e = 1.4426950408889634f;
// Log2 units that a row's maximum may rise by before O is rescaled (with 8 a sum
// near 2^28, where fp32 has steps of 16, would round up to twice as much).
constexpr float kRescale = 7.f;
constexpr int kColBytes = kTileKeys * 128;  // 64 columns of a tile: 128 rows of 128 bytes

// f16 numbers that are codes: what a request's codes were widened to.
struct Widened {
  uint16_t bits;
};

// A block of H halves: two of them one to an SM, or one half two to an SM.  St:
// what is read; the products' type C, or codes (widened here, or before).
template <int D, int H, typename C, typename St>
struct Shape {
  static constexpr bool kScaled = !std::is_same<St, C>::value;
  static constexpr bool kWiden = kScaled && !std::is_same<St, Widened>::value;
  static_assert(!kWiden || H == 1, "two halves read widened codes");
  static constexpr int kTile = D / 64 * kColBytes;  // bytes of 128 rows or keys
  // Ring of K and V.
  static constexpr int kSlots = (H == 2 ? 160 : 64) * 1024 / kTile - (H == 2 && D == 64 ? 2 : 0);
  // Ring of codes: a slot holds that many keys (or values).
  static constexpr int kRawKeys = D == 128 ? 64 : kTileKeys;
  static constexpr int kRaw = kRawKeys * D;
  static constexpr int kRawSlots = kWiden ? 2 : 0;
  static constexpr int kOffRing = H * kTile;        // after the halves' queries
  static constexpr int kOffRaw = kOffRing + kSlots * kTile;
  static constexpr int kOffBar = kOffRaw + kRawSlots * kRaw;
  static constexpr int kBarBytes = !kScaled ? 512 : H == 2 || D == 64 ? 2048 : 1024;
  // + barriers + alignment slack.  (Two blocks with a ring of codes have no room for
  // the slack; without static shared memory the base is aligned, and checked.)
  static constexpr int kSlack = kWiden ? 0 : 1024;
  static constexpr int kSmem = kOffBar + kBarBytes + kSlack;
  static_assert(kSmem <= 227 * 1024 / (3 - H) - (2 - H) * (kWiden ? 512 : 1024), "shared memory of an SM");
  // Warps: softmax 0 .. 4 H - 1, then the halves' MMA warps, then the loader
  // (with two halves one more fills the third warpgroup), then the wideners.
  static constexpr int kMmaWarp = 4 * H, kLoadWarp = 5 * H;
  static constexpr int kWidenWarp = 6, kWideners = 64;
  static constexpr int kThreads = H == 2 ? 384 : kWiden ? 256 : 192;
  static constexpr uint32_t kColumns = 256 * H, kColS = 128 * H;
  static constexpr int kRows = kHalf * H;
  // Tiles whose scales are kept: more than lie between the loader and the softmax.
  static constexpr int kTold = H == 2 ? 8 : D == 64 ? 4 : 2;
};

struct TileParams {
  CUtensorMap tm_k, tm_v;
  const void* q;
  int64_t q_stride;
  const int32_t* ids;
  int64_t ids_stride;
  int32_t columns;
  int32_t page_size, page_shift;
  int32_t box_rows;  // min(page_size, kTileKeys), of codes min(page_size, 64)
  int32_t group, heads;
  const void* v;  // the value pages, for values that are not finite
  int64_t pages, page_stride;
  const PagedSegment* segments;
  const int32_t* starts;
  float* stat;  // [part][2][rows of a block]: m, l
  float* part;  // [part][D / 4][rows of a block][4]: a warp's rows side by side
  void* out;
  float scale_log2;
  int least_power;  // power_floor of the scale
  int* err;
  const long long* wait_cycles;
  const float* k_scales;  // of codes: [page][kv_head][block], or of widened ones: [kv_head][block]
  const float* v_scales;
  int64_t scale_stride;   // from page to page, from head to head
  const int32_t* first_page;  // of each request's widened codes
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

// What is told of a tile of codes, twice where packed pairs are worked on.  Zero
// units become the smallest number, 2^-149 (a hidden score of -inf must not meet a
// zero); of blocks past the request's length, or with scales that are not finite
// (the rows that see a token of theirs become NaN), the rest is 1.
struct TileScales {
  float4 block[8];  // unit, unit, offset, offset: s_k * scale * log2 e, log2(s_v / r)
  float2 back[8];   // r / s_v
  float v_ref;      // r
  float fall;       // log2(r of the tile before / r)
  uint32_t events;  // bit b: a scale of block b is not finite; bit 8: r grew; bit 9: scales are far apart; bit 10:
                    // too far for scores far out
  uint32_t pad;
};
constexpr uint32_t kGrew = 256, kWide = 512, kSpread = 1024;
// Up to 2^9 a maximum and a logarithm add up to within 2^-15, 2e-5 of a weight.
constexpr float kApart = 512.f;
// The value scales of a segment (one half: those so far).
struct ScalesSeen {
  float ref = kLeastRef;    // r
  float lowest = INFINITY;
  bool wide = false;        // from here on l has a reference of its own
  __device__ __forceinline__ void add(float most, float least) {
    if (most > ref) ref = power_above(most);
    lowest = fminf(lowest, least);
    wide = wide || far_apart(lowest, ref);
  }
};
// Lane i of a warp, i < 8, has the scales of block i (the other lanes those of
// i % 8); the request's length ends in or after block `blocks` - 1.
__device__ __forceinline__ void tell(TileScales& to, float k, float v, float scale, ScalesSeen& seen, int blocks, int lane) {
  const bool there = (lane & 7) < blocks;
  const bool odd = there && !(fabsf(k) < INFINITY && fabsf(v) < INFINITY);
  const bool real = there && !odd;
  if (odd) k = 0.f;
  float most = real ? v : 0.f, least = real ? v : INFINITY;
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, off));
  }
  const float before = seen.ref;
  seen.add(most, least);
  const uint32_t odds = __ballot_sync(0xffffffffu, odd) & 0xffu;
  if (lane < 8) {
    const float unit = fmaxf(k * scale, 1.401298464e-45f), some = real ? v * inverse_of(seen.ref) : 1.f;
    const float offset = real && seen.wide ? log2f(v) - exponent_of(seen.ref) : log2f(some), back = 1.f / some;
    to.block[lane] = make_float4(unit, unit, offset, offset);
    to.back[lane] = make_float2(back, back);
    if (lane == 0) {
      to.v_ref = seen.ref;
      to.fall = exponent_of(before) - exponent_of(seen.ref);
      to.events = odds | (seen.ref != before ? kGrew : 0u) | (seen.wide ? kWide : 0u) |
                  (seen.lowest < seen.ref * kFarRatio ? kSpread : 0u);
    }
  }
}

// Whether a row that sees the tile's first `last` + 1 keys sees one of a block whose
// scale is not finite.
__device__ __forceinline__ bool sees_odd(uint32_t events, int last) {
  return last >= 0 && (events & ((2u << min(last / kScaleTokens, 7)) - 1u) & 0xffu);
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

// A warp's rows of O times a factor each.
template <int D>
__device__ __forceinline__ void rescale(uint32_t t_o, float factor) {
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

template <typename T, typename C, int D, int H, typename St>
__global__ void __launch_bounds__(Shape<D, H, C, St>::kThreads, 3 - H)
    paged_tile_kernel(const __grid_constant__ TileParams p) {
  using S = Shape<D, H, C, St>;
  constexpr bool kScaled = S::kScaled, kWiden = S::kWiden;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (S::kSlack == 0 && base != smem_raw) {  // does not happen
    if (threadIdx.x == 0) atomicCAS(p.err, 0, 92);
    return;
  }
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
  uint64_t* raw_full = baton + 6;               // [raw slots] TMA, and each lane's scales
  uint64_t* raw_empty = raw_full + S::kRawSlots;  // [raw slots] each warp of the wideners
  float* scales = reinterpret_cast<float*>(raw_empty + S::kRawSlots);  // [4 tiles][k, v][8]
  TileScales* told = reinterpret_cast<TileScales*>(scales + (kWiden ? 64 : 0));  // [kTold tiles]
  static_assert((12 + 2 * S::kSlots + 5) * 8 + sizeof(Control) <= 512, "barrier block");
  static_assert(!kScaled || (20 + 2 * S::kSlots + 2 * S::kRawSlots) * 8 + (kWiden ? 256 : 0) +
                                    S::kTold * sizeof(TileScales) <= S::kBarBytes, "barrier block");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* err = p.err;
  if (tid == 0) {
    for (int x = 0; x < H; ++x) {
      mbar_init(&q_full[x], kHalf);
      mbar_init(&s_full[x], kScaled ? 2 : 1);
      mbar_init(&p_full[2 * x], kHalf);
      mbar_init(&p_full[2 * x + 1], kHalf);
      mbar_init(&o_full[x], 2);
      mbar_init(&o_free[x], kHalf);
      mbar_init(&done[x], 1);
      mbar_init(&baton[x], 1);
    }
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(&kv_full[i], kWiden ? S::kWideners : 1);
      mbar_init(&kv_empty[i], H);
    }
    for (int i = 0; i < S::kRawSlots; ++i) {
      mbar_init(&raw_full[i], 33);
      mbar_init(&raw_empty[i], S::kWideners / 32);
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
    // 384 threads x 168 registers = 2 x 128 x 208 + 128 x 88, of codes 2 x 128 x 200 +
    // 128 x 104 (with 208 the softmax of f16 queries spilled); with wideners 256 x 128 =
    // 128 x 192 + 128 x 64.
    if constexpr (kWiden)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    else if constexpr (H == 2 && kScaled)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    else if constexpr (H == 2)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (kWiden && warp == S::kLoadWarp) {
      if constexpr (kWiden) {
        constexpr int kChunks = kTileKeys / S::kRawKeys;
        int m = 0, t = 0;  // chunks and tiles fetched
        bool ok = true;
        for (int seg = seg0; seg < seg1 && ok; ++seg) {
          const PagedSegment g = p.segments[seg];
          const View<H> view(g, p.group);
          const int32_t* ids = p.ids + g.request * p.ids_stride;
          const int box_bytes = p.box_rows * D;
          for (int j = 0; j < view.tiles && ok; ++j, ++t) {
            const int key0 = (g.tile0 + j) * kTileKeys;
            // Lane i brings the scale of block i % 8 of the tile's keys (i < 8) or values
            // (i < 16).
            int64_t scale_page = -1;
            const int scale_key = key0 + (lane & 7) * kScaleTokens;
            if (lane < 16 && scale_key < g.kv_len && scale_key >> p.page_shift < p.columns)
              scale_page = __ldg(ids + (scale_key >> p.page_shift));
#pragma unroll 1
            for (int c = 0; c < 2 * kChunks && ok; ++c, ++m) {
              const bool v = c >= kChunks;
              const int slot = m % S::kRawSlots, turn = m / S::kRawSlots;
              const int chunk0 = key0 + c % kChunks * S::kRawKeys;
              const int left = min(g.kv_len - chunk0, S::kRawKeys);
              const int boxes = left > 0 ? (left + p.box_rows - 1) / p.box_rows : 0;
              // Lane i fetches box i (at most 8 of the chunk's pages).
              int page = -1, row = 0;
              if (lane < boxes) {
                const int key = chunk0 + lane * p.box_rows, column = key >> p.page_shift;
                if (column < p.columns) page = __ldg(ids + column);
                row = g.kv_head * p.page_size + (key & (p.page_size - 1));
              }
              if (turn > 0 && !(ok = wait_warp(&raw_empty[slot], (uint32_t)((turn - 1) & 1), ctl, err, 93))) break;
              if (lane == 0) mbar_expect_tx(&raw_full[slot], (uint32_t)(boxes * box_bytes));
              __syncwarp();
              if (lane < boxes)
                tma_codes(base + S::kOffRaw + slot * S::kRaw + lane * box_bytes, v ? &p.tm_v : &p.tm_k, row, page,
                          &raw_full[slot]);
              if (c == 0 && lane < 16) {
                const bool real = scale_page >= 0 && scale_page < p.pages;
                const float* from = lane < 8 ? p.k_scales : p.v_scales;
                if (real)
                  from += scale_page * p.scale_stride + g.kv_head * (p.page_size / kScaleTokens) +
                          (scale_key & (p.page_size - 1)) / kScaleTokens;
                copy_value(scales + (t & 3) * 16 + lane, from, real);
              }
              arrive_with_copies(&raw_full[slot]);
            }
          }
        }
        // Copies in flight land before the block exits.
        for (int i = m > S::kRawSlots ? m - S::kRawSlots : 0; i < m; ++i)
          drain(&raw_full[i % S::kRawSlots], (uint32_t)((i / S::kRawSlots) & 1), err);
      }
    } else if (kWiden && warp >= S::kWidenWarp) {
      if constexpr (kWiden) {
        constexpr int kChunks = kTileKeys / S::kRawKeys;
        // A warp takes 8 rows by 64 columns at a time, 16 codes a thread: eight threads in a
        // row read two rows and write them to rows whose swizzles keep both apart in the
        // banks (of 128-byte rows r and r ^ 5, of 64-byte rows neighbours).
        constexpr int kGroupStep = 8 * (S::kWideners / 32);  // rows from one group of a warp to its next
        const int quarter = lane >> 3, other = (lane >> 2) & 1, vec = lane & 3;
        const int row8 = D == 128 ? (other ? quarter ^ 5 : quarter) : 2 * quarter + other;
        const int my_row = 8 * (warp - S::kWidenWarp) + row8;
        const int chunk = D == 128 ? vec ^ row8 : vec ^ ((row8 >> 1) & 3);  // the second half's lies 64 bytes on or back
        const int from_at = my_row * D + chunk * 16, flip = chunk & 4 ? -64 : 64;
        const int to_at = my_row * 128 + (((2 * vec) ^ row8) << 4), second = (row8 & 1) ? -16 : 16;
        int n = 0, m = 0, t = 0;  // slots of the ring, chunks, tiles
        bool ok = true;
        for (int seg = seg0; seg < seg1 && ok; ++seg) {
          const PagedSegment g = p.segments[seg];
          const View<H> view(g, p.group);
          ScalesSeen seen;
          for (int j = 0; j < view.tiles && ok; ++j, ++t) {
            const int have = g.kv_len - (g.tile0 + j) * kTileKeys;
#pragma unroll 1
            for (int v = 0; v < 2 && ok; ++v, ++n) {
              const int slot = n % S::kSlots, turn = n / S::kSlots;
              if (turn > 0 && !(ok = wait_warp(&kv_empty[slot], (uint32_t)((turn - 1) & 1), ctl, err, 94))) break;
              uint8_t* dst = base + S::kOffRing + slot * S::kTile;
#pragma unroll 1
              for (int c = 0; c < kChunks; ++c, ++m) {
                const int raw = m % S::kRawSlots;
                if (!(ok = wait_warp(&raw_full[raw], (uint32_t)((m / S::kRawSlots) & 1), ctl, err, 95))) break;
                if (c == 0 && v == 0 && warp == S::kWidenWarp) {
                  const float* from = scales + (t & 3) * 16;
                  tell(told[t % S::kTold], from[lane & 7], from[8 + (lane & 7)], p.scale_log2, seen,
                       (have + kScaleTokens - 1) / kScaleTokens, lane);
                }
                const uint8_t* src = base + S::kOffRaw + raw * S::kRaw + from_at;
                uint8_t* to = dst + c * S::kRawKeys * 128 + to_at;
                // The thread's vectors: column halves h, groups of 8 rows.
#pragma unroll
                for (int h = 0; h < D / 64; ++h) {
                  constexpr int kGroups = S::kRawKeys / 8 / (S::kWideners / 32);
                  uint4 w[kGroups];
#pragma unroll
                  for (int b = 0; b < kGroups; ++b)
                    w[b] = *reinterpret_cast<const uint4*>(src + b * kGroupStep * D + (h ? flip : 0));
                  if (have < kTileKeys) {
                    // Past the request's length anything may lie, NaN included: zeros.
#pragma unroll
                    for (int b = 0; b < kGroups; ++b)
                      if (c * S::kRawKeys + my_row + b * kGroupStep >= have) w[b] = make_uint4(0, 0, 0, 0);
                  }
#pragma unroll
                  for (int b = 0; b < kGroups; ++b) {
                    uint4 out[2];
                    Code<St>::widen(w[b].x, out[0].x, out[0].y);
                    Code<St>::widen(w[b].y, out[0].z, out[0].w);
                    Code<St>::widen(w[b].z, out[1].x, out[1].y);
                    Code<St>::widen(w[b].w, out[1].z, out[1].w);
                    uint8_t* at = to + h * kColBytes + b * kGroupStep * 128;
                    *reinterpret_cast<uint4*>(at) = out[0];
                    *reinterpret_cast<uint4*>(at + second) = out[1];
                  }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_empty[raw]);
              }
              if (!ok) break;
              fence_proxy_async();
              mbar_arrive(&kv_full[slot]);
            }
          }
        }
      }
    } else if (!kWiden && warp == S::kLoadWarp) {
      int n = 0;  // tiles fetched (K and V each count)
      bool ok = true;
      for (int seg = seg0; seg < seg1 && ok; ++seg) {
        const PagedSegment g = p.segments[seg];
        const View<H> view(g, p.group);
        const int32_t* ids = p.ids + g.request * p.ids_stride;
        const int box_bytes = p.box_rows * 128;
        // Of widened codes: the request's first page; lane i reads the scales of block
        // i % 8, a tile ahead.
        int first_page = 0;
        const float *k_from = nullptr, *v_from = nullptr;
        float k_scale = 0.f, v_scale = 0.f;
        ScalesSeen seen;
        if constexpr (kScaled) {
          first_page = __ldg(p.first_page + g.request);
          const int64_t at = g.kv_head * p.scale_stride + (int64_t)first_page * (p.page_size / kScaleTokens) +
                             g.tile0 * (kTileKeys / kScaleTokens) + (lane & 7);
          k_from = p.k_scales + at;
          v_from = p.v_scales + at;
        }
        auto look_at = [&](int j) {
          const bool real = (g.tile0 + j) * kTileKeys + (lane & 7) * kScaleTokens < g.kv_len;
          k_scale = real ? __ldg(k_from + 8 * j) : 0.f;
          v_scale = real ? __ldg(v_from + 8 * j) : 0.f;
        };
        if (kScaled && view.tiles > 0) {
          look_at(0);
          // Those of the whole segment: the loader is ahead, so the softmax need not look for
          // r to grow.
          float most = 0.f, least = INFINITY;
          const int blocks = min((g.kv_len + kScaleTokens - 1) / kScaleTokens - g.tile0 * 8, view.tiles * 8);
          const float* from = v_from - (lane & 7);
#pragma unroll 8
          for (int i = lane; i < blocks; i += 32) {
            const float v = __ldg(from + i);
            most = fmaxf(most, fabsf(v) < INFINITY ? v : 0.f);
            least = fminf(least, fabsf(v) < INFINITY ? v : INFINITY);
          }
          seen.add(warp_max(most), -warp_max(-least));
        }
        for (int j = 0; j < view.tiles && ok; ++j) {
          const int key0 = (g.tile0 + j) * kTileKeys;
          const int left = g.kv_len - key0;
          const int boxes = ((left < kTileKeys ? left : kTileKeys) + p.box_rows - 1) / p.box_rows;
          // Lane i fetches box i (at most 16 of the tile's pages).
          int page = -1, row = 0;
          if (lane < boxes) {
            const int key = key0 + lane * p.box_rows, column = key >> p.page_shift;
            if constexpr (kScaled)
              page = first_page + column;
            else if (column < p.columns)
              page = __ldg(ids + column);
            row = g.kv_head * p.page_size + (key & (p.page_size - 1));
          }
#pragma unroll
          for (int v = 0; v < 2; ++v, ++n) {
            const int slot = n % S::kSlots, turn = n / S::kSlots;
            if (turn > 0 && !(ok = wait_warp(&kv_empty[slot], (uint32_t)((turn - 1) & 1), ctl, err, 81))) break;
            if constexpr (kScaled) {
              if (v == 0) {  // seen with the keys
                tell(told[n / 2 % S::kTold], k_scale, v_scale, p.scale_log2, seen,
                     (left + kScaleTokens - 1) / kScaleTokens, lane);
                __syncwarp();
              } else if (j + 1 < view.tiles) {
                look_at(j + 1);
              }
            }
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
        if (kScaled && lane == 0) mbar_arrive(&s_full[x]);  // what is told of the tile has been seen
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
          if (!kWiden && have < kTileKeys) {  // (the wideners write zeros there)
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
          if (!kScaled && chunks > 0) {  // (codes are finite)
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
    if constexpr (kWiden)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else if constexpr (H == 2 && kScaled)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    else if constexpr (H == 2)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax of half x: thread r owns row r = TMEM lane r.
    const int x = warp >> 2;
    const int r = tid - kHalf * x;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_o = lane_base + kColO + 128 * x, t_s = lane_base + S::kColS + 128 * x;
    uint32_t s_turn = 0, o_turn = 0;
    int tiles_before = 0;
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
          uint32_t most[kBatch];
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
            bool outside = false;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              const uint4 v = values[b];
              most[b] = magnitude(v.w, magnitude(v.z, magnitude(v.y, magnitude(v.x, 0))));
#pragma unroll
              for (int off = 1; off < kChunks; off <<= 1)
                most[b] = max(most[b], __shfl_xor_sync(0xffffffffu, most[b], off));
              outside |= outside_f16(most[b]);
            }
            outside = __any_sync(0xffffffffu, outside);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              float f[8];
              unpack8<T>(values[b], f);
              if (outside) {
                const int over = beyond_f16(most[b], p.least_power);
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
      if (!kScaled && kHalf * x >= g.rows) continue;
      const View<H> view(g, p.group);
      const int tile_at = tiles_before;
      tiles_before += view.tiles;
      if (kScaled && kHalf * x >= g.rows) continue;
      const int count = view.count[x];
      // Threads past the rows follow the last one; what they make is dropped.
      const int pr = g.row0 + min(kHalf * x + r, g.rows - 1);
      const int token = pr / p.group;
      const int limit = g.kv_len - g.new_len + token;  // last key the row sees
      const int first_limit = g.kv_len - g.new_len + (g.row0 + kHalf * x) / p.group;
      const float scale = Act<T>::kDtype == Act<C>::kDtype ? p.scale_log2 : p.scale_log2 * boost;
      float m = -INFINITY, l = 0.f;
      float v_ref = 1.f;  // r of O
      float kappa = 0.f;  // O stands at 2^(m + kappa)
      const bool own_boost = kScaled && Act<T>::kDtype != Act<C>::kDtype && boost != 1.f;
      const bool boosted = kScaled && Act<T>::kDtype != Act<C>::kDtype && __any_sync(0xffffffffu, own_boost);
      // Of codes two loops: the second from the first tile on with which scales lie far
      // apart (in one loop that rare path cost 2 to 9 per cent of the time; with two halves
      // it is known of the segment's first tile).  The next tile's scores are awaited at a
      // tile's end, for a second wait before the loops made it spill.
      int j = 0;
      bool wide = false;
      if (kScaled && count > 0 && (ok = wait_warp(&s_full[x], s_turn & 1, ctl, err, 90)) && H == 2)
        wide = told[tile_at % S::kTold].events & kWide;
#pragma unroll
      for (int apart = 0; apart < (kScaled ? 2 : 1); ++apart)
      if (apart == 0 ? H == 1 || !wide : __builtin_expect(wide, 0))
      for (; j < count && ok; ++j) {
        if (!kScaled && !(ok = wait_warp(&s_full[x], s_turn & 1, ctl, err, 90))) break;
        tc_fence_after();
        const TileScales& of = told[(tile_at + j) % S::kTold];
        uint32_t events = 0;
        if constexpr (kScaled) {
          events = of.events;
          if (H == 1 && apart == 0 && __builtin_expect(events & kWide, 0)) {
            wide = true;
            break;
          }
          v_ref = of.v_ref;
        }
        ++s_turn;
        const int key0 = (g.tile0 + j) * kTileKeys;
        float factor = 1.f;
        if (apart) {
          // The scores are read three times, 32 at a time (what is rare takes little code): for
          // their maximum, for the sum and the largest share, for P.
          const float down = fminf(boost, 1.f), up = fmaxf(boost, 1.f), before = m;
          float own = -INFINITY, most = -INFINITY, from = 0.f, sub = 0.f;
#pragma unroll 1
          for (int pass = 0; pass < 3; ++pass) {
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
              float s[32];
              __syncwarp();
              tmem_ld32(t_s + c, s);
              const float4 first = of.block[c / 16], second = of.block[c / 16 + 1];
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                s[i] = s[i] * down * (i < 16 ? first.x : second.x) * up;
                s[i] = key0 + c + i > limit ? -INFINITY : s[i] - from;
              }
              if (pass == 0) {
#pragma unroll
                for (int i = 0; i < 32; ++i) own = max_nan(own, s[i]);
              } else if (pass == 1) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  l += fast_exp2(s[i]);
                  most = max_nan(most, s[i] + (i < 16 ? first.z : second.z));
                }
              } else {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  const float offset = i < 16 ? first.z : second.z;
                  pk[i / 2] = pack2<C>(fast_exp2(s[i] + offset - sub), fast_exp2(s[i + 1] + offset - sub));
                }
                __syncwarp();
                tmem_st16(t_s + c / 2, pk);  // over scores that have been read
                if (c & 32) {
                  tmem_st_wait();
                  tc_fence_before();
                  mbar_arrive(&p_full[2 * x + c / 64]);
                }
              }
            }
            if (pass == 0) {
              m = max_nan(m, own);
              from = m == -INFINITY ? 0.f : m;
              l *= before == -INFINITY ? 0.f : fast_exp2(before - from);
            } else if (pass == 1) {
              const float stands = kappa + of.fall + (before - from);
              kappa = max_nan(stands, most - kLift);
              sub = kappa == -INFINITY ? 0.f : kappa;
              if (stands != -INFINITY) factor = fast_exp2(stands - sub);  // else nothing stands in O yet
              if (__any_sync(0xffffffffu, factor != 1.f) && j > 0) rescale<D>(t_o, factor);
            }
          }
          if (kScaled && (events & 0xffu) && sees_odd(events, limit - key0)) l = __uint_as_float(0x7fc00000u);
          if (j + 1 < count) ok = wait_warp(&s_full[x], s_turn & 1, ctl, err, 90);
          continue;
        }
        float sc[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32_begin(t_s + c, sc + c);
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_wait32(sc + c);
        if constexpr (kScaled && Act<T>::kDtype != Act<C>::kDtype) {
          if (boosted) {
            // Powers below one before the units, those above after them: what lies
            // between stays in fp32's range.
            const float before = fminf(boost, 1.f), after = fmaxf(boost, 1.f);
#pragma unroll
            for (int c = 0; c < 128; ++c) sc[c] = own_boost ? sc[c] * before * of.block[c / 16].x * after : sc[c];
          }
        }
        // Of codes: what the scores are still to be multiplied with.
        const auto unit_of = [&](int block) { return own_boost ? 1.f : of.block[block].x; };
        if (key0 + kTileKeys - 1 > first_limit) {
          const int lim = limit - key0;  // later columns are masked
#pragma unroll
          for (int c = 0; c < 128; ++c) sc[c] = c > lim ? -INFINITY : sc[c];
        }
        // The maximum of the raw scores (the scale is positive), NaN kept.
        float mp[8];
        bool raw = true;  // the scores are not yet the exponents
        float mx;
        if constexpr (kScaled) {
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            float most = max_nan(sc[16 * b], sc[16 * b + 1]);
#pragma unroll
            for (int i = 2; i < 16; i += 2) most = max_nan(most, sc[16 * b + i], sc[16 * b + i + 1]);
            mp[b] = fmaf(most, unit_of(b), of.block[b].z);
          }
          mx = max_nan(max_nan(mp[0], mp[1], mp[2]), max_nan(mp[3], mp[4], mp[5]), max_nan(mp[6], mp[7]));
          // Far out the sum's rounding would lie between m and the products that it is
          // taken from: the scores' own maximum there.
          if (__any_sync(0xffffffffu, fabsf(mx) > kFar)) {
            if (events & kSpread) {  // nothing has changed yet: this tile again
              wide = true;
              --s_turn;
              break;
            }
            float own = -INFINITY;
#pragma unroll
            for (int c = 0; c < 128; ++c) own = max_nan(own, __fmul_rn(sc[c], unit_of(c / 16)));
            if (fabsf(mx) > kFar) mx = own;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) mp[i] = max_nan(sc[2 * i], sc[2 * i + 1]);
#pragma unroll
          for (int c = 16; c < 128; c += 16)
#pragma unroll
            for (int i = 0; i < 8; ++i) mp[i] = max_nan(mp[i], sc[c + 2 * i], sc[c + 2 * i + 1]);
          mx = max_nan(max_nan(mp[0], mp[1], mp[2]), max_nan(mp[3], mp[4], mp[5]), max_nan(mp[6], mp[7])) * scale;
        }
        if (mx == INFINITY) mx = __uint_as_float(0x7fc00000u);  // inf - inf: the row is NaN
        // Far out the product with the scale is rounded by more than the
        // exponential bears: there each score takes the maximum's rounding.
        float unit = scale;
        if (!kScaled && __any_sync(0xffffffffu, fabsf(mx) > kFar)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) sc[c] *= scale;
          unit = 1.f;
        }
        mx = lifted<C>(mx);
        if (kWiden && (events & kGrew) && m != -INFINITY) {
          // What m stands for fell with r; O stays, l is in the old units.
          const float before = m;
          m += of.fall;
          if (!(mx <= m + kRescale)) m = max_nan(m, mx);
          factor = fast_exp2((before - m) + of.fall);
          l *= fast_exp2(before - m);  // 2^61 at most: else the scales are far apart
        } else if (!(mx <= m + kRescale)) {  // also for NaN, and for the first key seen
          mx = max_nan(m, mx);  // a NaN stays
          factor = fast_exp2(m - mx);
          m = mx;
          l *= factor;
        }
        // This tile's scores were issued after the last tile's product: O is
        // stable, and P may overlay S.  (The vote is taken on the first tile too:
        // it brings the warp together for the stores of P.)
        if (__any_sync(0xffffffffu, factor != 1.f) && j > 0) rescale<D>(t_o, factor);
        // Exponent arguments and sums on packed pairs.  P goes out in two
        // parts of 64 keys, so the product of the first runs while the
        // second's exponentials do.
        const float sub = m == -INFINITY ? 0.f : -m;
        const uint64_t sl2 = f2_pack(unit, unit), nm = f2_pack(sub, sub);
        if constexpr (kScaled) {
          // Away from zero -m + log2(s_v / r) would lose the logarithm's bits (and far out
          // the product needs the maximum's rounding, as above): step by step there.
          if (__any_sync(0xffffffffu, fabsf(sub) > kApart)) {
            raw = false;
#pragma unroll
            for (int c = 0; c < 128; ++c)
              sc[c] = __fadd_rn(__fadd_rn(__fmul_rn(sc[c], unit_of(c / 16)), sub), of.block[c / 16].z);
          }
        }
        uint64_t sp[4], block_unit = 0ull, block_offset = 0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) sp[i] = 0ull;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int k0 = 64 * half + 2 * c;
            float a, b;
            if constexpr (kScaled) {
              const int block = k0 / 16;
              if (c % 8 == 0) {
                const ulonglong2 both = *reinterpret_cast<const ulonglong2*>(&of.block[block]);
                block_unit = raw && !own_boost ? both.x : f2_pack(1.f, 1.f);
                block_offset = raw ? f2_add(nm, both.y) : 0ull;
                sp[0] = sp[1] = 0ull;
              }
              f2_unpack(f2_fma(f2_pack(sc[k0], sc[k0 + 1]), block_unit, block_offset), a, b);
              a = fast_exp2(a);
              b = fast_exp2(b);
              sp[c & 1] = f2_add(sp[c & 1], f2_pack(a, b));
              pk[c] = pack2<C>(a, b);
              if (c % 8 == 7) {
                sp[2 + (block & 1)] = f2_fma(f2_add(sp[0], sp[1]),
                                             *reinterpret_cast<const uint64_t*>(&of.back[block]), sp[2 + (block & 1)]);
              }
              continue;
            }
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
        f2_unpack(kScaled ? f2_add(sp[2], sp[3]) : f2_add(f2_add(sp[0], sp[1]), f2_add(sp[2], sp[3])), s0, s1);
        l += s0 + s1;
        if (kScaled && (events & 0xffu) && sees_odd(events, limit - key0)) l = __uint_as_float(0x7fc00000u);
        if (kScaled && j + 1 < count) ok = wait_warp(&s_full[x], s_turn & 1, ctl, err, 90);
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
      const bool cleared = !kScaled && ctl->cleared != 0;
      // A row that has seen no key above -inf gives zeros.
      const float inv = m == -INFINITY ? 0.f : 1.f / l;
      // 2^kappa r may lie anywhere, but not what it makes of O / l.
      const float half = kScaled ? exp2_far(0.5f * kappa) : 1.f;
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
        if constexpr (kScaled) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = m == -INFINITY ? 0.f : o[i] * inv * half * (v_ref * half);
        }
        if (mine && g.part < 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            float f[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) f[k] = kScaled ? o[i + k] : m == -INFINITY ? 0.f : o[i + k] * inv;
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
// and 4 columns, so the pieces' outputs arrive 512 bytes at a time.  kDivided: a
// piece's outputs are divided by its sum (an 8-bit cache, whose values may lie
// anywhere in fp32's range: weights count down to 2^-149, and a power of two keeps
// their total below one).
constexpr int kMergeWarps = 8;

template <typename T, int D, int R, bool kDivided>
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
  float M = -INFINITY, most = 0.f;
#pragma unroll 4
  for (int i = 0; i < g.parts; ++i) {
    M = max_nan(M, st[(int64_t)i * 2 * R]);
    if (kDivided) most = fmaxf(most, st[(int64_t)i * 2 * R + R]);
  }
  // 2^-10 / (the sums' largest power of two): for up to 2^8 pieces.
  const float unit = __uint_as_float((245u << 23) - (__float_as_uint(most) & 0x7f800000u));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < g.parts; ++i) {
    const float m = st[(int64_t)i * 2 * R], own = st[(int64_t)i * 2 * R + R];
    float f;
    if (kDivided) {
      f = exp2_far(m - M);
      f = m == -INFINITY ? 0.f : f * (own * unit);  // an empty piece holds zeros
      sum += f;
    } else {
      f = m == -INFINITY ? 0.f : fast_exp2(m - M);
      sum = fmaf(f, own, sum);
    }
    const float4 v = *reinterpret_cast<const float4*>(o + (int64_t)i * R * D);
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

template <typename T, typename C, int D, int H, typename St>
tf_status launch(TileParams p, const Work& w, const char* table, bool early, cudaStream_t s) {
  using S = Shape<D, H, C, St>;
  if (w.blocks == 0) return TF_OK;
  static PerDeviceOnce attr;
  int dev = 0;
  if (attr.needed(&dev)) {
    TF_CUDA(cudaFuncSetAttribute(paged_tile_kernel<T, C, D, H, St>, cudaFuncAttributeMaxDynamicSharedMemorySize,
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
  TF_CUDA(cudaLaunchKernelEx(&cfg, paged_tile_kernel<T, C, D, H, St>, p));
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
  TF_CUDA(cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, D, S::kRows, S::kScaled>,
                             reinterpret_cast<const PagedSegment*>(table + w.merges), (const float*)p.stat,
                             (const float*)p.part, p.group, p.heads, static_cast<T*>(p.out)));
  return check_launch("paged_merge");
}

template <typename T, typename C, int D, typename St>
tf_status launch_both(const TileParams& p, const PagedArgs& a, cudaStream_t s, const TileParams& widened = TileParams()) {
  const tf_paged_plan& plan = *a.plan;
  float* stat = reinterpret_cast<float*>(a.workspace + split_workspace_bytes(plan));
  const Work tile = {plan.tile_segments_offset, plan.tile_starts_offset, plan.tile_merges_offset,
                     plan.tile_blocks, plan.tile_parts, plan.tile_merges, stat};
  const Work half = {plan.half_segments_offset, plan.half_starts_offset, plan.half_merges_offset,
                     plan.half_blocks, plan.half_parts, plan.half_merges,
                     stat + (int64_t)plan.tile_parts * kTileRows * (2 + D)};
  // The first kernel after the few-rows kernel starts on the SMs that it leaves.
  const bool after_split = plan.split_blocks > 0;
  if constexpr (Shape<D, 1, C, St>::kWiden) {
    TF_TRY((launch<T, C, D, 2, Widened>(widened, tile, a.plan_table, after_split, s)));
  } else {
    TF_TRY((launch<T, C, D, 2, St>(p, tile, a.plan_table, after_split, s)));
  }
  return launch<T, C, D, 1, St>(p, half, a.plan_table, after_split && plan.tile_blocks == 0, s);
}

// What all launches fill in alike.
tf_status tile_params(const PagedArgs& a, TileParams* out) {
  const tf_paged_plan& plan = *a.plan;
  TileParams& p = *out;
  memset(&p, 0, sizeof(p));
  p.box_rows = a.kv.page_size < kTileKeys ? a.kv.page_size : kTileKeys;
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
  p.least_power = power_floor(p.scale_log2);
  TF_TRY(tc_flags(&p.err, const_cast<long long**>(&p.wait_cycles)));
  return TF_OK;
}

}  // namespace

tf_status launch_paged_tile(const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  if (plan.tile_blocks == 0 && plan.half_blocks == 0) return TF_OK;
  TileParams p;
  TF_TRY(tile_params(a, &p));
  TF_TRY(make_page_map(&p.tm_k, a.kv.k, a.kv, p.box_rows, 64));
  TF_TRY(make_page_map(&p.tm_v, a.kv.v, a.kv, p.box_rows, 64));
#define TF_TILE(T, C) \
  return plan.head_dim == 128 ? launch_both<T, C, 128, C>(p, a, s) : launch_both<T, C, 64, C>(p, a, s)
  if (a.act == TF_DTYPE_F16) TF_TILE(__half, __half);
  if (a.kv.dtype == TF_DTYPE_F16) TF_TILE(__nv_bfloat16, __half);
  TF_TILE(__nv_bfloat16, __nv_bfloat16);
#undef TF_TILE
}

tf_status launch_paged_tile_8bit(const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  if (plan.tile_blocks == 0 && plan.half_blocks == 0) return TF_OK;
  TileParams p, w;
  TF_TRY(tile_params(a, &p));
  w = p;
  if (plan.half_blocks) {
    p.box_rows = a.kv.page_size < 64 ? a.kv.page_size : 64;
    TF_TRY(make_code_map(&p.tm_k, a.kv.k, a.kv, p.box_rows));
    TF_TRY(make_code_map(&p.tm_v, a.kv.v, a.kv, p.box_rows));
    p.k_scales = a.scales.k;
    p.v_scales = a.scales.v;
    p.scale_stride = a.scales.page_stride;
  }
  if (plan.tile_blocks) {
    const WidenedPages pages(a);
    TF_TRY(make_page_map(&w.tm_k, pages.kv.k, pages.kv, w.box_rows, 64));
    TF_TRY(make_page_map(&w.tm_v, pages.kv.v, pages.kv, w.box_rows, 64));
    w.k_scales = pages.k_scales;
    w.v_scales = pages.v_scales;
    w.scale_stride = pages.blocks;
    w.first_page = pages.first_page;
  }
  const bool ints = a.kv.dtype == TF_DTYPE_I8;
#define TF_TILE(T, S) \
  return plan.head_dim == 128 ? launch_both<T, __half, 128, S>(p, a, s, w) : launch_both<T, __half, 64, S>(p, a, s, w)
  if (a.act == TF_DTYPE_F16) {
    if (ints) TF_TILE(__half, I8);
    TF_TILE(__half, E4M3);
  }
  if (ints) TF_TILE(__nv_bfloat16, I8);
  TF_TILE(__nv_bfloat16, E4M3);
#undef TF_TILE
}

}  // namespace tf
