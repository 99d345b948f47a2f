// Log probabilities of given tokens, with entropy, rank and the top
// alternatives, in one pass over the logits.
//
//   m = max x,  s = sum e^(x - m),  w = sum (x - m) e^(x - m)
//   log p(t) = (x_t - m) - ln s,   entropy = ln s - w / s
//   rank(t)  = number of entries before t in the order (value down, index up)
//   alternatives: the first k entries of that order (NaN last)
//
// What bounds it: each logit is read once; 50304 fp32 logits are 0.2 MB, 31 ns
// of the whole GPU's bandwidth, and with 16-bit logits the exponentials come
// close behind (16 a clock on an SM: 0.7 of the time that the bytes take).  So
// the pass spends about five issue slots a value: a tile of 8 vectors of 16
// bytes a thread stays in registers for all of its uses while the next one
// loads; the sums run on packed fp32 pairs against the thread's running
// maximum (rescaled when that moves), and the maximum and the rank's
// comparisons of 16-bit logits on packed pairs of their own type.
//
// The alternatives ride along as candidates: a composite key (ordered value
// bits, then the inverted index) makes every entry distinct and ties fall to
// the lowest index.  The first tile yields a lower bound of the k-th key (the
// k-th largest of the warps' few largest thread maxima: k entries are at or
// above it).  A thread whose maximum of a tile meets the bound queues the tile
// and goes on; after 1, 2, 4, ... tiles (for few alternatives from 4 on) the
// block looks through the queue (the vectors come again, from L2), puts entries
// at or above the bound into a buffer, and prunes that to its k best, which
// raises the bound to an exact one.  (Looking through the vectors on the spot
// cost some 4000 clocks each time: a hundred instructions that are rare enough
// to be fetched from memory.)  After the first tile few threads meet the bound,
// so the pass stays a stream.  Should queue or buffer run over (values in
// rising order, say, or equal ones), the vectors since the last prune come
// again: for a better bound, the k-th largest of the threads' best vectors,
// then for what lies at or above it; and if the buffer runs over even so, in
// rounds of one entry a thread with a prune in between.
//
// A row may be shared by a cluster of 1, 2, 4 or 8 blocks (few rows: the whole
// GPU reads; one row of 50304 on one block would take its load latency 25
// times over); the blocks' sums and candidates meet in the first block's hands
// over distributed shared memory, so no scratch in device memory is needed.
//
// Measured: 4095 rows of 50304 bf16 logits with five alternatives 132 us (3.1
// TB/s; 116 where the given token is the largest, so that nothing is counted)
// and 97 with none (4.3 TB/s); with 64 251; 2048 rows of fp32 with twenty 103 us
// (93 with the largest token), in rising order 496 (in rounds alone 9450); one
// row 11 us, 64 rows 13.  At 18 warps an SM it is latency that is left: a
// scheduler issues in half of its clocks, and warps wait for their own dependent
// instructions, for instructions to be fetched and at the prunes' barriers.
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"
#include "internal.h"
#include "tc_ptx.cuh"

namespace tf {

namespace {

namespace cg = cooperative_groups;

constexpr int kVectors = 8;     // 16-byte vectors of a thread's tile
constexpr int kStages = 2;      // tiles in shared memory
constexpr int kMaxTop = 64;
constexpr int kQueue = 512;     // a thread's tiles that meet the bound between two looks
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct LogprobParams {
  const void* logits;
  int64_t row_stride;
  const int64_t* tokens;
  int64_t rows;
  int vocab;
  int top;
  float* logprob;
  float* entropy;
  int32_t* rank;
  float* top_logprob;
  int64_t* top_token;
  int* err;
  const long long* wait_cycles;
};

// Order-preserving bits of a value: NaN lowest, then -inf; -0 counts as +0.
__device__ __forceinline__ uint32_t order_bits(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  if (v != v) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  if (k == 0u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ uint64_t composite(float v, uint32_t index) {
  return ((uint64_t)order_bits(v) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// A 16-byte vector of logits: its values as floats, their maximum (NaN kept),
// and how many lie above (or at) the given token's.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kPer = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  __device__ __forceinline__ static float get(const uint4& v, int i) { return __uint_as_float(word(v, i)); }
  __device__ __forceinline__ static float max_of(const uint4& v) {
    return max_nan(max_nan(get(v, 0), get(v, 1)), max_nan(get(v, 2), get(v, 3)));
  }
  // Running maximum over vectors (NaN kept).
  using Max = float;
  __device__ __forceinline__ static Max lowest() { return -INFINITY; }
  __device__ __forceinline__ static void raise(Max& m, const uint4& v) { m = max_nan(m, max_of(v)); }
  __device__ __forceinline__ static float value(Max m) { return m; }
  // Bit i set: value i is not below t.
  __device__ __forceinline__ static uint32_t not_below(const uint4& v, float t) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (get(v, i) < t ? 0u : 1u) << i;
    return m;
  }
  __device__ __forceinline__ static float pick(const uint4& v, int i) {
    return __uint_as_float(i < 2 ? (i == 0 ? v.x : v.y) : (i == 2 ? v.z : v.w));
  }
  // Counts of values above (kAt: at or above) t, added up per thread.
  using Count = int;
  __device__ __forceinline__ static Count zero() { return 0; }
  template <bool kAt>
  __device__ __forceinline__ static void above(const uint4& v, float t, Count& n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) n += kAt ? get(v, i) >= t : get(v, i) > t;
  }
  __device__ __forceinline__ static int total(Count n) { return n; }
};
template <typename T, typename T2>
struct Vec16 {
  static constexpr int kPer = 8;
  __device__ __forceinline__ static float max_of(const uint4& v) {
    Max m = lowest();
    raise(m, v);
    return value(m);
  }
  using Max = T2;
  __device__ __forceinline__ static Max lowest() { return T2{from_f<T>(-INFINITY), from_f<T>(-INFINITY)}; }
  __device__ __forceinline__ static void raise(Max& m, const uint4& v) {
    const T2* h = reinterpret_cast<const T2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __hmax2_nan(m, h[i]);
  }
  __device__ __forceinline__ static float value(Max m) { return max_nan(__low2float(m), __high2float(m)); }
  // Bit i set: value i is not below t (t rounded to T, which for the value of
  // an entry is exact; else a few more pass, for the exact test to drop).
  __device__ __forceinline__ static uint32_t not_below(const uint4& v, float t) {
    const T2* h = reinterpret_cast<const T2*>(&v);
    const T tt = from_f<T>(t);
    const T2 t2 = {tt, tt};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t below = __hlt2_mask(h[i], t2);  // NaN: not below
      m |= (~below & 0x00010001u) << (2 * i);
    }
    return (m & 0xffu) | (m >> 15 & 0xaau);  // even values, odd values
  }
  __device__ __forceinline__ static float pick(const uint4& v, int i) {
    const uint32_t w = i < 4 ? (i < 2 ? v.x : v.y) : (i < 6 ? v.z : v.w);
    const uint16_t u = (uint16_t)((i & 1) ? w >> 16 : w);
    return to_f(*reinterpret_cast<const T*>(&u));
  }
  // The comparisons give packed 0 and 1; a tile adds at most 4 * kVectors = 32
  // to each half (bf16 counts exactly to 256).
  using Count = T2;
  __device__ __forceinline__ static Count zero() { return T2{from_f<T>(0.f), from_f<T>(0.f)}; }
  template <bool kAt>
  __device__ __forceinline__ static void above(const uint4& v, float t, Count& n) {
    const T2* h = reinterpret_cast<const T2*>(&v);
    const T tt = from_f<T>(t);  // exact: t is one of the row's values, or +inf
    const T2 t2 = {tt, tt};
#pragma unroll
    for (int i = 0; i < 4; ++i) n = __hadd2(n, kAt ? __hge2(h[i], t2) : __hgt2(h[i], t2));
  }
  __device__ __forceinline__ static int total(Count n) { return (int)(__low2float(n) + __high2float(n)); }
};
template <>
struct Vec<__half> : Vec16<__half, __half2> {
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  __device__ __forceinline__ static float get(const uint4& v, int i) {
    const uint32_t w = word(v, i >> 1);
    return __half2float(__ushort_as_half((unsigned short)((i & 1) ? w >> 16 : w & 0xffffu)));
  }
};
template <>
struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16, __nv_bfloat162> {
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  __device__ __forceinline__ static float get(const uint4& v, int i) {
    const uint32_t w = word(v, i >> 1);
    return __uint_as_float((i & 1) ? w & 0xffff0000u : w << 16);
  }
};

// Running sums relative to a maximum m, in log2 units: s = sum 2^d,
// w = sum d 2^d, d = x log2 e + c by one fused multiply-add, c the rounded
// -m log2 e.  At x = m that leaves a residue of c's rounding in d, the same for
// every x; total() takes it out again (exactly, where one entry holds all of
// the sum).  m = -inf: nothing but -inf so far.
//
// Up to |m| = kFar the residue stays below 2^-3.  m does not go below -kFar: that
// serves a thread that has met nothing but a finite mask's values (-1e30, say),
// unless the whole row stays there.  Rows that end with m at -kFar, or above
// kFar, are summed again, by far_sums().
constexpr float kFar = 1048576.f;

struct Sums {
  float m, s, w;
  __device__ __forceinline__ static float offset(float m) { return -__fmul_rn(m, kLog2e); }
  __device__ __forceinline__ void move(float to) {  // to >= m, or NaN
    if (m == -INFINITY) {
      m = to;
    } else if (to != m) {
      const float d = offset(to) - offset(m), f = exp2_fast(d);
      w = f == 0.f ? 0.f : f * fmaf(d, s, w);
      s *= f;
      m = to;
    }
  }
  // The sums of a warp's lanes: to their maximum, then plain additions.
  __device__ __forceinline__ void join_warp() {
    float to = m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) to = max_nan(to, __shfl_xor_sync(0xffffffffu, to, off));
    move(to);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, off);
      w += __shfl_xor_sync(0xffffffffu, w, off);
    }
  }
  // ln sum e^(x - m), and the entropy ln sum e^(x - m) - sum (x - m) p.
  __device__ __forceinline__ void total(float& log_sum, float& entropy) const {
    const float residue = fabsf(m) >= kFar ? 0.f : fmaf(m, kLog2e, offset(m));
    log_sum = logf(s / exp2_fast(residue));
    entropy = log_sum - (w / s - residue) * kLn2;
  }
  // Adds a tile of vectors whose maximum is tmax.
  template <typename T, int N>
  __device__ __forceinline__ void add(const uint4 (&r)[N], float tmax) {
    if (!(tmax <= m)) {
      const float to = max_nan(m, tmax);
      move(to < -kFar ? -kFar : to);
    }
    if (m == -INFINITY) return;
    const float c = offset(m);
    const uint64_t log2e = pair(kLog2e, kLog2e), c2 = pair(c, c);
    uint64_t s2[2] = {0, 0}, w2[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < Vec<T>::kPer; j += 2) {
        const uint64_t d = fma2(pair(Vec<T>::get(r[i], j), Vec<T>::get(r[i], j + 1)), log2e, c2);
        float d0, d1;
        unpair(d, d0, d1);
        const uint64_t e = pair(exp2_fast(d0), exp2_fast(d1));
        s2[(j >> 1) & 1] = add2(s2[(j >> 1) & 1], e);
        w2[(j >> 1) & 1] = fma2(d, e, w2[(j >> 1) & 1]);
      }
    float a, b, tw;
    unpair(add2(w2[0], w2[1]), a, b);
    tw = a + b;
    if (tw != tw) {
      // A logit of -inf made 0 * -inf (or the row is NaN anyway): again, with
      // d held above -150, where 2^d is zero in fp32.
      tw = 0.f;
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
        uint4 v = r[0];
#pragma unroll
        for (int u = 1; u < N; ++u)
          if (u == i) v = r[u];
#pragma unroll
        for (int j = 0; j < Vec<T>::kPer; ++j) {
          const float d = fmaxf(fmaf(Vec<T>::get(v, j), kLog2e, c), -150.f);
          tw = fmaf(d, exp2_fast(d), tw);
        }
      }
    }
    w += tw;
    unpair(add2(s2[0], s2[1]), a, b);
    s += a + b;
  }
};

// A row's sums relative to its maximum anywhere in the type's range, by the whole
// block: x - m first (exact near m), so no residue; d is held above -150, where
// 2^d is zero in fp32.
template <typename T, int W>
__device__ __noinline__ Sums far_sums(const T* x, int V, Sums* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto value = [&](int e) {
    if constexpr (sizeof(T) == 4)
      return x[e];
    else
      return to_f(x[e]);
  };
  const auto join = [&](Sums a) {  // of the threads' sums
    a.m = warp_max(a.m);
    a.s = warp_sum_butterfly(a.s);
    a.w = warp_sum_butterfly(a.w);
    __syncthreads();
    if (lane == 0) warps[warp] = a;
    __syncthreads();
    a = lane < W ? warps[lane] : Sums{-INFINITY, 0.f, 0.f};
    return Sums{warp_max(a.m), warp_sum_butterfly(a.s), warp_sum_butterfly(a.w)};
  };
  Sums a = {-INFINITY, 0.f, 0.f};
  for (int e = threadIdx.x; e < V; e += 32 * W) a.m = fmaxf(a.m, value(e));
  a = join(a);
  // In fp64: hundreds of equal terms to a thread would drift in fp32.
  double sum = 0., weighted = 0.;
  for (int e = threadIdx.x; e < V; e += 32 * W) {
    const float d = fmaxf((value(e) - a.m) * kLog2e, -150.f), p = exp2_fast(d);
    sum += p;
    weighted += d * p;
  }
  a.s = (float)sum;
  a.w = (float)weighted;
  return join(a);
}

// What a cluster's blocks leave in the first one's shared memory.
struct Gather {
  uint64_t best[kMaxCluster][kMaxTop];
  Sums sums[kMaxCluster];
  int before[kMaxCluster];
  int n[kMaxCluster];
};

template <int W>
struct Shared {
  // Two rounds of the block's threads, the cluster's join, and room for what a
  // first tile offers (64 alternatives, drawn tokens given: 320 places ran over,
  // 308 us against 252),
  // or 64 vectors of 8 values beside the kept ones (values in rising order).
  static constexpr int kBuffer = 640;
  static_assert(kBuffer >= 64 * W && kBuffer - 32 * W >= kMaxTop && kBuffer >= kMaxCluster * kMaxTop, "candidates");
  uint64_t full[kStages], empty[kStages];
  uint64_t buffer[kBuffer];
  int queue[kQueue];  // tiles of threads (their first vector) that met the bound since the last look
  int queued;
  int stalled;                 // a copy that never came
  uint64_t best[kMaxTop];      // sorted k best of the last prune
  int n;                       // candidates in the buffer
  uint64_t rough;              // the k-th largest of the threads' best vectors
  uint32_t warp_key[kMaxTop];  // the warps' largest thread maxima of the first tile
  Sums sums[W];                // the warps' totals
  int before[W];
  Gather gather[W == 8];
};

// Sorts the buffer's n distinct keys by counting and keeps the k best, in
// best[] and at the buffer's front; returns the bound that they make (`bound`
// while there are fewer than k).  Called by the whole block after a barrier;
// ends with one.
template <int W>
__device__ __forceinline__ uint64_t prune(Shared<W>& sh, int k, uint64_t bound) {
  constexpr int kThreads = 32 * W;
  const int n = sh.n;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = sh.buffer[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += sh.buffer[j] > mine;
    if (rank < k) sh.best[rank] = mine;
  }
  __syncthreads();
  const int keep = n < k ? n : k;
  for (int i = threadIdx.x; i < keep; i += kThreads) sh.buffer[i] = sh.best[i];
  if (threadIdx.x == 0) sh.n = keep;
  if (n >= k) bound = sh.best[k - 1] + 1;
  __syncthreads();
  return bound;
}

// Vector of kPer values from index e0, entries outside [0, V) read as -inf.
template <typename T>
__device__ __forceinline__ uint4 load_ragged(const T* x, int e0, int V) {
  constexpr int kPer = Vec<T>::kPer;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = Vec<T>::kNegInf;
    if constexpr (kPer == 4) {
      if (e0 + i >= 0 && e0 + i < V) w[i] = reinterpret_cast<const uint32_t*>(x)[e0 + i];
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int e = e0 + 2 * i + j;
        if (e >= 0 && e < V) {
          const uint32_t u = reinterpret_cast<const uint16_t*>(x)[e];
          w[i] = j ? (w[i] & 0xffffu) | (u << 16) : (w[i] & 0xffff0000u) | u;
        }
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void copy_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          tc::smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(tc::smem_addr(bar))
      : "memory");
}

// A slot's phase that was not met at once.  Past the wait limit (about a second,
// which only a stalled copy could take; a shortened limit polls) an error code
// is recorded, and the wait goes on: a slot must not be read, refilled or left
// behind by the block while its copy is in flight.  The copies always complete;
// were one not to, the second wait ends as well, and the block neither waits nor
// copies any more (false).
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, const long long* wait_cycles, int* err,
                                       volatile int* stalled) {
  const long long limit = *wait_cycles, t0 = clock64();
  const uint32_t suspend = limit < 2000000000LL ? 0u : tc::kSuspendNs;
  if (*stalled) return false;
  while (!tc::mbar_try(bar, parity, suspend))
    if (clock64() - t0 > limit) {
      atomicCAS(err, 0, 72);
      const long long t1 = clock64();
      while (!tc::mbar_try(bar, parity))
        if (*stalled || clock64() - t1 > 2000000000LL) {
          *stalled = 1;
          return false;
        }
      return true;
    }
  return true;
}
// Out of line but for the first try: with the whole wait in the stream of tiles
// 4095 rows of bf16 with 5 alternatives took 138 us instead of 132.
__device__ __forceinline__ bool wait_slot(uint64_t* bar, uint32_t parity, const LogprobParams& p,
                                          volatile int* stalled) {
  return tc::mbar_try(bar, parity, 0) || wait_long(bar, parity, p.wait_cycles, p.err, stalled);
}

template <typename T, int W>
__global__ void __launch_bounds__(32 * W, W == 8 ? 2 : 5) logprobs_kernel(const __grid_constant__ LogprobParams p) {
  constexpr int kWarps = W, kThreads = 32 * W, kTile = kThreads * kVectors;
  using L = Vec<T>;
  using S = Shared<W>;
  constexpr int kPer = L::kPer;
  extern __shared__ __align__(128) uint8_t ring[];  // [kStages][kTile] vectors
  __shared__ S sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = (int)cluster.num_blocks(), slice = (int)cluster.block_rank();
  const int shift = __popc(slices - 1);  // slices is a power of two
  const int64_t row = blockIdx.x >> shift;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int V = p.vocab, k = p.top;
  // Vectors are counted from the 16-byte boundary at or before the row; those
  // in [v_begin, v_end) of this slice lie wholly inside the row.  The row's
  // ragged first and last vectors go to the first slice.
  const int head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int whole0 = head ? 1 : 0, whole1 = (V + head) / kPer;
  const int whole = whole1 > whole0 ? whole1 - whole0 : 0;
  const int v_begin = whole0 + (int)(((int64_t)whole * slice) >> shift);
  const int v_end = whole0 + (int)(((int64_t)whole * (slice + 1)) >> shift);
  const int tiles = (v_end - v_begin + kTile - 1) / kTile;
  const bool edges = slice == 0 && (head || (V + head) % kPer);

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(&sh.full[i], 1);
      tc::mbar_init(&sh.empty[i], kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.n = 0;
    sh.queued = 0;
    sh.stalled = 0;
  }
  // The first block's shared memory may be written once every block of the
  // cluster is known to run: announced here (nothing has been written for
  // another block, so without an order), waited for before the push.
  if (W == 8 && slices > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  __syncthreads();
  auto fetch = [&](int tile) {  // one thread
    const int t0 = v_begin + tile * kTile, n = min(kTile, v_end - t0);
    uint64_t* bar = &sh.full[tile % kStages];
    tc::mbar_expect_tx(bar, (uint32_t)n * 16);
    copy_bulk(ring + (tile % kStages) * (kTile * 16), x + ((int64_t)t0 * kPer - head), (uint32_t)n * 16, bar);
  };
  if (tid == 0)
    for (int i = 0; i < kStages && i < tiles; ++i) fetch(i);

  const int64_t token64 = p.tokens[row];
  const bool given = token64 >= 0 && token64 < V;
  const int token = given ? (int)token64 : -1;
  float xt = INFINITY;  // nothing comes before it
  if (given) {
    if constexpr (kPer == 4)
      xt = reinterpret_cast<const float*>(x)[token];
    else
      xt = to_f(x[token]);
  }

  Sums acc = {-INFINITY, 0.f, 0.f};
  int before = 0;
  uint64_t bound = 0;
  float cut = -INFINITY;  // the bound's value: what is below is no candidate
  int kept = 0;           // candidates that the last prune left
  int group = v_begin;    // first vector after it
  int queued = 0;         // this thread queued vectors since the last look
  auto set_bound = [&](uint64_t to) {
    bound = to;
    const uint32_t bits = (uint32_t)(to >> 32);
    cut = bits ? order_value(bits) : -INFINITY;
  };
  auto rank_each = [&](const uint4& r, int e0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float u = L::get(r, j);
      before += u > xt || (u == xt && e0 + j >= 0 && e0 + j < token);
    }
  };
  // One vector's candidates into the buffer.
  auto offer = [&](const uint4& r, int e0) {
    for (uint32_t some = L::not_below(r, cut); some; some &= some - 1) {
      const int e = e0 + __ffs(some) - 1;
      const uint64_t c = composite(L::pick(r, e - e0), (uint32_t)e);
      if (c < bound || e < 0 || e >= V) continue;
      const int at = atomicAdd(&sh.n, 1);
      if (at < S::kBuffer) sh.buffer[at] = c;
    }
  };
  // Takes the queued vectors' candidates, and prunes them if they became many
  // (or the bound is still the rough first one).  Called by the whole block
  // after the tiles up to vector `to`.
  auto look = [&](int to, bool first) {
    if (!__syncthreads_or(queued)) return;
    queued = 0;
    const int entries = sh.queued;
    bool over = entries > kQueue;
    if (!over) {
      for (int i = tid; i < entries * kVectors; i += kThreads) {
        const int v = sh.queue[i / kVectors] + (i % kVectors) * kThreads, e0 = v * kPer - head;
        if (v < v_end) offer(ld_v4(x + e0), e0);
      }
      __syncthreads();
      over = sh.n > S::kBuffer;
    }
    if (over) {
      // The vectors since the last prune again, against a better bound.  A
      // vector's maximum is an entry at or above (maximum, last index); the
      // k-th largest of the threads' best vectors is below k entries.
      __syncthreads();
      uint64_t own = 0;
#pragma unroll 1
      for (int v = group + tid; v < to; v += kThreads) {
        const int e0 = v * kPer - head;
        own = max(own, composite(L::max_of(ld_v4(x + e0)), (uint32_t)(e0 + kPer - 1)));
      }
      uint64_t* keys = sh.buffer + (S::kBuffer - kThreads);  // past the kept ones
      keys[tid] = own;
      if (tid == 0) sh.n = kept;
      __syncthreads();
      int ahead = 0;
#pragma unroll 8
      for (int i = 0; i < kThreads; ++i) {
        const uint64_t other = keys[i];
        ahead += other > own || (other == own && i < tid);
      }
      if (ahead == k - 1) sh.rough = own;
      __syncthreads();
      set_bound(max(bound, sh.rough));
#pragma unroll 1
      for (int v = group + tid; v < to; v += kThreads) offer(ld_v4(x + (v * kPer - head)), v * kPer - head);
      __syncthreads();
      over = sh.n > S::kBuffer;
    }
    if (over) {
      // Still too many (some threads' own): kThreads entries at a time.
      __syncthreads();
      if (tid == 0) sh.n = kept;
      __syncthreads();
      const int e_last = to * kPer - head;
      for (int e = group * kPer - head; e < e_last; e += kThreads) {
        const int mine = e + tid;
        if (mine < e_last) {
          float u;
          if constexpr (kPer == 4)
            u = reinterpret_cast<const float*>(x)[mine];
          else
            u = to_f(x[mine]);
          const uint64_t c = composite(u, (uint32_t)mine);
          if (c >= bound) sh.buffer[atomicAdd(&sh.n, 1)] = c;
        }
        __syncthreads();
        const bool full = sh.n > S::kBuffer - kThreads;
        __syncthreads();
        if (full) {
          set_bound(prune(sh, k, bound));
        }
      }
    }
    if (tid == 0) sh.queued = 0;
    if (over || first || sh.n > 2 * k + 32) {
      kept = min(sh.n, k);
      set_bound(prune(sh, k, bound));
      group = to;
    } else {
      __syncthreads();
    }
  };

  // With few alternatives the first tile's rough bound serves for a while: 4095
  // rows of bf16, the largest token given, with 5 alternatives 121.5 us looking
  // at once, 117.1 after two tiles, 116.3 after four; with 20 141.6, 134.2 and
  // 136.2; with 64 241, 248 and 484 (the buffer runs over).
  const int first_look = k <= 8 ? 4 : k <= 24 ? 2 : 1;
  for (int tile = 0; tile < tiles; ++tile) {
    const int t0 = v_begin + tile * kTile, slot = tile % kStages;
    const uint4* src = reinterpret_cast<const uint4*>(ring + slot * (kTile * 16)) + tid;
    const bool full = t0 + kTile <= v_end;
    wait_slot(&sh.full[slot], (uint32_t)((tile / kStages) & 1), p, &sh.stalled);
    uint4 r[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      r[i] = full || t0 + tid + i * kThreads < v_end
                 ? src[i * kThreads]
                 : make_uint4(L::kNegInf, L::kNegInf, L::kNegInf, L::kNegInf);
    auto most = L::lowest();
#pragma unroll
    for (int i = 0; i < kVectors; ++i) L::raise(most, r[i]);
    const float tmax = L::value(most);
    // The tile is in registers: its slot may be refilled.
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&sh.empty[slot]);
    if (tid == 0 && tile + kStages < tiles) {
      if (wait_slot(&sh.empty[slot], (uint32_t)((tile / kStages) & 1), p, &sh.stalled)) fetch(tile + kStages);
    }
    if (full) {
      acc.add<T>(r, tmax);
    } else {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        const uint4 one[1] = {r[i]};
        if (t0 + tid + i * kThreads < v_end) acc.add<T>(one, L::max_of(r[i]));
      }
    }
    if (!(tmax < xt)) {
      const int first = t0 * kPer - head;  // entry of the tile's first value
      if (full && first > token) {
        auto n = L::zero();
#pragma unroll
        for (int i = 0; i < kVectors; ++i) L::template above<false>(r[i], xt, n);
        before += L::total(n);
      } else if (full && first + kTile * kPer <= token) {
        auto n = L::zero();
#pragma unroll
        for (int i = 0; i < kVectors; ++i) L::template above<true>(r[i], xt, n);
        before += L::total(n);
      } else {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
          const int v = t0 + tid + i * kThreads, e0 = v * kPer - head;
          if (v >= v_end) continue;
          auto n = L::zero();
          if (e0 > token)
            L::template above<false>(r[i], xt, n);
          else if (e0 + kPer <= token)
            L::template above<true>(r[i], xt, n);
          else
            rank_each(r[i], e0);
          before += L::total(n);
        }
      }
    }
    if (k == 0) continue;
    if (tile == 0) {
      // A first bound: see the top of the file.  A thread without a value
      // stands for the lowest key.
      const int each = min(kMaxTop / kWarps, (k + kWarps - 1) / kWarps + 2);
      uint32_t key = t0 + tid < v_end ? order_bits(tmax) : 0u;
      for (int i = 0; i < each; ++i) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, key);
        const uint32_t who = __ballot_sync(0xffffffffu, key == most);
        if (lane == __ffs(who) - 1) key = 0;
        if (lane == 0) sh.warp_key[i * kWarps + warp] = most;
      }
      __syncthreads();
      // The k-th largest of the up to 64 keys, two a lane, equal ones in list
      // order; every warp finds it for itself.
      const int n = each * kWarps;
      uint32_t kth = 0;
      for (int mine = lane; mine < n; mine += 32) {
        const uint32_t own = sh.warp_key[mine];
        int ahead = 0;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
          const uint32_t other = sh.warp_key[i];
          ahead += other > own || (other == own && i < mine);
        }
        if (ahead == k - 1) kth = own;
      }
      set_bound((uint64_t)__reduce_max_sync(0xffffffffu, kth) << 32);
    }
    if (!(tmax < cut)) {
      queued = 1;
      const int at = atomicAdd(&sh.queued, 1);
      if (at < kQueue) sh.queue[at] = t0 + tid;
    }
    // After 1, 2, 4, 8, ... tiles, from first_look on: each group adds about k
    // candidates.
    if (((tile & (tile + 1)) == 0 && tile + 1 >= first_look) || tile + 1 == tiles)
      look(min(v_end, t0 + kTile), group == v_begin);
  }
  if (edges) {
    // Thread 0 takes the row's first ragged vector, thread 1 its last.
    const int v = tid == 0 ? 0 : whole1;
    const bool mine = tid == 0 ? head != 0 : tid == 1 && (V + head) % kPer && !(head && whole1 == 0);
    if (mine) {
      const int e0 = v * kPer - head;
      const uint4 r[1] = {load_ragged<T>(x, e0, V)};
      acc.add<T>(r, L::max_of(r[0]));
      rank_each(r[0], e0);
      if (k) offer(r[0], e0);  // fits: a look leaves at most 2 k + 32 candidates
    }
  }

  // Block totals, then the cluster's in its first block.
  acc.join_warp();
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) {
    sh.sums[warp] = acc;
    sh.before[warp] = before;
  }
  __syncthreads();
  if (k) prune(sh, k, 0);
  Sums t = {-INFINITY, 0.f, 0.f};
  if (lane < W) t = sh.sums[lane];
  t.join_warp();  // by every warp: each needs it for its outputs
  before = __reduce_add_sync(0xffffffffu, lane < W ? sh.before[lane] : 0);
  if (W == 8 && slices > 1) {
    Gather* to = cluster.map_shared_rank(&sh, 0)->gather;
    const int n = k ? sh.n : 0;
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the first block has started
    if (tid < n) to->best[slice][tid] = sh.best[tid];
    if (tid == 0) {
      to->sums[slice] = t;
      to->before[slice] = before;
      to->n[slice] = n;
    }
    cluster.sync();
    if (slice != 0) return;
    t = {-INFINITY, 0.f, 0.f};
    if (lane < slices) t = sh.gather[0].sums[lane];
    t.join_warp();
    before = __reduce_add_sync(0xffffffffu, lane < slices ? sh.gather[0].before[lane] : 0);
    if (k) {
      for (int i = tid; i < slices * kMaxTop; i += kThreads) {
        const int from = i / kMaxTop, j = i % kMaxTop;
        int at = j;
        for (int u = 0; u < from; ++u) at += sh.gather[0].n[u];
        if (j < sh.gather[0].n[from]) sh.buffer[at] = sh.gather[0].best[from][j];
        if (from == slices - 1 && j == 0) sh.n = at + sh.gather[0].n[from];
      }
      __syncthreads();
      prune(sh, k, 0);
    }
  }
  const bool finite = fabsf(t.m) < INFINITY;  // no NaN, no +inf, not all -inf
  const bool far = finite && fabsf(t.m) >= kFar;  // the same for the whole block
  if (far) t = far_sums<T, W>(x, V, sh.sums);
  if (tid > 0 && tid >= k) return;
  float log_sum, entropy;
  t.total(log_sum, entropy);
  const float nan = __uint_as_float(0x7fc00000u);
  if (tid == 0) {
    p.logprob[row] = finite && given ? (xt - t.m) - log_sum : nan;
    p.entropy[row] = finite ? entropy : nan;
    p.rank[row] = finite && given ? before : -1;
  }
  if (tid < k) {
    const int i = tid;
    const uint64_t c = sh.best[i];
    p.top_logprob[row * k + i] = finite ? (order_value((uint32_t)(c >> 32)) - t.m) - log_sum : nan;
    p.top_token[row * k + i] = (int64_t)(0xffffffffu - (uint32_t)c);
  }
}

template <typename T, int W>
tf_status launch(const LogprobParams& p, int slices, cudaStream_t s) {
  constexpr int kThreads = 32 * W, kRing = kStages * kThreads * kVectors * 16;
  static PerDeviceOnce once;
  int dev = 0;
  if (once.needed(&dev)) {
    TF_CUDA(cudaFuncSetAttribute(logprobs_kernel<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing));
    once.mark(dev);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * slices));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kRing;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)slices;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T, W>, p);
  if (e != cudaSuccess) return set_error(TF_ERR_CUDA, "token_logprobs launch: %s", cudaGetErrorString(e));
  return check_launch("token_logprobs");
}

}  // namespace

tf_status launch_token_logprobs(const void* logits, int64_t row_stride, int64_t rows, int vocab, int dtype,
                                const int64_t* tokens, int top, float* logprob, float* entropy, int32_t* rank,
                                float* top_logprob, int64_t* top_token, cudaStream_t s) {
  if (rows == 0) return TF_OK;
  if (rows > 2147483647 / kMaxCluster) return set_error(TF_ERR_UNSUPPORTED, "token_logprobs: too many rows");
  LogprobParams p = {logits, row_stride, tokens, rows, vocab, top, logprob, entropy, rank, top_logprob, top_token,
                     nullptr, nullptr};
  TF_TRY(tc_flags(&p.err, const_cast<long long**>(&p.wait_cycles)));
  // Blocks a row: enough to fill the GPU (about two blocks an SM), each
  // with at least one vector a thread.  Whole rows go to blocks of 128 threads,
  // five to an SM: more rows at once cover one another's waits for the prunes.
  const int vectors = vocab / (dtype == TF_DTYPE_F32 ? 4 : 8);
  int slices = 1;
  while (slices < kMaxCluster && rows * slices * 2 <= 2 * 148 && vectors >= 2 * slices * 256) slices *= 2;
#define TF_LOGPROBS(T) return slices > 1 ? launch<T, 8>(p, slices, s) : launch<T, 4>(p, 1, s)
  switch (dtype) {
    case TF_DTYPE_F32: TF_LOGPROBS(float);
    case TF_DTYPE_F16: TF_LOGPROBS(__half);
    default: TF_LOGPROBS(__nv_bfloat16);
  }
#undef TF_LOGPROBS
}

}  // namespace tf
