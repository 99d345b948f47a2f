// Log probabilities of given tokens, with entropy, rank and the top
// alternatives, in one pass over the logits.
//
//   m = max x,  s = sum e^(x - m),  w = sum (x - m) e^(x - m)
//   log p(t) = (x_t - m) - ln s,   entropy = ln s - w / s
//   rank(t)  = number of entries before t in the order (value down, index up)
//   alternatives: the first k entries of that order (NaN last)
//
// What bounds it: each logit is read once; 50304 fp32 logits are 0.2 MB, 31 ns
// of the whole GPU's bandwidth.  So the pass keeps every value in registers
// for all of its uses: a tile of 8 vectors of 16 bytes a thread is loaded at
// once, its maximum taken, then the exponentials and both sums relative to the
// thread's running maximum (rescaled when that moves).  Differences are taken
// before the scaling by log2 e, so the leading terms carry no rounding of m.
//
// The alternatives ride along as candidates: a composite key (ordered value
// bits, then the inverted index) makes every entry distinct and ties fall to
// the lowest index.  The first tile yields a lower bound of the k-th key (the
// smallest over the warps of their ceil(k / 8)-th largest thread maximum: at
// least k entries are at or above it), entries at or above the bound go to a
// shared buffer, and pruning the buffer to its k best raises the bound to an
// exact one.  After the first tile a thread whose maximum is below the bound
// does nothing, so the pass stays a stream.  Should a tile's candidates not
// fit the buffer (values in rising order, say), they enter in rounds of one
// vector element a thread with a prune in between.
//
// A row may be shared by a cluster of 1, 2, 4 or 8 blocks (few rows: the whole
// GPU reads; one row of 50304 on one block would take its load latency 25
// times over); the blocks' sums and candidates meet in the first block's hands
// over distributed shared memory, so no scratch in device memory is needed.
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"
#include "internal.h"

namespace tf {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kVectors = 8;     // 16-byte vectors a thread holds
constexpr int kMaxTop = 64;
constexpr int kBuffer = 1024;   // candidates: the rounds need kMaxTop + kThreads, the cluster's join kMaxCluster * kMaxTop
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

template <typename T>
struct Lane;
template <>
struct Lane<float> {
  static constexpr int kPer = 4;
  __device__ __forceinline__ static float get(const uint4& v, int i) {
    return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static constexpr uint32_t kNegInf = 0xff800000u;
  __device__ __forceinline__ static float max_of(const uint4& v) {
    return max_nan(max_nan(get(v, 0), get(v, 1)), max_nan(get(v, 2), get(v, 3)));
  }
};
template <typename T>
struct Lane16 {
  static constexpr int kPer = 8;
  __device__ __forceinline__ static uint32_t word(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  }
};
template <>
struct Lane<__half> : Lane16<__half> {
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  __device__ __forceinline__ static float get(const uint4& v, int i) {
    const uint32_t w = word(v, i >> 1);
    return __half2float(__ushort_as_half((unsigned short)((i & 1) ? w >> 16 : w & 0xffffu)));
  }
  __device__ __forceinline__ static float max_of(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};
template <>
struct Lane<__nv_bfloat16> : Lane16<__nv_bfloat16> {
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  __device__ __forceinline__ static float get(const uint4& v, int i) {
    const uint32_t w = word(v, i >> 1);
    return __uint_as_float((i & 1) ? w & 0xffff0000u : w << 16);
  }
  __device__ __forceinline__ static float max_of(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};

// Running sums relative to a maximum m, in log2 units: s = sum 2^d, w = sum d 2^d, d = (x - m) log2 e.
struct Sums {
  float m, s, w;
  __device__ __forceinline__ void move(float to) {  // to >= m, or NaN
    if (m == -INFINITY) {  // nothing but -inf so far: s = w = 0
      m = to;
    } else if (to != m) {
      const float d = (m - to) * kLog2e, f = exp2_fast(d);
      w = f == 0.f ? 0.f : f * fmaf(d, s, w);
      s *= f;
      m = to;
    }
  }
  __device__ __forceinline__ void join(Sums o) {
    const float to = max_nan(m, o.m);
    move(to);
    o.move(to);
    s += o.s;
    w += o.w;
  }
};

struct Shared {
  uint64_t buffer[kBuffer];
  uint64_t best[kMaxTop];      // sorted k best of the last prune
  uint64_t bound;              // entries below it are no candidates
  int n;                       // candidates in the buffer
  int overflow;
  uint32_t warp_key[kWarps];
  Sums warp_sums[kWarps];
  int warp_before[kWarps];
  Sums sums;   // the block's totals, which the cluster's first block collects
  int before;
};

// Sorts the buffer's n distinct keys by counting, keeps the k best (in best[],
// and at the buffer's front) and raises the bound.  Called by the whole block
// after a barrier; ends with one.
__device__ __forceinline__ void prune(Shared& sh, int k) {
  const int n = sh.n;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = sh.buffer[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.buffer[j] > mine;
    if (rank < k) sh.best[rank] = mine;
  }
  __syncthreads();
  const int keep = n < k ? n : k;
  for (int i = threadIdx.x; i < keep; i += kThreads) sh.buffer[i] = sh.best[i];
  if (threadIdx.x == 0) {
    sh.n = keep;
    if (n >= k) sh.bound = sh.best[k - 1] + 1;
  }
  __syncthreads();
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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Vector of kPer values from index e0, entries outside [0, V) read as -inf.
template <typename T>
__device__ __forceinline__ uint4 load_ragged(const T* x, int e0, int V) {
  constexpr int kPer = Lane<T>::kPer;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = Lane<T>::kNegInf;
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) logprobs_kernel(const __grid_constant__ LogprobParams p) {
  using L = Lane<T>;
  constexpr int kPer = L::kPer;
  __shared__ Shared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = (int)cluster.num_blocks(), slice = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / slices;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int V = p.vocab, k = p.top;
  // Vectors are counted from the 16-byte boundary at or before the row.
  const int head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int vectors = (V + head + kPer - 1) / kPer;
  const int v_begin = (int)((int64_t)vectors * slice / slices);
  const int v_end = (int)((int64_t)vectors * (slice + 1) / slices);

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
  if (tid == 0) {
    sh.n = 0;
    sh.overflow = 0;
    sh.bound = 0;
  }
  __syncthreads();

  Sums acc = {-INFINITY, 0.f, 0.f};
  int before = 0;
  uint64_t bound = 0;
  int kept = 0;  // candidates in the buffer when the tile began
  for (int t0 = v_begin; t0 < v_end; t0 += kThreads * kVectors) {
    uint4 r[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int v = t0 + tid + i * kThreads;
      const int e0 = v * kPer - head;
      if (v >= v_end)
        r[i] = make_uint4(L::kNegInf, L::kNegInf, L::kNegInf, L::kNegInf);
      else if (e0 >= 0 && e0 + kPer <= V)
        r[i] = ld_stream_v4(x + e0);
      else
        r[i] = load_ragged<T>(x, e0, V);
    }
    float vmax[kVectors], tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      vmax[i] = L::max_of(r[i]);
      tmax = max_nan(tmax, vmax[i]);
    }
    // Sums.  d is held above -150, where 2^d is zero in fp32: a logit of -inf
    // adds 0 to both sums and not 0 * -inf.
    const float to = max_nan(acc.m, tmax);
    acc.move(to);
    if (to != -INFINITY) {
      const uint64_t sub = pair(-to, -to), log2e = pair(kLog2e, kLog2e);
      uint64_t s2[2] = {0, 0}, w2[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < kPer; j += 2) {
          float d0, d1;
          unpair(mul2(add2(pair(L::get(r[i], j), L::get(r[i], j + 1)), sub), log2e), d0, d1);
          d0 = fmaxf(d0, -150.f);
          d1 = fmaxf(d1, -150.f);
          const uint64_t e = pair(exp2_fast(d0), exp2_fast(d1));
          s2[i & 1] = add2(s2[i & 1], e);
          w2[i & 1] = fma2(pair(d0, d1), e, w2[i & 1]);
        }
      float a, b;
      unpair(add2(s2[0], s2[1]), a, b);
      acc.s += a + b;
      unpair(add2(w2[0], w2[1]), a, b);
      acc.w += a + b;
    }
    // Rank of the given token.
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int v = t0 + tid + i * kThreads, e0 = v * kPer - head;
      if (vmax[i] < xt || v >= v_end) continue;
      if (e0 > token) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) before += L::get(r[i], j) > xt;
      } else if (e0 >= 0 && e0 + kPer <= token) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) before += L::get(r[i], j) >= xt;
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const float v = L::get(r[i], j);
          before += v > xt || (v == xt && e0 + j >= 0 && e0 + j < token);
        }
      }
    }
    if (k == 0) continue;
    // Candidates.
    if (t0 == v_begin) {
      const int each = (k + kWarps - 1) / kWarps;
      uint32_t key = t0 + tid < v_end ? order_bits(tmax) : 0u, kth = 0;
      for (int i = 0; i < each; ++i) {
        kth = __reduce_max_sync(0xffffffffu, key);
        const uint32_t who = __ballot_sync(0xffffffffu, key == kth);
        if (lane == __ffs(who) - 1) key = 0;
      }
      if (lane == 0) sh.warp_key[warp] = kth;
      __syncthreads();
      uint32_t low = sh.warp_key[0];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) low = min(low, sh.warp_key[i]);
      bound = (uint64_t)low << 32;
      if (tid == 0) sh.bound = bound;
    }
    const uint32_t bound_bits = (uint32_t)(bound >> 32);
    const float cut = bound_bits ? order_value(bound_bits) : -INFINITY;
    if (!(tmax < cut)) {
      int count = 0;
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        if (vmax[i] < cut) continue;
        const int v = t0 + tid + i * kThreads, e0 = v * kPer - head;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          count += v < v_end && e0 + j >= 0 && e0 + j < V && composite(L::get(r[i], j), (uint32_t)(e0 + j)) >= bound;
      }
      if (count) {
        int at = atomicAdd(&sh.n, count);
        if (at + count > kBuffer) {
          sh.overflow = 1;
        } else {
#pragma unroll
          for (int i = 0; i < kVectors; ++i) {
            if (vmax[i] < cut) continue;
            const int v = t0 + tid + i * kThreads, e0 = v * kPer - head;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
              const uint64_t c = composite(L::get(r[i], j), (uint32_t)(e0 + j));
              if (v < v_end && e0 + j >= 0 && e0 + j < V && c >= bound) sh.buffer[at++] = c;
            }
          }
        }
      }
    }
    __syncthreads();
    const int n = sh.n;
    const bool overflow = sh.overflow != 0;
    __syncthreads();
    if (overflow) {
      // The tile again, kThreads entries at a time from memory.
      if (tid == 0) {
        sh.n = kept;
        sh.overflow = 0;
      }
      __syncthreads();
      const int v_last = min(v_end, t0 + kThreads * kVectors);
      const int e_last = min(V, v_last * kPer - head);
      for (int e = t0 * kPer - head; e < e_last; e += kThreads) {
        const int mine = e + tid;
        if (mine >= 0 && mine < e_last) {
          float v;
          if constexpr (kPer == 4)
            v = reinterpret_cast<const float*>(x)[mine];
          else
            v = to_f(x[mine]);
          const uint64_t c = composite(v, (uint32_t)mine);
          if (c >= bound) sh.buffer[atomicAdd(&sh.n, 1)] = c;
        }
        __syncthreads();
        const bool full = sh.n > kBuffer - kThreads;
        __syncthreads();
        if (full) {
          prune(sh, k);
          bound = sh.bound;
        }
      }
      prune(sh, k);
      bound = sh.bound;
    } else if (n > 2 * k + 32 || t0 == v_begin) {
      prune(sh, k);
      bound = sh.bound;
    }
    kept = sh.n;
    __syncthreads();
  }

  // Block totals.
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    Sums o;
    o.m = __shfl_xor_sync(0xffffffffu, acc.m, off);
    o.s = __shfl_xor_sync(0xffffffffu, acc.s, off);
    o.w = __shfl_xor_sync(0xffffffffu, acc.w, off);
    acc.join(o);
    before += __shfl_xor_sync(0xffffffffu, before, off);
  }
  if (lane == 0) {
    sh.warp_sums[warp] = acc;
    sh.warp_before[warp] = before;
  }
  __syncthreads();
  if (k) prune(sh, k);
  if (tid == 0) {
    Sums t = sh.warp_sums[0];
    int b = sh.warp_before[0];
    for (int i = 1; i < kWarps; ++i) {
      t.join(sh.warp_sums[i]);
      b += sh.warp_before[i];
    }
    sh.sums = t;
    sh.before = b;
  }
  if (slices > 1) {
    cluster.sync();
    if (slice == 0) {
      if (tid == 0) {
        Sums t = sh.sums;
        int b = sh.before;
        for (int i = 1; i < slices; ++i) {
          const Shared* o = cluster.map_shared_rank(&sh, i);
          t.join(o->sums);
          b += o->before;
        }
        sh.sums = t;
        sh.before = b;
      }
      if (k) {
        int at = sh.n;
        for (int i = 1; i < slices; ++i) {
          const Shared* o = cluster.map_shared_rank(&sh, i);
          const int n = o->n;
          for (int j = tid; j < n; j += kThreads) sh.buffer[at + j] = o->best[j];
          at += n;
        }
        __syncthreads();
        if (tid == 0) sh.n = at;
        __syncthreads();
        prune(sh, k);
      }
    }
    cluster.sync();  // the other blocks' shared memory stays until it has been read
    if (slice != 0) return;
  }
  __syncthreads();
  const Sums t = sh.sums;
  const bool finite = fabsf(t.m) < INFINITY;  // no NaN, no +inf, not all -inf
  const float log_sum = logf(t.s);
  const float nan = __uint_as_float(0x7fc00000u);
  if (tid == 0) {
    p.logprob[row] = finite && given ? (xt - t.m) - log_sum : nan;
    p.entropy[row] = finite ? log_sum - t.w / t.s * kLn2 : nan;
    p.rank[row] = finite && given ? sh.before : -1;
  }
  for (int i = tid; i < k; i += kThreads) {
    const uint64_t c = sh.best[i];
    p.top_logprob[row * k + i] = finite ? (order_value((uint32_t)(c >> 32)) - t.m) - log_sum : nan;
    p.top_token[row * k + i] = (int64_t)(0xffffffffu - (uint32_t)c);
  }
}

template <typename T>
tf_status launch(const LogprobParams& p, int slices, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * slices));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)slices;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p);
  if (e != cudaSuccess) return set_error(TF_ERR_CUDA, "token_logprobs launch: %s", cudaGetErrorString(e));
  return check_launch("token_logprobs");
}

}  // namespace

tf_status launch_token_logprobs(const void* logits, int64_t row_stride, int64_t rows, int vocab, int dtype,
                                const int64_t* tokens, int top, float* logprob, float* entropy, int32_t* rank,
                                float* top_logprob, int64_t* top_token, cudaStream_t s) {
  if (rows == 0) return TF_OK;
  if (rows > 2147483647 / kMaxCluster) return set_error(TF_ERR_UNSUPPORTED, "token_logprobs: too many rows");
  const LogprobParams p = {logits, row_stride, tokens, rows, vocab, top, logprob, entropy, rank, top_logprob,
                           top_token};
  // Blocks a row: enough to fill the GPU (about three blocks an SM), each
  // with at least one vector a thread.
  const int vectors = vocab / (dtype == TF_DTYPE_F32 ? 4 : 8);
  int slices = 1;
  while (slices < kMaxCluster && rows * slices * 2 <= 3 * 148 && vectors >= 2 * slices * kThreads) slices *= 2;
  switch (dtype) {
    case TF_DTYPE_F32: return launch<float>(p, slices, s);
    case TF_DTYPE_F16: return launch<__half>(p, slices, s);
    default: return launch<__nv_bfloat16>(p, slices, s);
  }
}

}  // namespace tf
