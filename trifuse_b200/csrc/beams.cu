// Beam selection: the best continuations of a request over its beams and the
// vocabulary.
//
//   total(b, t) = score_b + (x_bt - m_b) - ln sum_t e^(x_bt - m_b)
//
// The pass over the logits (logprobs.cu) leaves of each beam its m, its log sum
// and its first `count` tokens, in order.  No other token can be among the
// first `count` of the request, so a block a request merges these lists: a
// candidate's place is its place in its own list plus, for every other list,
// the number of entries ahead of it (a binary search).
//
// Totals are formed in fp64, but the pass sums fp32 exponentials: a log sum was
// off by up to 4.6e-7 (flat, rising, scattered and peaked rows of 1000 to 600000
// logits; 1.0e-6 at two million, rising in steps).  Where two candidates of
// different beams that matter lie closer than ten times the sum of two such errors,
// their rows are summed again in fp64, so which beam goes on does not hang on a
// rounding; an exact total may lie close to another rough one, so this goes on
// until none does (each row is summed again once at most, one after the other).  At
// eight beams a batch of 64 requests meets that about once in fifty steps, and a
// pair of rows of 50304 then takes 120 to 135 us more; 64 beams with equal totals
// sum 64 rows, 3.8 ms.
//
// What bounds it: the logits, read once; this kernel's block is latency (some
// 64 candidates, a few round trips).  Measured: 64 x 8 beams over 50304 fp32 logits
// 29.5 us, of which the pass 26 (3.9 TB/s: 512 rows are 3 or 4 to an SM, and a row's
// prunes meet at barriers), f16 or bf16 ones 24.5; one request of 4 beams 11.2 to 11.7.
#include <math.h>

#include "beams.h"
#include "common.cuh"

namespace tf {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBeams = TF_MAX_BEAMS;
constexpr int kMaxCount = TF_MAX_TOP;
// Closer than this, totals are told apart in fp64.  Of the roundings only a thread's
// additions to its sum grow with the row: V / 4096 of them (a tile each), of 2^-24
// at most and possibly all one way, in two rows 2.9e-11 V.
__device__ __forceinline__ double near_by(int V) { return fmax(1e-5, 3e-11 * V); }

// From here down totals are -inf in fp32: -(2^128 - 2^103).
constexpr double kNone = -3.4028235677973366e38;

struct SelectParams {
  BeamArgs a;
  int each;
};

// The first index in [0, n) of a falling list whose entry is not ahead of
// `total`: entries that are greater, or (kEqual) equal, are ahead.
template <bool kEqual>
__device__ __forceinline__ int ahead(const double* list, int n, double total) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (kEqual ? list[mid] >= total : list[mid] > total)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v, double* warps) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  double sum = 0.;
  for (int w = 0; w < kThreads / 32; ++w) sum += warps[w];
  return sum;
}

// ln sum e^(x - m) of a row in fp64, by the whole block.
template <typename T>
__device__ __noinline__ double row_log_sum(const T* x, int V, float m, double* warps) {
  double sum = 0.;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    float v;
    if constexpr (sizeof(T) == 4)
      v = x[i];
    else
      v = to_f(x[i]);
    const double d = (double)v - (double)m;
    if (d > -60.) sum += exp(d);  // below e^-60 a million of them are nothing in fp64
  }
  return log(block_sum(sum, warps));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) beam_select_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ double totals[];  // [beams][each]
  __shared__ int n_of[kMaxBeams];
  __shared__ double base[kMaxBeams];  // score - log sum: what a token's x - m is added to
  __shared__ float m_of[kMaxBeams];
  __shared__ double best[kMaxCount];
  __shared__ int best_at[kMaxCount];  // beam * each + place
  __shared__ int near[kMaxBeams];
  __shared__ int any_near;
  __shared__ double warps[kThreads / 32];
  const BeamArgs& a = p.a;
  const int tid = threadIdx.x, beams = a.beams, each = p.each, count = a.count;
  const int64_t row0 = (int64_t)blockIdx.x * beams;
  const uint64_t* keys = a.keys() + row0 * each;
  float score = 0.f;
  bool ended = false;
  if (tid < beams) {
    score = a.scores[row0 + tid];
    ended = a.finished && a.finished[row0 + tid];
    near[tid] = 0;
  }
  if (tid < count) best_at[tid] = -1;
  if (tid == 0) any_near = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows are written
  if (tid < beams) {
    const BeamRow r = a.rows()[row0 + tid];
    const bool live = fabsf(score) < INFINITY;
    n_of[tid] = !live ? 0 : ended ? 1 : r.n;
    base[tid] = (double)score - r.log_sum;
    m_of[tid] = ended ? INFINITY : r.m;  // +inf: an ended beam, whose one candidate is its score
  }
  __syncthreads();
  const auto fill = [&](int b, int j) {
    if (m_of[b] == INFINITY) {
      totals[b * each + j] = base[b];
      return;
    }
    const float x = order_value((uint32_t)(keys[b * each + j] >> 32));
    totals[b * each + j] = base[b] + ((double)x - (double)m_of[b]);
  };
  for (int i = tid; i < beams * each; i += kThreads) {
    const int b = i / each, j = i % each;
    if (j < n_of[b]) fill(b, j);
  }
  __syncthreads();
  // Tokens at -inf cannot follow, nor those whose score fp32 does not hold; they end
  // their lists.  (Rows that are summed again below move by less than fp64's steps
  // there.)
  if (tid < beams) {
    const double* list = totals + tid * each;
    n_of[tid] = ahead<false>(list, n_of[tid], kNone);
  }
  __syncthreads();
  const auto order = [&]() {
    for (int i = tid; i < beams * each; i += kThreads) {
      const int b = i / each, j = i % each;
      if (j >= n_of[b]) continue;
      const double total = totals[i];
      int place = j;
      for (int o = 0; o < beams && place < count; ++o) {
        if (o == b) continue;
        // More than `count` of another list need not be told apart.
        const int n = min(n_of[o], count - place);
        place += o < b ? ahead<true>(totals + o * each, n, total) : ahead<false>(totals + o * each, n, total);
      }
      if (place < count) {
        best[place] = total;
        best_at[place] = i;
      }
    }
    __syncthreads();
  };
  order();
  // Until no pair is left that hangs on a rounding: neighbours among the picked
  // ones, and the last of them with all that were not picked.
  for (;;) {
    const auto close = [&](int one, int other, double apart) {
      const int b = one / each, c = other / each;
      if (b == c || !(fabs(apart) < near_by(a.vocab))) return;
      for (int beam : {b, c})
        if (near[beam] == 0) near[beam] = any_near = 1;  // 2: summed again
    };
    if (tid + 1 < count && best_at[tid + 1] >= 0) close(best_at[tid], best_at[tid + 1], best[tid] - best[tid + 1]);
    if (best_at[count - 1] >= 0)
      for (int i = tid; i < beams * each; i += kThreads)
        if (i % each < n_of[i / each]) close(best_at[count - 1], i, best[count - 1] - totals[i]);
    __syncthreads();
    if (!any_near) break;
    for (int b = 0; b < beams; ++b) {
      if (near[b] != 1) continue;
      if (m_of[b] != INFINITY) {
        const double log_sum =
            row_log_sum(static_cast<const T*>(a.logits) + (row0 + b) * a.row_stride, a.vocab, m_of[b], warps);
        if (tid == 0) base[b] = (double)a.scores[row0 + b] - log_sum;
        __syncthreads();
        if (tid < n_of[b]) fill(b, tid);
      }
    }
    __syncthreads();
    if (tid < beams && near[tid] == 1) near[tid] = 2;
    if (tid == 0) any_near = 0;
    order();
  }
  if (tid < count) {
    const int64_t to = (int64_t)blockIdx.x * count + tid;
    const int at = best_at[tid];
    a.score[to] = at < 0 ? -INFINITY : (float)best[tid];
    a.parent[to] = at < 0 ? -1 : at / each;
    a.token[to] = at < 0                              ? -1
                  : m_of[at / each] == INFINITY ? a.end
                                                      : (int64_t)(0xffffffffu - (uint32_t)keys[at]);
  }
}

template <typename T>
tf_status launch(const SelectParams& p, cudaStream_t s) {
  const size_t smem = (size_t)p.a.beams * p.each * sizeof(double);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.a.requests);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  // Launched while the rows' last blocks still run; it waits on the device.
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TF_CUDA(cudaLaunchKernelEx(&cfg, beam_select_kernel<T>, p));
  return check_launch("beam_select");
}

}  // namespace

tf_status launch_beam_select(const BeamArgs& a, cudaStream_t s) {
  TF_TRY(launch_beam_rows(a, s));
  const SelectParams p = {a, a.each()};
  switch (a.dtype) {
    case TF_DTYPE_F32: return launch<float>(p, s);
    case TF_DTYPE_F16: return launch<__half>(p, s);
    default: return launch<__nv_bfloat16>(p, s);
  }
}

}  // namespace tf
