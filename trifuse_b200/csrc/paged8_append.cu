// New tokens into a paged cache held in 8 bits: full-width RMSNorm of q and k,
// rotation by halves, and codes with a scale for each block of 16 tokens and
// key head.
//
//   k:  x = rope(k * rsqrt(mean(k^2) + eps) * w),   v:  x = v
//   s' = max(s if the block has earlier tokens, max |x| / L),  L = 127 or 448
//   code = rne(x / s'),   earlier codes c become rne(c s / s') where s' > s
//
// What bounds it: each value is read once and written once, half as wide for
// the cache.  A block's scale needs all of its tokens, and a token's norm all
// of its heads, so a thread block takes a window of rows: 16, or one where
// rows are few and latency counts.  A part of a row (q, k, v) goes to thread
// blocks of its own.  Blocks of the cache ("units") belong to the window in
// which their first new row lies; the rows tell by themselves where a unit
// begins (another request, a position that does not follow, a multiple of
// 16), so the call needs no list from the host and can be replayed.
//
// A warp takes one unit of one head at a time: 16 tokens of D values are 64 fp32
// values a thread, from which the maximum, the scale and the codes follow
// without another read.  The sums of squares need the heads of the warps beside
// it, so k and q are read twice, the second time from L1.
//
// fp32 throughout, one rounding to q's type or to a code; the angle is reduced
// in fp64 as in the 16-bit append.
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "paged.h"
#include "paged_codes.cuh"
#include "paged_pairs.cuh"

namespace tf {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kWindow = 16;  // rows of a window where rows are many

struct Append8Params {
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
  uint8_t* codes[2];  // k, v
  float* scales[2];
  int64_t pages, page_stride, scale_stride;
  int page_size, page_shift;
  void* q_out;
  int window;
  unsigned windows;
  int rotate;
  double turns[64];  // theta^(-2d/D) / (2 pi)
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

template <typename T, typename S, int D>
__global__ void __launch_bounds__(kThreads, 2) paged_append_8bit_kernel(const __grid_constant__ Append8Params p) {
  constexpr int kLanes = D / 16;          // threads of a token of a head, 8 values of either half each
  constexpr int kTokens = 32 / kLanes;    // tokens of a pass
  constexpr int kPasses = kScaleTokens / kTokens;
  __shared__ float rot[2][2 * kWindow][D / 2];  // cos and sin of the rows
  __shared__ float sums[kWarps][2 * kWindow];   // a warp's share of the rows' sums of squares
  __shared__ float norm_of[2 * kWindow];
  __shared__ int unit_row[kWindow], unit_rows[kWindow];  // relative to the window; rows of the unit
  __shared__ int64_t unit_page[kWindow];                 // -1: the slot does not exist
  __shared__ int unit_slot[kWindow];
  __shared__ int unit_count, row_end;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = blockIdx.x < p.windows ? 1 : blockIdx.x < 2 * p.windows ? 2 : 0;  // k, v, q
  const int64_t r0 = (int64_t)(blockIdx.x % p.windows) * p.window;
  const int heads = part == 0 ? p.heads : p.kv_heads;

  if (warp == 0) {
    // Lane i looks at row r0 + i; a unit that begins in the window ends within
    // the 31 rows after its start.
    const int64_t row = r0 + lane;
    const bool real = row < p.rows;
    const int pos = real ? p.positions[row] : 0, req = real ? p.requests[row] : 0;
    int before_pos = __shfl_up_sync(0xffffffffu, pos, 1), before_req = __shfl_up_sync(0xffffffffu, req, 1);
    bool first = part == 0 && lane == 0;
    if (part != 0 && real) {
      if (lane == 0 && row > 0) before_pos = p.positions[row - 1], before_req = p.requests[row - 1];
      first = row == 0 || before_req != req || (uint32_t)pos != (uint32_t)before_pos + 1u ||
              (pos & (kScaleTokens - 1)) == 0;
    }
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    const int end = (int)min((int64_t)32, p.rows - r0);  // rows that exist
    if (first && lane < p.window) {
      const uint32_t later = lane < 31 ? firsts >> (lane + 1) : 0u;
      int next = later ? lane + __ffs(later) : end;
      if (part == 0) next = min(p.window, end);
      const int at = __popc(firsts & ((1u << lane) - 1u));
      unit_row[at] = lane;
      unit_rows[at] = next - lane;
      int64_t page = -1;
      if (part != 0) {
        const int column = pos >> p.page_shift;
        if (pos >= 0 && req >= 0 && req < p.table.requests && column < p.table.columns) {
          const int64_t id = p.table.ids[req * p.table.stride + column];
          if (id >= 0 && id < p.pages) page = id;
        }
      }
      unit_page[at] = page;
      unit_slot[at] = pos & (p.page_size - 1);
    }
    if (lane == 0) {
      const uint32_t mine = firsts & ((1u << p.window) - 1u);
      unit_count = __popc(mine);
      const int last = mine ? 31 - __clz(mine) : 0;
      const uint32_t later = last < 31 ? firsts >> (last + 1) : 0u;
      row_end = part == 0 ? min(p.window, end) : later ? last + __ffs(later) : end;
    }
  }
  __syncthreads();
  const int units = unit_count;
  if (units == 0) return;
  const int first_row = unit_row[0], rows = row_end - first_row;  // rows of all units
  const T* src = static_cast<const T*>(p.qkv) + r0 * p.qkv_stride +
                 (int64_t)(part == 0 ? 0 : part == 1 ? p.heads : p.heads + p.kv_heads) * D;
  const __half* norm = part == 0 ? p.q_norm : part == 1 ? p.k_norm : nullptr;
  const bool rotate = p.rotate && part < 2;
  const int tasks = units * heads;
  const int at = lane % kLanes, sub = lane / kLanes;

  uint4 raw[kPasses][2];
  auto load = [&](int task) {
    const int u = task / heads, h = task % heads, n = unit_rows[u];
    const T* x = src + (int64_t)unit_row[u] * p.qkv_stride + h * D + 8 * at;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int t = i * kTokens + sub;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        raw[i][j] = t < n ? ld_v4(x + t * p.qkv_stride + j * (D / 2)) : make_uint4(0, 0, 0, 0);
    }
  };
  const bool once = tasks <= kWarps;  // a warp's only task stays in its registers
  if (warp < tasks) load(warp);

  if (rotate) {
    for (int i = tid; i < rows * (D / 2); i += kThreads) {
      const int r = i / (D / 2), d = i % (D / 2);
      const double t = (double)p.positions[r0 + first_row + r] * p.turns[d];
      float sn, cs;
      sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
      rot[0][r][d] = cs;
      rot[1][r][d] = sn;
    }
  }
  if (norm) {
    sums[warp][lane] = 0.f;
    __syncwarp();
    for (int task = warp; task < tasks; task += kWarps) {
      if (task != warp) load(task);
      const int u = task / heads, n = unit_rows[u];
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float2 f[4];
          unpack4<T>(raw[i][j], f);
#pragma unroll
          for (int k = 0; k < 4; ++k) sum = fma2(f[k], f[k], sum);
        }
        float all = sum.x + sum.y;
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
        const int t = i * kTokens + sub;
        if (at == 0 && t < n) sums[warp][unit_row[u] - first_row + t] += all;  // a token always has the same thread
      }
    }
    __syncthreads();
    if (tid < rows) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += sums[w][tid];
      norm_of[tid] = rms_scale(sum, heads * D, p.eps);
    }
  }
  if (norm || rotate) __syncthreads();

  for (int task = warp; task < tasks; task += kWarps) {
    if (!once && (norm || task != warp)) load(task);
    const int u = task / heads, h = task % heads, n = unit_rows[u], local = unit_row[u] - first_row;
    float2 weight[2][4];
    if (norm) {
#pragma unroll
      for (int j = 0; j < 2; ++j) unpack4<__half>(ld_v4(norm + h * D + j * (D / 2) + 8 * at), weight[j]);
    }
    // Pass i's values: 8 of the first half, their partners in the second.
    auto values = [&](int i, float2 (&f)[2][4]) {
      const int row = min(local + i * kTokens + sub, rows - 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        unpack4<T>(raw[i][j], f[j]);
        if (norm) {
          const float2 scale = make_float2(norm_of[row], norm_of[row]);
#pragma unroll
          for (int k = 0; k < 4; ++k) f[j][k] = mul2(mul2(f[j][k], scale), weight[j][k]);
        }
      }
      if (rotate) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 cs = *reinterpret_cast<const float2*>(&rot[0][row][8 * at + 2 * k]);
          const float2 sn = *reinterpret_cast<const float2*>(&rot[1][row][8 * at + 2 * k]);
          const float2 a = f[0][k], b = f[1][k];
          f[0][k] = fma2(a, cs, mul2(b, make_float2(-sn.x, -sn.y)));
          f[1][k] = fma2(a, sn, mul2(b, cs));
        }
      }
    };
    if (part == 0) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int t = i * kTokens + sub;
        float2 f[2][4];
        values(i, f);
        if (t < n) {
          T* out = static_cast<T*>(p.q_out) + ((r0 + unit_row[u] + t) * heads + h) * D + 8 * at;
#pragma unroll
          for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4*>(out + j * (D / 2)) = pack4<T>(f[j]);
        }
      }
      continue;
    }
    const int64_t page = unit_page[u];
    if (page < 0) continue;
    const int slot = unit_slot[u], earlier = slot & (kScaleTokens - 1);
    uint8_t* block = p.codes[part - 1] + page * p.page_stride + (int64_t)(h * p.page_size + slot - earlier) * D;
    float* scale_at = p.scales[part - 1] + page * p.scale_stride + h * (p.page_size / kScaleTokens) +
                      slot / kScaleTokens;
    const float old = earlier ? *scale_at : 0.f;
    float2 f[kPasses][2][4];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      values(i, f[i]);
      if (i * kTokens + sub < n) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) most = max_nan(most, max_nan(fabsf(f[i][j][k].x), fabsf(f[i][j][k].y)));
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
    float scale = __fdiv_rn(most, Code<S>::kLargest);
    if (most > 0.f) scale = max_nan(scale, 1.17549435e-38f);  // its reciprocal is finite
    if (!(most < INFINITY)) scale = __uint_as_float(0x7fc00000u);
    scale = max_nan(scale, old);
    const float inverse = scale > 0.f && scale < INFINITY ? __fdiv_rn(1.f, scale) : 0.f;
    if (lane == 0) *scale_at = scale;
    if (earlier && scale > old) {
      const float ratio = old * inverse;
      for (int i = lane; i < earlier * (D / 16); i += 32) {
        uint4* at16 = reinterpret_cast<uint4*>(block) + i;
        uint4 v = *at16;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a, b;
          Code<S>::widen(w[k], a, b);
          const float2 x = __half22float2(bits_half2(a)), y = __half22float2(bits_half2(b));
          w[k] = Code<S>::narrow(x.x * ratio, x.y * ratio, y.x * ratio, y.y * ratio);
        }
        *at16 = v;
      }
    }
    const bool finite = scale < INFINITY;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int t = i * kTokens + sub;
      if (t >= n) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 x = f[i][j][2 * k], y = f[i][j][2 * k + 1];
          w[k] = finite ? Code<S>::narrow(x.x * inverse, x.y * inverse, y.x * inverse, y.y * inverse) : 0u;
        }
        *reinterpret_cast<uint2*>(block + (earlier + t) * D + j * (D / 2) + 8 * at) = make_uint2(w[0], w[1]);
      }
    }
  }
}

}  // namespace

tf_status launch_paged_append_8bit(const AppendArgs& a, const tf_paged_scales& scales, cudaStream_t s) {
  if (a.rows == 0) return TF_OK;
  const int D = a.kv.head_dim;
  Append8Params p;
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
  p.codes[0] = static_cast<uint8_t*>(a.kv.k);
  p.codes[1] = static_cast<uint8_t*>(a.kv.v);
  p.scales[0] = scales.k;
  p.scales[1] = scales.v;
  p.pages = a.kv.pages;
  p.page_stride = a.kv.page_stride;
  p.scale_stride = scales.page_stride;
  p.page_size = a.kv.page_size;
  while ((1 << p.page_shift) < a.kv.page_size) ++p.page_shift;
  p.q_out = a.q_out;
  p.rotate = a.theta != 0.f;
  if (p.rotate) {
    // One power, then products: 63 roundings of 2^-53 stay far below fp32.
    const double step = pow((double)a.theta, -2.0 / D);
    double f = 0.15915494309189535;  // 1 / (2 pi)
    for (int d = 0; d < D / 2; ++d, f *= step) p.turns[d] = f;
  }
  // Windows of 16 rows where they give every SM a block of each part.
  p.window = a.rows >= 148 * kWindow / 3 ? kWindow : 1;
  const int64_t windows = (a.rows + p.window - 1) / p.window;
  if (windows > 2147483647LL / 3) return set_error(TF_ERR_UNSUPPORTED, "paged_append: too many rows");
  p.windows = (unsigned)windows;
  const unsigned grid = 3 * p.windows;
#define TF_APPEND8(T, S)                                                              \
  do {                                                                                \
    if (D == 128)                                                                     \
      paged_append_8bit_kernel<T, S, 128><<<grid, kThreads, 0, s>>>(p);               \
    else                                                                              \
      paged_append_8bit_kernel<T, S, 64><<<grid, kThreads, 0, s>>>(p);                \
    return check_launch("paged_append_8bit");                                         \
  } while (0)
  const bool ints = a.kv.dtype == TF_DTYPE_I8;
  if (a.act == TF_DTYPE_F16) {
    if (ints) TF_APPEND8(__half, I8);
    TF_APPEND8(__half, E4M3);
  }
  if (ints) TF_APPEND8(__nv_bfloat16, I8);
  TF_APPEND8(__nv_bfloat16, E4M3);
#undef TF_APPEND8
}

}  // namespace tf
