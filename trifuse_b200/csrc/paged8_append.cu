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
// A warp takes two heads of a unit at a time and keeps their 16-bit values in
// registers (with more than 16 heads to 8 warps it reads them again, from L1);
// what it makes of them is made twice, for the block's maximum and for the
// codes, which is less than to keep it.  A norm's factor is the same for a
// token's values, so the maximum is taken before it; here it comes after the weight
// and the rotation, on the path of single tokens before them, as in the 16-bit
// append: the last bit of a value may depend on the number of rows of a call.  A window's rows are under
// way before its units are known, for in a long prompt they are all one unit.
// One token (a decode step) takes a path without windows: three dependent round
// trips to memory, a head on 8 threads.
//
// fp32 throughout, one rounding to q's type or to a code; the angle is reduced
// in fp64 as in the 16-bit append.
//
// Measured: 16384 rows of 16 + 2 x 16 heads of 128 with norms and rotation, e4m3:
// 91 us, 3.7 TB/s (without either 73; in 16 bits 85, of 1.3 times the bytes), at 16
// warps an SM (24 and 32 with one head each were no faster); 64 single tokens 4.0
// us (on the windows' path 10.5).
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

// The largest magnitude of 16 values, NaN kept.
__device__ __forceinline__ float largest(const float2 (&f)[2][4]) {
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(f[j][k].x), "f"(f[j][k].y));
  return most;
}

// A block's scale: `most` of its new tokens, `old` of its earlier ones (0: none).
template <typename S>
__device__ __forceinline__ float block_scale(float most, float old) {
  float scale = __fdiv_rn(most, Code<S>::kLargest);
  if (most > 0.f) scale = max_nan(scale, 1.17549435e-38f);  // its reciprocal is finite
  if (!(most < INFINITY)) scale = __uint_as_float(0x7fc00000u);
  return max_nan(scale, old);
}

// `n` vectors of earlier codes at the scale `old`; lane `lane` of `lanes`.
template <typename S>
__device__ __forceinline__ void round_anew(uint8_t* block, int n, float old, const Divisor& over, int lane, int lanes) {
  const float2 old2 = make_float2(old, old);
  for (int i = lane; i < n; i += lanes) {
    uint4* at = reinterpret_cast<uint4*>(block) + i;
    uint4 v = *at;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t a, b;
      Code<S>::widen(w[k], a, b);
      const float2 x = __half22float2(bits_half2(a)), y = __half22float2(bits_half2(b));
      w[k] = Code<S>::narrow(over(mul2(x, old2)), over(mul2(y, old2)));
    }
    *at = v;
  }
}

// 16 values as codes: 8 at `to`, 8 half a head on.
template <typename S, int D>
__device__ __forceinline__ void put_codes(uint8_t* to, const float2 (&f)[2][4], bool finite, const Divisor& over) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint2 w = make_uint2(Code<S>::narrow(over(f[j][0]), over(f[j][1])), Code<S>::narrow(over(f[j][2]), over(f[j][3])));
    if (!finite) w = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(to + j * (D / 2)) = w;
  }
}

// cos and sin of an angle of `turns` turns.  For keys, what the angle loses by its
// rounding turns them on (half as many codes fall to the other side of a
// rounding); q's angle is the 16-bit append's.
__device__ __forceinline__ void turn(double turns, bool key, float& cs, float& sn) {
  const double half = 2. * (turns - rint(turns));  // half turns
  const float rough = (float)half;
  sincospif(rough, &sn, &cs);
  if (key) {
    const float rest = (float)(half - (double)rough) * 3.14159265f, c = cs;
    cs = fmaf(-rest, sn, c);
    sn = fmaf(rest, c, sn);
  }
}

// Eight values of a head's first half and their partners: normalised, rotated.
__device__ __forceinline__ void rotate_pairs(float2 (&f)[2][4], const float* cs, const float* sn) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const float4 c = *reinterpret_cast<const float4*>(cs + 2 * k), s = *reinterpret_cast<const float4*>(sn + 2 * k);
#pragma unroll
    for (int l = 0; l < 2; ++l) {
      const float2 c2 = l ? make_float2(c.z, c.w) : make_float2(c.x, c.y);
      const float2 s2 = l ? make_float2(s.z, s.w) : make_float2(s.x, s.y);
      const float2 a = f[0][k + l], b = f[1][k + l];
      f[0][k + l] = fma2(a, c2, mul2(b, make_float2(-s2.x, -s2.y)));
      f[1][k + l] = fma2(a, s2, mul2(b, c2));
    }
  }
}

// The page of a token, -1 where its slot does not exist.
__device__ __forceinline__ int64_t page_of(const Append8Params& p, int pos, int req) {
  const int column = pos >> p.page_shift;
  if (pos < 0 || req < 0 || req >= p.table.requests || column >= p.table.columns) return -1;
  const int64_t id = p.table.ids[req * p.table.stride + column];
  return id >= 0 && id < p.pages ? id : -1;
}

struct Window {
  float rot[2][2 * kWindow][64];       // cos and sin of the rows
  float sums[kWarps][2 * kWindow];     // a warp's share of the rows' sums of squares
  float norm_of[2 * kWindow];
  int64_t unit_page[kWindow];          // -1: the slot does not exist
  int unit_slot[kWindow];
  int unit_row[kWindow], unit_rows[kWindow];  // relative to the window; rows of the unit
  int unit_count, row_end;
};

// One token that is a unit of its own: what a decode step brings.  All loads
// whose addresses are known are under way at once: the token's values, its
// position and those beside it, then the page, then the blocks' scales.  A head
// takes kLanes threads, so a block of 8 warps 32 heads (of 128) at a time.
template <typename T, typename S, int D>
__device__ __forceinline__ bool append_one(const Append8Params& p, int part, int64_t row, Window& w) {
  constexpr int kLanes = D / 16, kHeads = kThreads / kLanes;  // heads at a time
  constexpr int kKept = 2;                                    // rounds of heads that stay in registers
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, at = tid % kLanes;
  const int heads = part == 0 ? p.heads : p.kv_heads;
  const T* x = static_cast<const T*>(p.qkv) + row * p.qkv_stride +
               (int64_t)(part == 0 ? 0 : part == 1 ? p.heads : p.heads + p.kv_heads) * D + 8 * at;
  uint4 raw[kKept][2];
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    const int h = tid / kLanes + i * kHeads;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      raw[i][j] = h < heads ? ld_v4(x + h * D + j * (D / 2)) : make_uint4(0, 0, 0, 0);
  }
  const int pos = p.positions[row], req = p.requests[row];
  if (part != 0) {
    const bool has_next = row + 1 < p.rows, has_last = row > 0;
    const int next = has_next ? p.positions[row + 1] : 0, next_req = has_next ? p.requests[row + 1] : 0;
    const int last = has_last ? p.positions[row - 1] : 0, last_req = has_last ? p.requests[row - 1] : 0;
    const bool joins = has_last && last_req == req && (uint32_t)pos == (uint32_t)last + 1u &&
                       (pos & (kScaleTokens - 1)) != 0;
    if (joins) return true;  // its unit's first row brings it
    if (has_next && next_req == req && (uint32_t)next == (uint32_t)pos + 1u && (next & (kScaleTokens - 1)) != 0)
      return false;  // more rows in the unit
  }
  const __half* norm = part == 0 ? p.q_norm : part == 1 ? p.k_norm : nullptr;
  const bool rotate = p.rotate && part < 2;
  const int64_t page = part == 0 ? -1 : page_of(p, pos, req);
  const int slot = pos & (p.page_size - 1), earlier = slot & (kScaleTokens - 1);
  const auto scale_of = [&](int h) {
    return p.scales[part - 1] + page * p.scale_stride + h * (p.page_size / kScaleTokens) + slot / kScaleTokens;
  };
  float old[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    const int h = tid / kLanes + i * kHeads;
    old[i] = page >= 0 && earlier && h < heads ? *scale_of(h) : 0.f;
  }
  if (rotate && tid < D / 2) turn((double)pos * p.turns[tid], part == 1, w.rot[0][0][tid], w.rot[1][0][tid]);
  if (norm) {
    float2 sum = make_float2(0.f, 0.f);
    for (int h = tid / kLanes, i = 0; h < heads; h += kHeads, ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float2 f[4];
        unpack4<T>(i == 0 ? raw[0][j] : i == 1 ? raw[1][j] : ld_v4(x + h * D + j * (D / 2)), f);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum = fma2(f[k], f[k], sum);
      }
    const float all = warp_sum_butterfly(sum.x + sum.y);
    if (lane == 0) w.sums[warp][0] = all;
  }
  if (norm || rotate) __syncthreads();
  float2 scale2 = make_float2(1.f, 1.f);
  if (norm) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) sum += w.sums[i][0];
    scale2.x = scale2.y = rms_scale(sum, heads * D, p.eps);
  }
  if (part != 0 && page < 0) return true;
  // Whole warps go round, for the maxima of their heads.
  for (int h0 = 0, i = 0; h0 < heads; h0 += kHeads, ++i) {
    const int h = h0 + tid / kLanes;
    const bool mine = h < heads;
    float2 f[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unpack4<T>(i == 0   ? raw[0][j]
                 : i == 1 ? raw[1][j]
                 : mine   ? ld_v4(x + h * D + j * (D / 2))
                          : make_uint4(0, 0, 0, 0),
                 f[j]);
      if (norm && mine) {
        float2 g[4];
        unpack4<__half>(ld_v4(norm + h * D + j * (D / 2) + 8 * at), g);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[j][k] = mul2(mul2(f[j][k], scale2), g[k]);
      }
    }
    if (rotate) rotate_pairs(f, &w.rot[0][0][8 * at], &w.rot[1][0][8 * at]);
    if (part == 0) {
      T* out = static_cast<T*>(p.q_out) + (row * heads + h) * D + 8 * at;
      if (mine) {
#pragma unroll
        for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4*>(out + j * (D / 2)) = pack4<T>(f[j]);
      }
      continue;
    }
    // Read before the head's threads meet in the shuffles, written after.
    const float before = i == 0 ? old[0] : i == 1 ? old[1] : earlier && mine ? *scale_of(h) : 0.f;
    float most = largest(f);
#pragma unroll
    for (int off = 1; off < kLanes; off <<= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
    if (!mine) continue;
    const float scale = block_scale<S>(most, before);
    const Divisor over(scale);
    uint8_t* block = p.codes[part - 1] + page * p.page_stride + (int64_t)(h * p.page_size + slot - earlier) * D;
    if (earlier && scale > before) round_anew<S>(block, earlier * (D / 16), before, over, at, kLanes);
    if (at == 0) *scale_of(h) = scale;
    put_codes<S, D>(block + earlier * D + 8 * at, f, scale < INFINITY, over);
  }
  return true;
}

// The units of a window (part 0: its rows as one), by warp 0.
__device__ __forceinline__ void find_units(const Append8Params& p, int part, int64_t r0, int lane, Window& w) {
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
    w.unit_row[at] = lane;
    w.unit_rows[at] = next - lane;
    w.unit_page[at] = part != 0 ? page_of(p, pos, req) : -1;
    w.unit_slot[at] = pos & (p.page_size - 1);
  }
  if (lane == 0) {
    const uint32_t mine = firsts & ((1u << p.window) - 1u);
    w.unit_count = __popc(mine);
    const int last = mine ? 31 - __clz(mine) : 0;
    const uint32_t later = last < 31 ? firsts >> (last + 1) : 0u;
    w.row_end = part == 0 ? min(p.window, end) : later ? last + __ffs(later) : end;
  }
}

// One part of a window's rows: q (0), k (1) or v (2).
template <typename T, typename S, int D, int kPart, bool kRotate>
__device__ __forceinline__ void append_window(const Append8Params& p, int64_t r0, Window& w) {
  constexpr int kLanes = D / 16;          // threads of a token of a head, 8 values of either half each
  constexpr int kTokens = 32 / kLanes;    // tokens of a pass
  constexpr int kPasses = kScaleTokens / kTokens;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = kPart == 0 ? p.heads : p.kv_heads;
  const __half* norm = kPart == 0 ? p.q_norm : p.k_norm;
  const T* src = static_cast<const T*>(p.qkv) + r0 * p.qkv_stride +
                 (int64_t)(kPart == 0 ? 0 : kPart == 1 ? p.heads : p.heads + p.kv_heads) * D;
  const int pairs = (heads + 1) / 2;  // a warp's task: two heads of a unit
  const int at = lane % kLanes, sub = lane / kLanes;

  uint4 raw[2][kPasses][2];
  auto load_rows = [&](int row, int n, int h0) {
    const T* x = src + (int64_t)row * p.qkv_stride + h0 * D + 8 * at;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int t = i * kTokens + sub;
        const bool mine = t < n && h0 + e < heads;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          raw[e][i][j] = mine ? ld_v4(x + t * p.qkv_stride + e * D + j * (D / 2)) : make_uint4(0, 0, 0, 0);
      }
  };
  auto load = [&](int task) {
    const int u = task / pairs;
    load_rows(w.unit_row[u], w.unit_rows[u], task % pairs * 2);
  };
  // A window of a long prompt is one unit as a rule: its rows are under way while
  // the units are found.
  const int likely = (int)min((int64_t)p.window, p.rows - r0);
  if (warp < pairs) load_rows(0, likely, warp * 2);
  if (warp == 0) find_units(p, kPart, r0, lane, w);
  __syncthreads();
  const int units = w.unit_count;
  if (units == 0) return;
  const int first_row = w.unit_row[0], rows = w.row_end - first_row;  // rows of all units
  const int tasks = units * pairs;
  // The first task stays in the registers.
  if (warp < tasks && !(warp < pairs && first_row == 0 && w.unit_rows[0] == likely)) load(warp);
  if constexpr (kRotate) {
    for (int i = tid; i < rows * (D / 2); i += kThreads) {
      const int r = i / (D / 2), d = i % (D / 2);
      turn((double)p.positions[r0 + first_row + r] * p.turns[d], kPart == 1, w.rot[0][r][d], w.rot[1][r][d]);
    }
    __syncthreads();
  }
  float2 weight[2][4];
  auto fetch_weight = [&](int h) {
    if constexpr (kPart < 2) {  // without a norm ones
      const uint32_t one = 0x3c003c00u;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        unpack4<__half>(norm ? ld_v4(norm + h * D + j * (D / 2) + 8 * at) : make_uint4(one, one, one, one), weight[j]);
    }
  };
  // A token's values but for the factor of its norm.
  auto values = [&](const uint4 (&in)[2], int row, float2 (&f)[2][4]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unpack4<T>(in[j], f[j]);
      if constexpr (kPart < 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[j][k] = mul2(f[j][k], weight[j][k]);
      }
    }
    if constexpr (kRotate) rotate_pairs(f, &w.rot[0][row][8 * at], &w.rot[1][row][8 * at]);
  };

  // First pass: the rows' sums of squares, where there is a norm.
  if (kPart < 2 && norm) {
    w.sums[warp][lane] = 0.f;
    __syncwarp();
    for (int task = warp; task < tasks; task += kWarps) {
      if (task != warp) load(task);
      const int u = task / pairs, n = w.unit_rows[u], local = w.unit_row[u] - first_row;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float2 f[4];
            unpack4<T>(raw[e][i][j], f);
#pragma unroll
            for (int k = 0; k < 4; ++k) sum = fma2(f[k], f[k], sum);
          }
        float all = sum.x + sum.y;
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
        const int t = i * kTokens + sub;
        if (at == 0 && t < n) w.sums[warp][local + t] += all;  // a token always has the same thread
      }
    }
    __syncthreads();
    if (tid < rows) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) sum += w.sums[i][tid];
      w.norm_of[tid] = rms_scale(sum, heads * D, p.eps);
    }
    __syncthreads();
  }

  // Second pass: out.
  for (int task = warp; task < tasks; task += kWarps) {
    if (task != warp || (kPart < 2 && norm && tasks > kWarps)) load(task);
    const int u = task / pairs, n = w.unit_rows[u], local = w.unit_row[u] - first_row;
    const int64_t page = w.unit_page[u];
    const int slot = w.unit_slot[u], earlier = slot & (kScaleTokens - 1);
    if (kPart != 0 && page < 0) continue;
    float factor[kPasses];  // of the thread's tokens
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
      factor[i] = kPart < 2 && norm ? w.norm_of[min(local + i * kTokens + sub, rows - 1)] : 1.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int h = task % pairs * 2 + e;
      if (h >= heads) break;
      fetch_weight(h);
      if constexpr (kPart == 0) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          if (i * kTokens >= n) break;
          const int t = i * kTokens + sub;
          float2 f[2][4];
          values(raw[e][i], min(local + t, rows - 1), f);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) f[j][k] = mul2(f[j][k], make_float2(factor[i], factor[i]));
          if (t < n) {
            T* out = static_cast<T*>(p.q_out) + ((r0 + w.unit_row[u] + t) * heads + h) * D + 8 * at;
#pragma unroll
            for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4*>(out + j * (D / 2)) = pack4<T>(f[j]);
          }
        }
      } else {
        uint8_t* block = p.codes[kPart - 1] + page * p.page_stride + (int64_t)(h * p.page_size + slot - earlier) * D;
        float* scale_at = p.scales[kPart - 1] + page * p.scale_stride + h * (p.page_size / kScaleTokens) +
                          slot / kScaleTokens;
        const float old = earlier ? *scale_at : 0.f;
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          if (i * kTokens >= n) break;
          const int t = i * kTokens + sub;
          float2 f[2][4];
          values(raw[e][i], min(local + t, rows - 1), f);
          if (t < n) most = max_nan(most, largest(f) * factor[i]);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
        const float scale = block_scale<S>(most, old);
        const Divisor over(scale);
        if (lane == 0) *scale_at = scale;
        if (earlier && scale > old) round_anew<S>(block, earlier * (D / 16), old, over, lane, 32);
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          if (i * kTokens >= n) break;
          const int t = i * kTokens + sub;
          float2 f[2][4];
          values(raw[e][i], min(local + t, rows - 1), f);
          if constexpr (kPart == 1) {
            const float2 by = make_float2(factor[i], factor[i]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int k = 0; k < 4; ++k) f[j][k] = mul2(f[j][k], by);
          }
          if (t < n) put_codes<S, D>(block + (earlier + t) * D + 8 * at, f, scale < INFINITY, over);
        }
      }
    }
  }
}

template <typename T, typename S, int D>
__global__ void __launch_bounds__(kThreads, 2) paged_append_8bit_kernel(const __grid_constant__ Append8Params p) {
  __shared__ __align__(16) Window w;
  const int part = blockIdx.x < p.windows ? 1 : blockIdx.x < 2 * p.windows ? 2 : 0;
  const int64_t r0 = (int64_t)(blockIdx.x % p.windows) * p.window;
  if (p.window == 1 && append_one<T, S, D>(p, part, r0, w)) return;
  if (part == 2)
    append_window<T, S, D, 2, false>(p, r0, w);
  else if (part == 1)
    p.rotate ? append_window<T, S, D, 1, true>(p, r0, w) : append_window<T, S, D, 1, false>(p, r0, w);
  else
    p.rotate ? append_window<T, S, D, 0, true>(p, r0, w) : append_window<T, S, D, 0, false>(p, r0, w);
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
