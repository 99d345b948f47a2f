// Beam selection: what the pass over the logits leaves of each beam for the
// selection over all of them, and the launchers behind the C ABI.
#pragma once

#include <math.h>

#include "internal.h"

namespace tf {

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

// A row of logits: ln sum e^(x - m) and m; how many keys it has (0: none of its
// tokens can follow).
struct BeamRow {
  double log_sum;
  float m;
  int32_t n;
};

struct BeamArgs {
  const void* logits = nullptr;
  int64_t row_stride = 0;
  int64_t requests = 0;
  int beams = 0;
  int vocab = 0;
  int dtype = TF_DTYPE_F32;
  const float* scores = nullptr;
  const uint8_t* finished = nullptr;
  int64_t end = 0;
  int count = 0;
  float* score = nullptr;
  int32_t* parent = nullptr;
  int64_t* token = nullptr;
  char* workspace = nullptr;
  int each() const { return count < vocab ? count : vocab; }  // candidates of a beam
  __host__ __device__ BeamRow* rows() const { return reinterpret_cast<BeamRow*>(workspace); }
  __host__ __device__ uint64_t* keys() const {
    return reinterpret_cast<uint64_t*>(workspace + requests * beams * sizeof(BeamRow));
  }
  size_t workspace_bytes() const { return (size_t)requests * beams * (sizeof(BeamRow) + 8 * (size_t)each()); }
};
tf_status launch_beam_rows(const BeamArgs& a, cudaStream_t s);
tf_status launch_beam_select(const BeamArgs& a, cudaStream_t s);

}  // namespace tf
