// The few-rows kernel over a cache of 8-bit codes.
#include "paged_split.cuh"

namespace tf {

tf_status launch_paged_split_8bit(const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  if (plan.split_blocks == 0) return TF_OK;
  SplitParams p;
  TF_TRY(split_params(a, &p));
  TF_TRY(make_code_map(&p.tm_k, a.kv.k, a.kv, p.box_rows));
  TF_TRY(make_code_map(&p.tm_v, a.kv.v, a.kv, p.box_rows));
  p.k_scales = a.scales.k;
  p.v_scales = a.scales.v;
  p.scale_stride = a.scales.page_stride;
  p.pages = a.kv.pages;
  const bool ints = a.kv.dtype == TF_DTYPE_I8;
  if (a.act == TF_DTYPE_F16)
    return ints ? launch_rows<__half, __half, I8>(p, plan, s) : launch_rows<__half, __half, E4M3>(p, plan, s);
  return ints ? launch_rows<__nv_bfloat16, __half, I8>(p, plan, s)
              : launch_rows<__nv_bfloat16, __half, E4M3>(p, plan, s);
}

}  // namespace tf
