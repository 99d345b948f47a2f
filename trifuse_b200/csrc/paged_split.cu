// The few-rows kernel over a 16-bit cache, and the tensor maps of pages.
#include "paged_split.cuh"

namespace tf {

namespace {

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

tf_status make_code_map(void* map, const void* base, const tf_paged_kv& kv, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.kv_heads * kv.page_size, (cuuint64_t)kv.pages};
  const cuuint64_t strides[2] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page_stride};
  const cuuint32_t box[3] = {(cuuint32_t)kv.head_dim, (cuuint32_t)box_rows, 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  const EncodeFn encode = encode_fn();
  if (!encode) return set_error(TF_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const CUresult r = encode(static_cast<CUtensorMap*>(map), CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base),
                            dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            kv.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(TF_ERR_CUDA, "paged attention: tensor map (%d)", (int)r);
  return TF_OK;
}

tf_status launch_paged_split(const PagedArgs& a, cudaStream_t s) {
  const tf_paged_plan& plan = *a.plan;
  if (plan.split_blocks == 0) return TF_OK;
  SplitParams p;
  TF_TRY(split_params(a, &p));
  TF_TRY(make_page_map(&p.tm_k, a.kv.k, a.kv, p.box_rows, a.kv.head_dim));
  TF_TRY(make_page_map(&p.tm_v, a.kv.v, a.kv, p.box_rows, a.kv.head_dim));
  if (a.act == TF_DTYPE_F16) return launch_rows<__half, __half, __half>(p, plan, s);
  if (a.kv.dtype == TF_DTYPE_F16) return launch_rows<__nv_bfloat16, __half, __half>(p, plan, s);
  return launch_rows<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(p, plan, s);
}

}  // namespace tf
