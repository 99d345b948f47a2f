// C ABI of the paged key/value cache and of token log probabilities: argument
// checks, all of them before any launch.
#include <exception>

#include "internal.h"
#include "paged.h"

using namespace tf;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

tf_status check_geometry(int heads, int kv_heads, int head_dim, int page_size) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    return set_error(TF_ERR_SHAPE, "paged: heads %d must be a positive multiple of kv_heads %d", heads, kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return set_error(TF_ERR_UNSUPPORTED, "paged: head_dim %d (64 or 128)", head_dim);
  if ((int64_t)heads * head_dim > 16384)
    return set_error(TF_ERR_UNSUPPORTED, "paged: heads * head_dim %lld above 16384", (long long)heads * head_dim);
  if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)))
    return set_error(TF_ERR_UNSUPPORTED, "paged: page_size %d (a power of two from 8 to 256)", page_size);
  return TF_OK;
}

tf_status check_kv(const tf_paged_kv* kv, int heads, int act) {
  if (!kv) return set_error(TF_ERR_INVALID_ARGUMENT, "paged: cache descriptor is NULL");
  TF_TRY(check_geometry(heads, kv->kv_heads, kv->head_dim, kv->page_size));
  if (!act_ok(act)) return set_error(TF_ERR_INVALID_ARGUMENT, "activation dtype must be f16 or bf16");
  if (!(kv->dtype == act || (kv->dtype == TF_DTYPE_F16 && act == TF_DTYPE_BF16)))
    return set_error(TF_ERR_UNSUPPORTED, "paged: the cache has the activations' dtype, or f16 under bf16");
  if (kv->pages <= 0 || kv->pages > 2147483647LL ||
      kv->page_stride < (int64_t)kv->kv_heads * kv->page_size * kv->head_dim || kv->page_stride % 8 ||
      kv->page_stride >= (int64_t)1 << 38)
    return set_error(TF_ERR_SHAPE, "paged: pages %lld, page_stride %lld", (long long)kv->pages,
                     (long long)kv->page_stride);
  if (!kv->k || !kv->v || !aligned16(kv->k) || !aligned16(kv->v))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged: NULL or unaligned cache pointer");
  return TF_OK;
}

tf_status check_table(const tf_page_table* t) {
  if (!t) return set_error(TF_ERR_INVALID_ARGUMENT, "paged: page table is NULL");
  if (t->requests < 0 || t->columns < 0 || t->stride < t->columns)
    return set_error(TF_ERR_SHAPE, "paged: page table %d x %d, stride %lld", t->requests, t->columns,
                     (long long)t->stride);
  if (!t->ids && t->requests && t->columns)
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged: page table is NULL");
  return TF_OK;
}

tf_status check_lengths(const int32_t* new_lengths, const int32_t* kv_lengths, int requests, int group,
                        int64_t* rows) {
  if (requests < 0 || (requests && (!new_lengths || !kv_lengths)))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged plan: bad lengths");
  *rows = 0;
  for (int r = 0; r < requests; ++r) {
    if (new_lengths[r] < 0 || kv_lengths[r] < 0)
      return set_error(TF_ERR_SHAPE, "paged plan: request %d has a negative length", r);
    if ((int64_t)new_lengths[r] * group > 1 << 30 || kv_lengths[r] > 1 << 30)
      return set_error(TF_ERR_UNSUPPORTED, "paged plan: request %d is too long", r);
    *rows += new_lengths[r];
  }
  if (*rows > 1 << 30) return set_error(TF_ERR_UNSUPPORTED, "paged plan: %lld rows", (long long)*rows);
  return TF_OK;
}

cudaStream_t st(void* s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

int tf_paged_append(const void* qkv, int64_t qkv_stride, int64_t rows, int32_t heads, int act, const void* q_norm,
                    const void* k_norm, float eps, float rope_theta, const int32_t* positions,
                    const int32_t* requests, const tf_page_table* table, const tf_paged_kv* kv, void* q_out,
                    void* stream) {
  TF_TRY(check_kv(kv, heads, act));
  TF_TRY(check_table(table));
  if (rows < 0 || qkv_stride < ((int64_t)heads + 2 * kv->kv_heads) * kv->head_dim || qkv_stride % 8)
    return set_error(TF_ERR_SHAPE, "paged_append: rows %lld, stride %lld", (long long)rows, (long long)qkv_stride);
  if (!q_norm != !k_norm)
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_append: q_norm and k_norm go together");
  if ((q_norm && !(eps > 0)) || !(rope_theta == 0.f || rope_theta > 1))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_append: eps must be positive, rope_theta above 1 (or 0)");
  if (rows == 0) return TF_OK;
  if (!qkv || !positions || !requests || !q_out || !aligned16(qkv) || !aligned16(q_out) || !aligned16(q_norm) ||
      !aligned16(k_norm))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_append: NULL or unaligned pointer");
  AppendArgs a;
  a.qkv = qkv;
  a.qkv_stride = qkv_stride;
  a.rows = rows;
  a.heads = heads;
  a.act = act;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.theta = rope_theta;
  a.positions = positions;
  a.requests = requests;
  a.table = *table;
  a.kv = *kv;
  a.q_out = q_out;
  return launch_paged_append(a, st(stream));
}

int tf_paged_plan_make(const int32_t* new_lengths, const int32_t* kv_lengths, int32_t requests, int32_t heads,
                       int32_t kv_heads, int32_t head_dim, int32_t page_size, tf_paged_plan* plan, void* table,
                       size_t table_capacity) {
  if (!plan || (!table && table_capacity)) return set_error(TF_ERR_INVALID_ARGUMENT, "paged plan: NULL plan or table");
  TF_TRY(check_geometry(heads, kv_heads, head_dim, page_size));
  tf_paged_plan p{};
  TF_TRY(check_lengths(new_lengths, kv_lengths, requests, heads / kv_heads, &p.rows));
  p.requests = requests;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.head_dim = head_dim;
  p.page_size = page_size;
  for (int r = 0; r < requests; ++r) {
    const int32_t pages = new_lengths[r] ? (kv_lengths[r] + page_size - 1) / page_size : 0;
    if (pages > p.columns) p.columns = pages;
  }
  try {
    const tf_status s = paged_plan_make(new_lengths, kv_lengths, &p, static_cast<char*>(table), table_capacity);
    *plan = p;
    return s;
  } catch (const std::exception&) {  // bad_alloc, or a length past what a vector holds
    return set_error(TF_ERR_OUT_OF_MEMORY, "paged plan: out of host memory");
  }
}

int tf_paged_attention(const void* q, int64_t q_stride, const tf_page_table* table, const tf_paged_kv* kv,
                       const tf_paged_plan* plan, void* plan_table, float scale, int act, void* out, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (!plan) return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: NULL plan");
  TF_TRY(check_kv(kv, plan->heads, act));
  TF_TRY(check_table(table));
  if (kv->kv_heads != plan->kv_heads || kv->head_dim != plan->head_dim || kv->page_size != plan->page_size)
    return set_error(TF_ERR_SHAPE, "paged_attention: the plan was made for another cache geometry");
  if (table->requests < plan->requests || table->columns < plan->columns)
    return set_error(TF_ERR_SHAPE, "paged_attention: page table %d x %d, the plan needs %d x %d", table->requests,
                     table->columns, plan->requests, plan->columns);
  // The kernels work with scale * log2(e) in fp32.
  if (!(scale > 0) || !(scale <= 2.3e38f))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: scale must be positive and below 2.3e38");
  if (q_stride < (int64_t)plan->heads * plan->head_dim || q_stride % 8)
    return set_error(TF_ERR_SHAPE, "paged_attention: q stride %lld", (long long)q_stride);
  if (plan->rows == 0) return TF_OK;
  if (!q || !out || !plan_table || !aligned16(q) || (reinterpret_cast<uintptr_t>(out) & 31u) || !aligned16(plan_table))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: NULL or unaligned pointer");
  if (workspace_bytes < plan->workspace_bytes ||
      (plan->workspace_bytes && (!workspace || !aligned16(workspace))))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: workspace too small or unaligned");
  PagedArgs a;
  a.q = q;
  a.q_stride = q_stride;
  a.table = *table;
  a.kv = *kv;
  a.plan = plan;
  a.plan_table = static_cast<char*>(plan_table);
  a.scale = scale;
  a.act = act;
  a.out = out;
  a.workspace = static_cast<char*>(workspace);
  TF_TRY(launch_paged_split(a, st(stream)));
  return launch_paged_tile(a, st(stream));
}

int tf_token_logprobs(const void* logits, int64_t row_stride, int64_t rows, int32_t vocab, int dtype,
                      const int64_t* tokens, int32_t top, float* logprob, float* entropy, int32_t* rank,
                      float* top_logprob, int64_t* top_token, void* stream) {
  if (!act_ok(dtype) && dtype != TF_DTYPE_F32)
    return set_error(TF_ERR_INVALID_ARGUMENT, "token_logprobs: logits must be f32, f16 or bf16");
  if (rows < 0 || vocab < 1 || vocab > 1 << 30 || row_stride < vocab)
    return set_error(TF_ERR_SHAPE, "token_logprobs: rows %lld, vocab %d, stride %lld", (long long)rows, vocab,
                     (long long)row_stride);
  if (top < 0 || top > TF_MAX_TOP || top > vocab)
    return set_error(TF_ERR_INVALID_ARGUMENT, "token_logprobs: top %d outside [0, min(%d, vocab)]", top, TF_MAX_TOP);
  if (rows == 0) return TF_OK;
  const size_t element = dtype == TF_DTYPE_F32 ? 4 : 2;
  if (!logits || !tokens || !logprob || !entropy || !rank || (top && (!top_logprob || !top_token)) ||
      reinterpret_cast<uintptr_t>(logits) % element)
    return set_error(TF_ERR_INVALID_ARGUMENT, "token_logprobs: NULL or unaligned pointer");
  return launch_token_logprobs(logits, row_stride, rows, vocab, dtype, tokens, top, logprob, entropy, rank,
                               top_logprob, top_token, st(stream));
}

}  // extern "C"
