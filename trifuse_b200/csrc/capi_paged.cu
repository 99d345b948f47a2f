// C ABI of the paged key/value cache, token log probabilities and beam selection:
// argument checks, all of them before any launch.
#include <exception>

#include "beams.h"
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

tf_status check_pages(const tf_paged_kv* kv, int heads, int act, int align) {
  TF_TRY(check_geometry(heads, kv->kv_heads, kv->head_dim, kv->page_size));
  if (!act_ok(act)) return set_error(TF_ERR_INVALID_ARGUMENT, "activation dtype must be f16 or bf16");
  if (kv->pages <= 0 || kv->pages > 2147483647LL ||
      kv->page_stride < (int64_t)kv->kv_heads * kv->page_size * kv->head_dim || kv->page_stride % align ||
      kv->page_stride >= (int64_t)1 << 38)
    return set_error(TF_ERR_SHAPE, "paged: pages %lld, page_stride %lld", (long long)kv->pages,
                     (long long)kv->page_stride);
  if (!kv->k || !kv->v || !aligned16(kv->k) || !aligned16(kv->v))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged: NULL or unaligned cache pointer");
  return TF_OK;
}

tf_status check_kv(const tf_paged_kv* kv, int heads, int act) {
  if (!kv) return set_error(TF_ERR_INVALID_ARGUMENT, "paged: cache descriptor is NULL");
  TF_TRY(check_geometry(heads, kv->kv_heads, kv->head_dim, kv->page_size));
  if (!act_ok(act)) return set_error(TF_ERR_INVALID_ARGUMENT, "activation dtype must be f16 or bf16");
  if (!(kv->dtype == act || (kv->dtype == TF_DTYPE_F16 && act == TF_DTYPE_BF16)))
    return set_error(TF_ERR_UNSUPPORTED, "paged: the cache has the activations' dtype, or f16 under bf16");
  return check_pages(kv, heads, act, 8);
}

// A cache of codes and its scales.
tf_status check_kv_8bit(const tf_paged_kv* kv, const tf_paged_scales* scales, int heads, int act) {
  if (!kv || !scales) return set_error(TF_ERR_INVALID_ARGUMENT, "paged: cache descriptor is NULL");
  if (kv->dtype != TF_DTYPE_I8 && kv->dtype != TF_DTYPE_E4M3)
    return set_error(TF_ERR_UNSUPPORTED, "paged: an 8-bit cache holds int8 or e4m3 codes");
  TF_TRY(check_pages(kv, heads, act, 16));
  if (kv->page_size < kScaleTokens)
    return set_error(TF_ERR_UNSUPPORTED, "paged: page_size %d below the %d tokens of a scale", kv->page_size,
                     kScaleTokens);
  if (scales->page_stride < (int64_t)kv->kv_heads * (kv->page_size / kScaleTokens) ||
      scales->page_stride >= (int64_t)1 << 38)
    return set_error(TF_ERR_SHAPE, "paged: the scales' page_stride %lld", (long long)scales->page_stride);
  if (!scales->k || !scales->v || (reinterpret_cast<uintptr_t>(scales->k) & 3u) ||
      (reinterpret_cast<uintptr_t>(scales->v) & 3u))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged: NULL or unaligned scales");
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

tf_status check_beams(int64_t requests, int beams, int vocab, int count) {
  if (requests < 0 || requests > 1 << 24 || beams < 1 || beams > TF_MAX_BEAMS || vocab < 1 || vocab > 1 << 30)
    return set_error(TF_ERR_SHAPE, "beam_select: requests %lld, beams %d (up to %d), vocab %d", (long long)requests,
                     beams, TF_MAX_BEAMS, vocab);
  if (count < 1 || count > TF_MAX_TOP)
    return set_error(TF_ERR_INVALID_ARGUMENT, "beam_select: count %d outside [1, %d]", count, TF_MAX_TOP);
  return TF_OK;
}

AppendArgs append_args(const void* qkv, int64_t qkv_stride, int64_t rows, int heads, int act, const void* q_norm,
                       const void* k_norm, float eps, float rope_theta, const int32_t* positions,
                       const int32_t* requests, const tf_page_table* table, const tf_paged_kv* kv, void* q_out) {
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
  return a;
}

tf_status check_append(const AppendArgs& a) {
  if (a.rows < 0 || a.qkv_stride < ((int64_t)a.heads + 2 * a.kv.kv_heads) * a.kv.head_dim || a.qkv_stride % 8)
    return set_error(TF_ERR_SHAPE, "paged_append: rows %lld, stride %lld", (long long)a.rows,
                     (long long)a.qkv_stride);
  if (!a.q_norm != !a.k_norm)
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_append: q_norm and k_norm go together");
  if ((a.q_norm && !(a.eps > 0)) || !(a.theta == 0.f || a.theta > 1))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_append: eps must be positive, rope_theta above 1 (or 0)");
  if (a.rows == 0) return TF_OK;
  if (!a.qkv || !a.positions || !a.requests || !a.q_out || !aligned16(a.qkv) || !aligned16(a.q_out) ||
      !aligned16(a.q_norm) || !aligned16(a.k_norm))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_append: NULL or unaligned pointer");
  return TF_OK;
}

PagedArgs attention_args(const void* q, int64_t q_stride, const tf_page_table* table, const tf_paged_kv* kv,
                         const tf_paged_plan* plan, void* plan_table, float scale, int act, void* out,
                         void* workspace) {
  PagedArgs a;
  a.q = q;
  a.q_stride = q_stride;
  if (table) a.table = *table;
  a.kv = *kv;
  a.plan = plan;
  a.plan_table = static_cast<char*>(plan_table);
  a.scale = scale;
  a.act = act;
  a.out = out;
  a.workspace = static_cast<char*>(workspace);
  return a;
}

tf_status check_attention(const PagedArgs& a, const tf_page_table* table, size_t workspace_bytes) {
  const tf_paged_plan* plan = a.plan;
  TF_TRY(check_table(table));
  if (a.kv.kv_heads != plan->kv_heads || a.kv.head_dim != plan->head_dim || a.kv.page_size != plan->page_size)
    return set_error(TF_ERR_SHAPE, "paged_attention: the plan was made for another cache geometry");
  if (table->requests < plan->requests || table->columns < plan->columns)
    return set_error(TF_ERR_SHAPE, "paged_attention: page table %d x %d, the plan needs %d x %d", table->requests,
                     table->columns, plan->requests, plan->columns);
  // The kernels work with scale * log2(e) in fp32.
  if (!(a.scale > 0) || !(a.scale <= 2.3e38f))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: scale must be positive and below 2.3e38");
  if (a.q_stride < (int64_t)plan->heads * plan->head_dim || a.q_stride % 8)
    return set_error(TF_ERR_SHAPE, "paged_attention: q stride %lld", (long long)a.q_stride);
  if (plan->rows == 0) return TF_OK;
  if (!a.q || !a.out || !a.plan_table || !aligned16(a.q) || (reinterpret_cast<uintptr_t>(a.out) & 31u) ||
      !aligned16(a.plan_table))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: NULL or unaligned pointer");
  if (workspace_bytes < plan->workspace_bytes ||
      (plan->workspace_bytes && (!a.workspace || !aligned16(a.workspace))))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: workspace too small or unaligned");
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
  const AppendArgs a = append_args(qkv, qkv_stride, rows, heads, act, q_norm, k_norm, eps, rope_theta, positions,
                                   requests, table, kv, q_out);
  TF_TRY(check_append(a));
  return rows == 0 ? TF_OK : launch_paged_append(a, st(stream));
}

int tf_paged_append_8bit(const void* qkv, int64_t qkv_stride, int64_t rows, int32_t heads, int act,
                         const void* q_norm, const void* k_norm, float eps, float rope_theta,
                         const int32_t* positions, const int32_t* requests, const tf_page_table* table,
                         const tf_paged_kv* kv, const tf_paged_scales* scales, void* q_out, void* stream) {
  TF_TRY(check_kv_8bit(kv, scales, heads, act));
  TF_TRY(check_table(table));
  const AppendArgs a = append_args(qkv, qkv_stride, rows, heads, act, q_norm, k_norm, eps, rope_theta, positions,
                                   requests, table, kv, q_out);
  TF_TRY(check_append(a));
  return rows == 0 ? TF_OK : launch_paged_append_8bit(a, *scales, st(stream));
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
  const PagedArgs a = attention_args(q, q_stride, table, kv, plan, plan_table, scale, act, out, workspace);
  TF_TRY(check_attention(a, table, workspace_bytes));
  if (plan->rows == 0) return TF_OK;
  TF_TRY(launch_paged_split(a, st(stream)));
  return launch_paged_tile(a, st(stream));
}

int tf_paged_attention_8bit(const void* q, int64_t q_stride, const tf_page_table* table, const tf_paged_kv* kv,
                            const tf_paged_scales* scales, const tf_paged_plan* plan, void* plan_table, float scale,
                            int act, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (!plan) return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: NULL plan");
  TF_TRY(check_kv_8bit(kv, scales, plan->heads, act));
  PagedArgs a = attention_args(q, q_stride, table, kv, plan, plan_table, scale, act, out, workspace);
  a.scales = *scales;
  TF_TRY(check_attention(a, table, workspace_bytes));
  if (plan->rows == 0) return TF_OK;
  if (plan->widened_bytes &&
      (!a.workspace || !aligned16(a.workspace) || workspace_bytes < plan->workspace_bytes + plan->widened_bytes))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_attention: workspace too small for an 8-bit cache");
  TF_TRY(launch_paged_widen(a, st(stream)));
  TF_TRY(launch_paged_split_8bit(a, st(stream)));
  return launch_paged_tile_8bit(a, st(stream));
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

int tf_paged_copy(const tf_copy_array* arrays, int32_t count, int32_t layers, int64_t pages, const int32_t* src,
                  const int32_t* dst, int64_t pairs, void* stream) {
  if (count < 0 || count > TF_MAX_COPY_ARRAYS || (count && !arrays))
    return set_error(TF_ERR_INVALID_ARGUMENT, "paged_copy: %d arrays (up to %d)", count, TF_MAX_COPY_ARRAYS);
  if (layers < 0 || pages < 0 || pages > 2147483647LL || pairs < 0 || pairs > 1 << 30)
    return set_error(TF_ERR_SHAPE, "paged_copy: layers %d, pages %lld, pairs %lld", layers, (long long)pages,
                     (long long)pairs);
  if (pairs && (!src || !dst)) return set_error(TF_ERR_INVALID_ARGUMENT, "paged_copy: NULL pairs");
  for (int i = 0; i < count; ++i) {
    const tf_copy_array& a = arrays[i];
    if (a.page_bytes < 0 || a.page_bytes > (int64_t)1 << 32 || (pages > 1 && a.page_stride < a.page_bytes) ||
        a.page_stride < 0 || a.page_stride >= (int64_t)1 << 40 || a.layer_stride < 0 ||
        a.layer_stride >= (int64_t)1 << 50)
      return set_error(TF_ERR_SHAPE, "paged_copy: array %d has pages of %lld bytes, %lld apart", i,
                       (long long)a.page_bytes, (long long)a.page_stride);
    if (!a.base && a.page_bytes && layers && pairs)
      return set_error(TF_ERR_INVALID_ARGUMENT, "paged_copy: array %d is NULL", i);
  }
  return launch_paged_copy(arrays, count, layers, pages, src, dst, pairs, st(stream));
}

int tf_beam_select_workspace_size(int64_t requests, int32_t beams, int32_t vocab, int32_t count, size_t* bytes) {
  if (!bytes) return set_error(TF_ERR_INVALID_ARGUMENT, "beam_select: NULL size");
  TF_TRY(check_beams(requests, beams, vocab, count));
  BeamArgs a;
  a.requests = requests;
  a.beams = beams;
  a.vocab = vocab;
  a.count = count;
  *bytes = a.workspace_bytes();
  return TF_OK;
}

int tf_beam_select(const void* logits, int64_t row_stride, int64_t requests, int32_t beams, int32_t vocab, int dtype,
                   const float* scores, const uint8_t* finished, int64_t end, int32_t count, float* score,
                   int32_t* parent, int64_t* token, void* workspace, size_t workspace_bytes, void* stream) {
  if (!act_ok(dtype) && dtype != TF_DTYPE_F32)
    return set_error(TF_ERR_INVALID_ARGUMENT, "beam_select: logits must be f32, f16 or bf16");
  TF_TRY(check_beams(requests, beams, vocab, count));
  if (row_stride < vocab) return set_error(TF_ERR_SHAPE, "beam_select: rows %lld apart", (long long)row_stride);
  if (requests == 0) return TF_OK;
  const size_t element = dtype == TF_DTYPE_F32 ? 4 : 2;
  if (!logits || !scores || !score || !parent || !token || reinterpret_cast<uintptr_t>(logits) % element)
    return set_error(TF_ERR_INVALID_ARGUMENT, "beam_select: NULL or unaligned pointer");
  BeamArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.requests = requests;
  a.beams = beams;
  a.vocab = vocab;
  a.dtype = dtype;
  a.scores = scores;
  a.finished = finished;
  a.end = end;
  a.count = count;
  a.score = score;
  a.parent = parent;
  a.token = token;
  a.workspace = static_cast<char*>(workspace);
  if (!workspace || !aligned16(workspace) || workspace_bytes < a.workspace_bytes())
    return set_error(TF_ERR_INVALID_ARGUMENT, "beam_select: workspace too small or unaligned");
  return launch_beam_select(a, st(stream));
}

}  // extern "C"
