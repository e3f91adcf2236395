// capi_paged.cu -- C ABI of the paged-cache operators (declared in
// include/qwen_b200.h): argument checks, then one launcher call each.
#include <cstdint>

#include "paged.h"
#include "paged_checks.h"
#include "qwen_common.cuh"
#include "qwen_internal.h"

using namespace qwen;

namespace {

int check_tiles(const char* op, const qwen_paged_kv* kv, uint32_t n_heads, uint32_t n_list) {
  if (paged_decode_fits(*kv, (int)n_heads, (int)n_list)) return QWEN_OK;
  return set_error(QWEN_ERR_INVALID_ARGUMENT,
                   "%s: %u sequences of %u kv heads and up to %llu positions are more than one call takes", op,
                   kv->n_seq, kv->n_kv_heads,
                   (unsigned long long)(n_list ? n_list : kv->max_pages) * kv->page_size);
}
int check_prefix_len(const char* op, uint32_t prefix_len) {
  if (prefix_len <= kMaxPositions) return QWEN_OK;
  return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: prefix_len=%u", op, prefix_len);
}
int check_n_select(const char* op, uint32_t n_select) {
  if (n_select != 0 && n_select <= (1u << 20)) return QWEN_OK;
  return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_select=%u", op, n_select);
}
// Whether an attention call (n_list listed pages, 0 without a list) can need a workspace:
// not without sequences, nor where its sizes will be refused.
bool attention_runs(const char* op, const qwen_paged_kv* kv, uint32_t n_heads, uint32_t n_list) {
  int shift;
  return kv && kv->n_seq != 0 && check_sizes(op, kv, n_heads, &shift) == QWEN_OK &&
         check_tiles(op, kv, n_heads, n_list) == QWEN_OK;
}

int check_kv(const char* op, const qwen_paged_kv* kv, uint32_t n_heads, int* page_shift) {
  if (!kv) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null kv", op);
  if (!kv->k || !kv->v || (!kv->page_table && kv->n_seq))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null cache buffer", op);
  QWEN_TRY(check_sizes(op, kv, n_heads, page_shift));
  const int64_t strides[3] = {kv->page_stride, kv->pos_stride, kv->head_stride};
  for (int64_t x : strides)
    if (x <= 0 || x % 8 != 0 || x >= (1ll << 38))
      return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: cache stride %lld must be a positive multiple of 8",
                       op, (long long)x);
  if (!aligned16(kv->k) || !aligned16(kv->v) || !aligned16(kv->bounds))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: cache buffers must be 16-byte aligned", op);
  return QWEN_OK;
}

int attention(const char* op, PagedAttnArgs& a, const qwen_paged_kv* kv, const uint16_t* q,
              int64_t q_stride, uint16_t* out, int64_t out_stride, float* lse, uint32_t n_heads,
              const uint32_t* seq_len, float scale, void* workspace, size_t workspace_bytes,
              size_t need, void* stream) {
  QWEN_TRY(check_kv(op, kv, n_heads, &a.page_shift));
  if (kv->n_seq == 0) return QWEN_OK;
  QWEN_TRY(check_rows(op, "q", q, q_stride, n_heads * kv->head_dim));
  QWEN_TRY(check_rows(op, "out", out, out_stride, n_heads * kv->head_dim));
  if (!seq_len) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null seq_len", op);
  QWEN_TRY(check_workspace(op, workspace, workspace_bytes, need));
  QWEN_TRY(check_tiles(op, kv, n_heads, (uint32_t)a.n_list));
  a.kv = *kv;
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.lse = lse;
  a.n_heads = (int)n_heads;
  a.seq_len = seq_len;
  a.scale = scale;
  a.workspace = workspace;
  QWEN_TRY(ops_status_word(&a.err));
  return finish(op, a.prefix_len ? launch_paged_prefix(a, static_cast<cudaStream_t>(stream))
                                 : launch_paged_decode(a, static_cast<cudaStream_t>(stream)));
}

}  // namespace

extern "C" {

int qwen_rope_append_paged(const qwen_paged_kv* kv, const uint16_t* q, int64_t q_stride,
                           const uint16_t* k, int64_t k_stride, const uint16_t* v,
                           int64_t v_stride, uint16_t* q_out, int64_t q_out_stride,
                           uint32_t n_heads, uint32_t n_tokens, const uint32_t* seq_len,
                           const int32_t* cu_tokens, const float* inv_freq, uint32_t rot_dim,
                           int interleaved, void* stream) {
  const char* op = "rope_append_paged";
  PagedAppendArgs a{};
  QWEN_TRY(check_kv(op, kv, n_heads, &a.page_shift));
  if (!cu_tokens && n_tokens != kv->n_seq)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_tokens=%u for %u sequences without cu_tokens", op,
                     n_tokens, kv->n_seq);
  if (kv->n_seq == 0 || n_tokens == 0) return QWEN_OK;
  QWEN_TRY(check_rows(op, "q", q, q_stride, n_heads * kv->head_dim));
  QWEN_TRY(check_rows(op, "q_out", q_out, q_out_stride, n_heads * kv->head_dim));
  QWEN_TRY(check_rows(op, "k", k, k_stride, kv->n_kv_heads * kv->head_dim));
  QWEN_TRY(check_rows(op, "v", v, v_stride, kv->n_kv_heads * kv->head_dim));
  if (!seq_len || !inv_freq)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null seq_len or inv_freq", op);
  if (rot_dim == 0 || rot_dim % 16 != 0 || rot_dim > kv->head_dim)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: rot_dim=%u must be a multiple of 16, at most %u", op,
                     rot_dim, kv->head_dim);
  if (n_tokens > (1u << 24)) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_tokens=%u", op, n_tokens);
  a.kv = *kv;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out_stride = q_out_stride;
  a.n_heads = (int)n_heads;
  a.n_tokens = (int)n_tokens;
  a.seq_len = seq_len;
  a.cu_tokens = cu_tokens;
  a.inv_freq = inv_freq;
  a.rot_dim = (int)rot_dim;
  a.interleaved = interleaved ? 1 : 0;
  QWEN_TRY(ops_status_word(&a.err));
  return finish(op, launch_rope_append(a, static_cast<cudaStream_t>(stream)));
}

size_t qwen_attention_paged_workspace(const qwen_paged_kv* kv, uint32_t n_heads) {
  return attention_runs("attention_paged", kv, n_heads, 0) ? paged_decode_workspace(*kv, (int)n_heads) : 0;
}

int qwen_attention_paged(const qwen_paged_kv* kv, const uint16_t* q, int64_t q_stride,
                         uint16_t* out, int64_t out_stride, float* lse, uint32_t n_heads,
                         const uint32_t* seq_len, float scale, void* workspace,
                         size_t workspace_bytes, void* stream) {
  PagedAttnArgs a{};
  return attention("attention_paged", a, kv, q, q_stride, out, out_stride, lse, n_heads, seq_len, scale,
                   workspace, workspace_bytes, qwen_attention_paged_workspace(kv, n_heads), stream);
}

size_t qwen_attention_prefix_paged_workspace(const qwen_paged_kv* kv, uint32_t n_heads, uint32_t prefix_len) {
  const char* op = "attention_prefix_paged";
  return attention_runs(op, kv, n_heads, 0) && check_prefix_len(op, prefix_len) == QWEN_OK
             ? paged_prefix_workspace(*kv, (int)n_heads, prefix_len)
             : 0;
}

int qwen_attention_prefix_paged(const qwen_paged_kv* kv, const uint16_t* q, int64_t q_stride,
                                uint16_t* out, int64_t out_stride, float* lse, uint32_t n_heads,
                                const uint32_t* seq_len, const int32_t* prefix_pages,
                                uint32_t prefix_len, float scale, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* op = "attention_prefix_paged";
  QWEN_TRY(check_prefix_len(op, prefix_len));
  if (prefix_len && !prefix_pages)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null prefix_pages", op);
  PagedAttnArgs a{};
  a.prefix_pages = prefix_pages;
  a.prefix_len = prefix_len;
  return attention(op, a, kv, q, q_stride, out, out_stride, lse, n_heads, seq_len, scale, workspace,
                   workspace_bytes, qwen_attention_prefix_paged_workspace(kv, n_heads, prefix_len), stream);
}

size_t qwen_select_pages_workspace(const qwen_paged_kv* kv) {
  int shift;   // (query heads: not known here, any that pass)
  return kv && kv->n_seq != 0 && check_sizes("select_pages", kv, kv->n_kv_heads, &shift) == QWEN_OK
             ? (size_t)kv->n_seq * kv->n_kv_heads * kv->max_pages * sizeof(double)
             : 0;
}

int qwen_select_pages(const qwen_paged_kv* kv, const uint16_t* q, int64_t q_stride,
                      uint32_t n_heads, const uint32_t* seq_len, uint32_t n_select,
                      uint32_t n_first, uint32_t n_last, int32_t* pages, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const char* op = "select_pages";
  PagedSelectArgs a{};
  QWEN_TRY(check_kv(op, kv, n_heads, &a.page_shift));
  if (kv->n_seq == 0) return QWEN_OK;
  QWEN_TRY(check_rows(op, "q", q, q_stride, n_heads * kv->head_dim));
  if (!kv->bounds) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: the cache keeps no bounds", op);
  if (!seq_len || !pages) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null seq_len or pages", op);
  QWEN_TRY(check_n_select(op, n_select));
  if ((uint64_t)n_first + n_last > n_select)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_select=%u n_first=%u n_last=%u", op, n_select,
                     n_first, n_last);
  QWEN_TRY(check_workspace(op, workspace, workspace_bytes, qwen_select_pages_workspace(kv)));
  a.kv = *kv;
  a.q = q;
  a.q_stride = q_stride;
  a.n_heads = (int)n_heads;
  a.seq_len = seq_len;
  a.n_select = (int)n_select;
  a.n_first = (int)n_first;
  a.n_last = (int)n_last;
  a.pages = pages;
  a.scores = static_cast<double*>(workspace);
  QWEN_TRY(ops_status_word(&a.err));
  return finish(op, launch_select_pages(a, static_cast<cudaStream_t>(stream)));
}

size_t qwen_attention_sparse_paged_workspace(const qwen_paged_kv* kv, uint32_t n_heads, uint32_t n_select) {
  const char* op = "attention_sparse_paged";
  return check_n_select(op, n_select) == QWEN_OK && attention_runs(op, kv, n_heads, n_select)
             ? paged_decode_workspace(*kv, (int)n_heads)
             : 0;
}

int qwen_attention_sparse_paged(const qwen_paged_kv* kv, const int32_t* pages, uint32_t n_select,
                                const uint16_t* q, int64_t q_stride, uint16_t* out,
                                int64_t out_stride, float* lse, uint32_t n_heads,
                                const uint32_t* seq_len, float scale, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* op = "attention_sparse_paged";
  if (!pages && kv && kv->n_seq) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null pages", op);
  QWEN_TRY(check_n_select(op, n_select));
  PagedAttnArgs a{};
  a.list = pages;
  a.n_list = (int)n_select;
  return attention(op, a, kv, q, q_stride, out, out_stride, lse, n_heads, seq_len, scale, workspace,
                   workspace_bytes, qwen_attention_sparse_paged_workspace(kv, n_heads, n_select), stream);
}

}  // extern "C"
