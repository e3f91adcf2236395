// capi_paged_q4.cu -- C ABI of the operators over a 4-bit paged cache (declared in
// include/qwen_b200.h): argument checks, then one launcher call each.
#include <cstdint>

#include "paged_checks.h"
#include "paged_q4.h"
#include "qwen_internal.h"

using namespace qwen;

namespace {

// Type and sizes as the 16-bit operators check them.
int check_q4_sizes(const char* op, const qwen_paged_kv_q4* kv, uint32_t n_heads, int* page_shift) {
  qwen_paged_kv s{};
  s.n_pages = kv->n_pages;
  s.page_size = kv->page_size;
  s.n_kv_heads = kv->n_kv_heads;
  s.head_dim = kv->head_dim;
  s.n_seq = kv->n_seq;
  s.max_pages = kv->max_pages;
  s.table_stride = kv->table_stride;
  s.dtype = kv->dtype;
  return check_sizes(op, &s, n_heads, page_shift);
}

int check_q4(const char* op, const qwen_paged_kv_q4* kv, uint32_t n_heads, int* page_shift) {
  if (!kv) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null kv", op);
  if (!kv->pool || (!kv->page_table && kv->n_seq))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null cache buffer", op);
  QWEN_TRY(check_q4_sizes(op, kv, n_heads, page_shift));
  for (int64_t x : {kv->page_stride, kv->head_stride})
    if (x <= 0 || x % 16 != 0 || x >= (1ll << 39))
      return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: cache stride %lld must be a positive multiple of 16", op,
                       (long long)x);
  if (!aligned16(kv->pool) || !aligned16(kv->weights) || !aligned16(kv->positions))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: cache buffers must be 16-byte aligned", op);
  return QWEN_OK;
}

int check_q4_tiles(const char* op, const qwen_paged_kv_q4* kv, uint32_t n_heads) {
  if (attention_q4_fits(*kv, (int)n_heads)) return QWEN_OK;
  return set_error(QWEN_ERR_INVALID_ARGUMENT,
                   "%s: %u sequences of %u kv heads and up to %llu positions are more than one call takes", op,
                   kv->n_seq, kv->n_kv_heads, (unsigned long long)kv->max_pages * kv->page_size);
}
int check_keep(const char* op, uint32_t n_keep) {
  if (n_keep != 0 && n_keep <= kMaxPositions) return QWEN_OK;
  return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_keep=%u", op, n_keep);
}

}  // namespace

extern "C" {

int qwen_rope_append_paged_q4(const qwen_paged_kv_q4* kv, const uint16_t* q, int64_t q_stride,
                              const uint16_t* k, int64_t k_stride, const uint16_t* v,
                              int64_t v_stride, uint16_t* q_out, int64_t q_out_stride,
                              uint32_t n_heads, uint32_t n_tokens, const uint32_t* seq_len,
                              const int32_t* cu_tokens, const int32_t* positions,
                              int64_t position_stride, uint32_t n_axes, const uint8_t* pair_axis,
                              const float* inv_freq, uint32_t rot_dim, int interleaved,
                              void* stream) {
  const char* op = "rope_append_paged_q4";
  Q4AppendArgs a{};
  QWEN_TRY(check_q4(op, kv, n_heads, &a.page_shift));
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
  if (n_tokens > (1u << 24) || (uint64_t)n_tokens * (n_heads + kv->n_kv_heads) >= (1ull << 33))   // (blocks of the grid)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_tokens=%u of %u heads are more than one call takes", op, n_tokens,
                     n_heads);
  if (n_axes == 0 || n_axes > 4 || (n_axes > 1 && (!positions || !pair_axis)))
    return set_error(QWEN_ERR_INVALID_ARGUMENT,
                     "%s: n_axes=%u must be 1 to 4, with positions and pair_axis where it is over 1", op, n_axes);
  if (n_axes > 1 && (position_stride < 0 || position_stride >= (1ll << 38)))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: position_stride=%lld", op, (long long)position_stride);
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
  a.positions = positions;
  a.position_stride = position_stride;
  a.n_axes = (int)n_axes;
  a.pair_axis = pair_axis;
  a.inv_freq = inv_freq;
  a.rot_dim = (int)rot_dim;
  a.interleaved = interleaved ? 1 : 0;
  QWEN_TRY(ops_status_word(&a.err));
  return finish(op, launch_rope_append_q4(a, static_cast<cudaStream_t>(stream)));
}

size_t qwen_attention_paged_q4_workspace(const qwen_paged_kv_q4* kv, uint32_t n_heads) {
  int shift;
  const char* op = "attention_paged_q4";
  return kv && kv->n_seq != 0 && check_q4_sizes(op, kv, n_heads, &shift) == QWEN_OK &&
                 check_q4_tiles(op, kv, n_heads) == QWEN_OK
             ? attention_q4_workspace(*kv, (int)n_heads)
             : 0;
}

int qwen_attention_paged_q4(const qwen_paged_kv_q4* kv, const uint16_t* q, int64_t q_stride,
                            uint16_t* out, int64_t out_stride, float* lse, uint32_t n_heads,
                            const uint32_t* seq_len, float scale, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* op = "attention_paged_q4";
  Q4AttnArgs a{};
  QWEN_TRY(check_q4(op, kv, n_heads, &a.page_shift));
  if (kv->n_seq == 0) return QWEN_OK;
  QWEN_TRY(check_rows(op, "q", q, q_stride, n_heads * kv->head_dim));
  QWEN_TRY(check_rows(op, "out", out, out_stride, n_heads * kv->head_dim));
  if (!seq_len) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null seq_len", op);
  QWEN_TRY(check_workspace(op, workspace, workspace_bytes, qwen_attention_paged_q4_workspace(kv, n_heads)));
  QWEN_TRY(check_q4_tiles(op, kv, n_heads));
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
  return finish(op, launch_attention_q4(a, static_cast<cudaStream_t>(stream)));
}

int qwen_expand_paged_q4(const qwen_paged_kv_q4* kv, const uint32_t* seq_len,
                         const int32_t* cu_rows, uint32_t n_rows, uint16_t* k, int64_t k_stride,
                         uint16_t* v, int64_t v_stride, void* stream) {
  const char* op = "expand_paged_q4";
  Q4ExpandArgs a{};
  QWEN_TRY(check_q4(op, kv, kv ? kv->n_kv_heads : 0, &a.page_shift));
  if (!cu_rows && n_rows != kv->n_seq)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_rows=%u for %u sequences without cu_rows", op, n_rows,
                     kv->n_seq);
  if (kv->n_seq == 0 || n_rows == 0) return QWEN_OK;
  QWEN_TRY(check_rows(op, "k", k, k_stride, kv->n_kv_heads * kv->head_dim));
  QWEN_TRY(check_rows(op, "v", v, v_stride, kv->n_kv_heads * kv->head_dim));
  if (!seq_len) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null seq_len", op);
  if (n_rows > (1u << 30)) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_rows=%u", op, n_rows);
  a.kv = *kv;
  a.seq_len = seq_len;
  a.cu_rows = cu_rows;
  a.n_rows = (int)n_rows;
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  QWEN_TRY(ops_status_word(&a.err));
  return finish(op, launch_expand_q4(a, static_cast<cudaStream_t>(stream)));
}

size_t qwen_evict_paged_q4_workspace(const qwen_paged_kv_q4* kv, uint32_t n_keep) {
  int shift;
  const char* op = "evict_paged_q4";
  return kv && kv->n_seq != 0 && check_q4_sizes(op, kv, kv->n_kv_heads, &shift) == QWEN_OK &&
                 check_keep(op, n_keep) == QWEN_OK
             ? evict_q4_workspace(*kv, n_keep)
             : 0;
}

int qwen_evict_paged_q4(const qwen_paged_kv_q4* kv, const uint32_t* seq_len, uint32_t n_keep,
                        uint32_t n_first, uint32_t n_recent, uint32_t* new_len, void* workspace,
                        size_t workspace_bytes, void* stream) {
  const char* op = "evict_paged_q4";
  Q4EvictArgs a{};
  QWEN_TRY(check_q4(op, kv, kv ? kv->n_kv_heads : 0, &a.page_shift));
  if (kv->n_seq == 0) return QWEN_OK;
  if (!kv->weights || !kv->positions)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: the cache keeps no weights or positions", op);
  if (!seq_len || !new_len) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null seq_len or new_len", op);
  QWEN_TRY(check_keep(op, n_keep));
  if (n_first > (1u << 30) || n_recent > (1u << 30))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_first=%u n_recent=%u", op, n_first, n_recent);
  QWEN_TRY(check_workspace(op, workspace, workspace_bytes, qwen_evict_paged_q4_workspace(kv, n_keep)));
  a.kv = *kv;
  a.seq_len = seq_len;
  a.n_keep = (int)n_keep;
  a.n_first = (int)n_first;
  a.n_recent = (int)n_recent;
  a.new_len = new_len;
  a.workspace = workspace;
  QWEN_TRY(ops_status_word(&a.err));
  return finish(op, launch_evict_q4(a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
