// paged_q4.h -- operators over a paged cache held in 4 bits (qwen_paged_kv_q4 of
// include/qwen_b200.h): parameters the entry points hand to the launchers.
#pragma once
#include "paged.h"

namespace qwen {

struct Q4AppendArgs {
  qwen_paged_kv_q4 kv;
  int page_shift;
  const uint16_t *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  uint16_t* q_out;
  long long q_out_stride;
  int n_heads;
  int n_tokens;
  const uint32_t* seq_len;
  const int32_t* cu_tokens;     // null: one token per sequence
  const int32_t* positions;     // null: slots
  long long position_stride;    // between axes
  int n_axes;
  const uint8_t* pair_axis;     // null: axis 0
  const float* inv_freq;
  int rot_dim;
  int interleaved;
  int* err;
};
int launch_rope_append_q4(const Q4AppendArgs& a, cudaStream_t st);

struct Q4ExpandArgs {
  qwen_paged_kv_q4 kv;
  int page_shift;
  const uint32_t* seq_len;
  const int32_t* cu_rows;       // null: a row per sequence
  int n_rows;
  uint16_t *k, *v;
  long long k_stride, v_stride;
  int* err;
};
int launch_expand_q4(const Q4ExpandArgs& a, cudaStream_t st);

struct Q4AttnArgs {
  qwen_paged_kv_q4 kv;
  int page_shift;
  const uint16_t* q;
  long long q_stride;
  uint16_t* out;
  long long out_stride;
  float* lse;                   // may be null
  int n_heads;
  const uint32_t* seq_len;
  float scale;
  void* workspace;
  int* err;
};
int launch_attention_q4(const Q4AttnArgs& a, cudaStream_t st);
// Whether its tiles can be counted in 31 bits.
bool attention_q4_fits(const qwen_paged_kv_q4& kv, int n_heads);
size_t attention_q4_workspace(const qwen_paged_kv_q4& kv, int n_heads);

struct Q4EvictArgs {
  qwen_paged_kv_q4 kv;
  int page_shift;
  const uint32_t* seq_len;
  int n_keep, n_first, n_recent;
  uint32_t* new_len;
  void* workspace;
  int* err;
};
int launch_evict_q4(const Q4EvictArgs& a, cudaStream_t st);
size_t evict_q4_workspace(const qwen_paged_kv_q4& kv, uint32_t n_keep);

}  // namespace qwen
