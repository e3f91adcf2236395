// paged.h -- operators over a paged key/value cache (qwen_paged_kv of
// include/qwen_b200.h): parameters the entry points hand to the launchers.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/qwen_b200.h"

namespace qwen {

constexpr int kMaxGroup = 64;   // query heads per kv head

// What an attention launch reads and writes.  Rows are [heads][head_dim].
struct PagedAttnArgs {
  qwen_paged_kv kv;
  int page_shift;               // page_size = 1 << page_shift
  const uint16_t* q;
  long long q_stride;
  uint16_t* out;
  long long out_stride;
  float* lse;                   // may be null
  int n_heads;
  const uint32_t* seq_len;
  float scale;
  const int32_t* list;          // sparse: [n_seq][n_kv_heads][n_list] page_table columns
  int n_list;
  const int32_t* prefix_pages;  // shared prefix: pool pages, null without one
  uint32_t prefix_len;
  void* workspace;
  int* err;                     // operator status word
};
// Decode attention over own or listed pages (paged_decode.cu); 0, or -1 for a
// launch failure.  Beside a kernel that reads a shared prefix (the launch before it, which
// it does not wait for, though its end does): o, ml get unnormalised rows and (max,
// sum) per query head instead of outputs, and up to few_tiles tiles are divided among
// the `few` CTAs that find room at once.
struct PagedOwn {
  float* o = nullptr;
  float2* ml = nullptr;
  int few = 1;
  uint32_t few_tiles = 0;
};
int launch_paged_decode(const PagedAttnArgs& a, cudaStream_t st, const PagedOwn& own = {});
// Whether its tiles can be counted in 31 bits; n_list: listed pages, 0 without a list.
bool paged_decode_fits(const qwen_paged_kv& kv, int n_heads, int n_list);
size_t paged_decode_workspace(const qwen_paged_kv& kv, int n_heads);
// The same over a shared prefix (prefix_len > 0) and own pages (paged_prefix.cu).
int launch_paged_prefix(const PagedAttnArgs& a, cudaStream_t st);
size_t paged_prefix_workspace(const qwen_paged_kv& kv, int n_heads, uint32_t prefix_len);
int paged_sm_count();
// Tensor map of a pool, (element of 64, slot, half, head, page), boxes of box_rows
// slots and box_halves halves; 0 or -1.
int encode_pages_map(CUtensorMap* map, const qwen_paged_kv& kv, const uint16_t* base, int box_rows, int box_halves);

// A kernel's dynamic shared memory limit, raised before its first launch on each
// device, and again where a launch fails (a device that was reset forgets it).
class OncePerDevice {
 public:
  template <typename Launch>
  cudaError_t launch(const void* kernel, int smem, Launch&& go) {
    int d = 0;
    cudaError_t e = cudaGetDevice(&d);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (d & 63);
    if (d < 64 && mask_.load(std::memory_order_acquire) & bit) {
      e = go();
      if (e != cudaErrorInvalidValue) return e;
      cudaGetLastError();
    }
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    mask_.fetch_or(bit, std::memory_order_release);
    return go();
  }

 private:
  std::atomic<unsigned long long> mask_{0};
};

struct PagedAppendArgs {
  qwen_paged_kv kv;
  int page_shift;
  const uint16_t *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  uint16_t* q_out;
  long long q_out_stride;
  int n_heads;
  int n_tokens;
  const uint32_t* seq_len;
  const int32_t* cu_tokens;     // null: one token per sequence
  const float* inv_freq;
  int rot_dim;
  int interleaved;
  int* err;
};
int launch_rope_append(const PagedAppendArgs& a, cudaStream_t st);

struct PagedSelectArgs {
  qwen_paged_kv kv;
  int page_shift;
  const uint16_t* q;
  long long q_stride;
  int n_heads;
  const uint32_t* seq_len;
  int n_select, n_first, n_last;
  int32_t* pages;               // [n_seq][n_kv_heads][n_select]
  double* scores;               // workspace: [n_seq][n_kv_heads][max_pages]
  int* err;
};
int launch_select_pages(const PagedSelectArgs& a, cudaStream_t st);

}  // namespace qwen
