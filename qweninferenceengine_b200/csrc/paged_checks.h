// paged_checks.h -- argument checks of the paged-cache entry points, of 16-bit caches
// (capi_paged.cu) and of 4-bit ones (capi_paged_q4.cu).
#pragma once
#include <cstdint>

#include "paged.h"
#include "status.h"

namespace qwen {
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr uint32_t kMaxPositions = 1u << 24;   // of a sequence: positions are exact in fp32
constexpr uint32_t kMaxSeqs = 65535;           // of a call: grid rows

bool heads_fit(const qwen_paged_kv& kv, uint32_t n_heads) {
  return kv.n_kv_heads != 0 && kv.n_kv_heads <= 1024 && n_heads != 0 && n_heads % kv.n_kv_heads == 0 &&
         n_heads / kv.n_kv_heads <= (uint32_t)kMaxGroup;
}
// What a call and its workspace query both look at: type and sizes.
int check_sizes(const char* op, const qwen_paged_kv* kv, uint32_t n_heads, int* page_shift) {
  if (kv->dtype != QWEN_DTYPE_F16 && kv->dtype != QWEN_DTYPE_BF16)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: dtype=%d", op, kv->dtype);
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: head_dim=%u must be 64 or 128", op, kv->head_dim);
  int shift = 4;
  while (shift < 8 && (1u << shift) != kv->page_size) ++shift;
  if ((1u << shift) != kv->page_size)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: page_size=%u must be a power of two in [16, 256]",
                     op, kv->page_size);
  *page_shift = shift;
  if (kv->n_pages == 0 || kv->n_pages > (1u << 30))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_pages=%u", op, kv->n_pages);
  if (kv->n_seq > kMaxSeqs) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: n_seq=%u", op, kv->n_seq);
  if (kv->max_pages == 0 || (uint64_t)kv->max_pages * kv->page_size > kMaxPositions ||
      kv->table_stride < kv->max_pages)
    return set_error(QWEN_ERR_INVALID_ARGUMENT,
                     "%s: max_pages=%u (at most 2^24 positions) table_stride=%u", op, kv->max_pages,
                     kv->table_stride);
  if (!heads_fit(*kv, n_heads))
    return set_error(QWEN_ERR_INVALID_ARGUMENT,
                     "%s: n_heads=%u must be a multiple of n_kv_heads=%u, at most %d times it", op,
                     n_heads, kv->n_kv_heads, kMaxGroup);
  return QWEN_OK;
}

// A [rows][width] buffer with a row stride (asked where there are rows).
int check_rows(const char* op, const char* name, const void* p, int64_t stride, uint32_t width) {
  if (!p) return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: null %s", op, name);
  if (!aligned16(p) || stride % 8 != 0 || stride < (int64_t)width || stride >= (1ll << 38))
    return set_error(QWEN_ERR_INVALID_ARGUMENT,
                     "%s: %s must be 16-byte aligned, its row stride %lld a multiple of 8 and at least %u",
                     op, name, (long long)stride, width);
  return QWEN_OK;
}

int check_workspace(const char* op, const void* p, size_t bytes, size_t need) {
  if (bytes < need)
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, %zu needed", op, bytes, need);
  if (need && (!p || (reinterpret_cast<uintptr_t>(p) & 255)))
    return set_error(QWEN_ERR_INVALID_ARGUMENT, "%s: workspace must be 256-byte aligned memory", op);
  return QWEN_OK;
}

int finish(const char* op, int launched) {
  QWEN_TRY(launch_status(op));
  return launched == 0 ? QWEN_OK : set_error(QWEN_ERR_CUDA, "%s: launch failed", op);
}

}  // namespace
}  // namespace qwen
