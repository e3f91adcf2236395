// paged_q4.cuh -- device helpers of the 4-bit paged cache: where its parts lie, its
// quantisation.
#pragma once
#include "paged_common.cuh"
#include "paged_q4.h"

namespace qwen {

// A block of 16 slots (20 D bytes): key codes [D/32][16][16 B], value codes from 8 D on,
// (step, low) of keys [D/32][16][4 B] from 16 D on, of values from 18 D on.
template <int D>
struct Q4Block {
  static constexpr int kGroups = D / 32, kBytes = 20 * D;
  static constexpr int kValues = 8 * D, kKeySteps = 16 * D, kValueSteps = 18 * D;
};
// Block of a slot of head h in a page, counted from the page's first slot.
template <int D>
__device__ __forceinline__ uint8_t* q4_block(const qwen_paged_kv_q4& kv, int page, int h, int slot) {
  return kv.pool + (long long)page * kv.page_stride + (long long)h * kv.head_stride + (slot >> 4) * Q4Block<D>::kBytes;
}
// The pool page of a table entry, or -1 with the status word set.
__device__ __forceinline__ int q4_page(const qwen_paged_kv_q4& kv, int* err, int s, int col) {
  const int page = kv.page_table[(long long)s * kv.table_stride + col];
  if (page >= 0 && (uint32_t)page < kv.n_pages) return page;
  raise_error(err, kDevBadArgument);
  return -1;
}
__device__ __forceinline__ uint32_t q4_capacity(const qwen_paged_kv_q4& kv) { return kv.max_pages * kv.page_size; }

// Quantises a group of 32 values, of which this lane holds 8 (fp32, exact) and its three
// neighbours (lane ^ 1, ^ 2, ^ 3) the rest; all 32 lanes take part.  Returns the lane's
// codes, element i in bits 4i .. 4i+3, and (step, low) as the cache keeps them.
//
// A code is exact, as if (x - low) / step were rounded from its true value: the fp32
// quotient is off by at most 15 (2^-24 + 2^-23 + 2^-24) < 4e-6 (difference, reciprocal,
// product), and where it stands nearer than 1e-5 to a border between two codes (once in
// 50,000 values), 64 bits decide.
template <typename T>
__device__ __forceinline__ uint32_t quantise_group(const float (&x)[8], uint32_t* params) {
  float lo = x[0], hi = x[0], bad = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad += x[i] * 0.f;   // NaN for an infinity or NaN
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad += __shfl_xor_sync(0xffffffffu, bad, o);
  }
  if (bad != 0.f) lo = hi = bad;
  const uint32_t p = pack2(T{}, (float)(((double)hi - (double)lo) / 15.0), lo);
  *params = p;
  const float step = unpack2(T{}, p).x;
  uint32_t codes = 0;
  if (!(step > 0.f)) return 0;   // 0 or NaN
  const float inv = __frcp_rn(step);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = (x[i] - lo) * inv, c = rintf(t);
    uint32_t code = (uint32_t)(int)c;
    if (!(fabsf(fabsf(t - c) - 0.5f) > 1e-5f) || !(inv < INFINITY))
      code = (uint32_t)rint(((double)x[i] - (double)lo) / (double)step);
    codes |= min(code, 15u) << (4 * i);
  }
  return codes;
}

// Values low + code step of 8 codes, rounded to fp32.
template <typename T>
__device__ __forceinline__ void expand_word(uint32_t codes, uint32_t params, float (&x)[8]) {
  const float2 p = unpack2(T{}, params);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf((float)(codes >> (4 * i) & 15), p.x, p.y);
}

}  // namespace qwen
