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

// c, the nearest whole number to t = (x - low) / step or, from rounding, its neighbour at a
// border, put right: on which side of the border b the true quotient lies is the sign of x -
// low - b step.  r + e is x - low exactly; b step has 16 bits, so that its difference from r,
// near 0 where it matters, is exact, and a sum's sign is right.
__device__ __forceinline__ float exact_code(float x, float low, float step, float t, float c) {
  const float r = __fadd_rn(x, -low), z = __fadd_rn(r, -x);
  const float e = __fadd_rn(__fadd_rn(x, -__fadd_rn(r, -z)), -__fadd_rn(low, z));
  const float b = c + (t < c ? -0.5f : 0.5f), d = __fadd_rn(fmaf(-b, step, r), e);
  const float below = b - 0.5f, even = 2.f * rintf(0.5f * b);   // (of below and below + 1)
  return fminf(d == 0.f ? even : d > 0.f ? below + 1.f : below, 15.f);
}
// The same where the step's reciprocal is beyond fp32 (bf16 steps below 2^-128): everything
// times 2^64, which is exact.
static __device__ __noinline__ uint32_t tiny_codes(float4 a, float4 b, float low, float step) {
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const float k = 18446744073709551616.f, inv = __frcp_rn(step * k);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fminf((x[i] * k - low * k) * inv, 15.f);
    codes |= (uint32_t)exact_code(x[i] * k, low * k, step * k, t, rintf(t)) << (4 * i);
  }
  return codes;
}
// Quantises a group of 32 values, of which this lane holds 8 (fp32, exact) and its three
// neighbours (lane ^ 1, ^ 2, ^ 3) the rest; all 32 lanes take part.  Returns the lane's
// codes, element i in bits 4i .. 4i+3, and (step, low) as the cache keeps them.
//
// The fp32 quotient is off by at most 15 (2^-24 + 2^-24 + 2^-24) < 3e-6 (difference,
// reciprocal, product); where one stands nearer than 1e-5 to a border between two codes,
// exact_code decides (of bf16's few values one in some hundred is on one).  Rounded by an
// addition, and packed four at a time by multiplication: conversions run at an eighth of the
// rate.
template <typename T>
__device__ __forceinline__ uint32_t quantise_group(const float (&x)[8], uint32_t* params) {
  float lo = x[0], hi = x[0], bad = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad = fmaf(x[i], 0.f, bad);   // NaN for an infinity or NaN
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad += __shfl_xor_sync(0xffffffffu, bad, o);
  }
  if (bad != 0.f) lo = hi = bad;
  const uint32_t p = pack2(T{}, (float)(((double)hi - (double)lo) * (1.0 / 15.0)), lo);
  *params = p;
  const float step = unpack2(T{}, p).x;
  if (!(step > 0.f)) return 0;   // 0 or NaN
  constexpr float kMagic = 12582912.f;   // 1.5 2^23: sums are rounded to whole numbers, ties to even
  const float inv = __frcp_rn(step);
  float c[8], off = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fminf((x[i] - lo) * inv, 15.f);
    c[i] = __fadd_rn(__fadd_rn(t, kMagic), -kMagic);
    off = fmaxf(off, fabsf(t - c[i]));
  }
  if (!(inv < INFINITY)) return tiny_codes(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), lo, step);
  if (off > 0.49999f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = (x[i] - lo) * inv;
      if (fabsf(t - c[i]) > 0.49999f) c[i] = exact_code(x[i], lo, step, t, c[i]);
    }
  }
  const float a = fmaf(c[3], 4096.f, fmaf(c[2], 256.f, fmaf(c[1], 16.f, c[0])));
  const float b = fmaf(c[7], 4096.f, fmaf(c[6], 256.f, fmaf(c[5], 16.f, c[4])));
  return __byte_perm(__float_as_uint(a + 8388608.f), __float_as_uint(b + 8388608.f), 0x5410);
}

// Values low + code step of 8 codes, rounded to fp32.
template <typename T>
__device__ __forceinline__ void expand_word(uint32_t codes, uint32_t params, float (&x)[8]) {
  const float2 p = unpack2(T{}, params);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf((float)(codes >> (4 * i) & 15), p.x, p.y);
}

}  // namespace qwen
