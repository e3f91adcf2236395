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

// Values low + code step of 8 codes in the cache's type, rounded once.  (1024 + code in fp16
// and 128 + code in bf16 are codes at the bottom of the mantissa.)
__device__ __forceinline__ uint4 expand_word(__half, uint32_t codes, uint32_t params) {
  const __half2 p = *reinterpret_cast<const __half2*>(&params), step = __low2half2(p), low = __high2half2(p);
  const __half2 k1024 = __float2half2_rn(1024.f), k64 = __float2half2_rn(64.f), k16th = __float2half2_rn(0.0625f);
  const uint32_t v = codes >> 8;
  uint32_t y[4];   // elements (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = lop3_and_or(i < 2 ? codes : v, i & 1 ? 0x00f000f0u : 0x000f000fu, 0x64006400u);
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    const __half2 c = i & 1 ? __hfma2(h, k16th, __hneg2(k64)) : __hsub2(h, k1024);   // (1024 + 16 code) / 16 - 64
    const __half2 r = __hfma2(c, step, low);
    y[i] = *reinterpret_cast<const uint32_t*>(&r);
  }
  return make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632),
                    __byte_perm(y[2], y[3], 0x7632));
}
__device__ __forceinline__ uint4 expand_word(__nv_bfloat16, uint32_t codes, uint32_t params) {
  const __nv_bfloat162 p = *reinterpret_cast<const __nv_bfloat162*>(&params), step = __low2bfloat162(p), low = __high2bfloat162(p);
  const __nv_bfloat162 k128 = __float2bfloat162_rn(128.f);
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = lop3_and_or(codes >> (4 * i), 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 r = __hfma2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&w), k128), step, low);
    y[i] = *reinterpret_cast<const uint32_t*>(&r);
  }
  return make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632),
                    __byte_perm(y[2], y[3], 0x7632));
}

}  // namespace qwen
