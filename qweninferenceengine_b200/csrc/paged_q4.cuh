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
__device__ __forceinline__ float rcp_fast(float x) {   // 1 step of fp32; a subnormal gives infinity
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Codes of 8 values by exact_code alone, for steps near their type's ends: everything times
// 2^64 or 1/4, which is exact (the reciprocal of bf16's least steps and the difference of its
// greatest values are beyond fp32).
static __device__ __noinline__ uint32_t end_codes(float4 a, float4 b, float low, float step) {
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const float k = step < 1.f ? 18446744073709551616.f : 0.25f, inv = rcp_fast(step * k);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fminf((x[i] * k - low * k) * inv, 15.f);
    codes |= (uint32_t)exact_code(x[i] * k, low * k, step * k, t, rintf(t)) << (4 * i);
  }
  return codes;
}
__device__ __forceinline__ uint32_t least2(__half, uint32_t a, uint32_t b) {   // NaN if either is
  const __half2 r = __hmin2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t least2(__nv_bfloat16, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t most2(__half, uint32_t a, uint32_t b) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t most2(__nv_bfloat16, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Quantises a group of 32 values, of which this lane holds 8 and its three neighbours (lane ^ 1,
// ^ 2, ^ 3) the rest; all 32 lanes take part.  Returns the lane's codes, element i in bits 4i
// .. 4i+3, and (step, low) as the cache keeps them.
//
// The least and the greatest are found in pairs, and exchanged as one word (least, -greatest).
// Quotients are formed in fixed point: 1.5 2^11 + (x - low) / step + 1/2 has steps of 2^-12, so
// that one multiply-add leaves a code in bits 12 .. 15.  It is off by two roundings (that of
// its constant, as |low / step| < 1000, and its own: one 2^-12) and 15.1 2^-23 from the
// reciprocal, less than 1.01 2^-12 in all; where it stands within 2 2^-12 of a border between two
// codes, exact_code decides (of bf16's few values one in some hundred is on one).
template <typename T>
__device__ __forceinline__ uint32_t quantise_group(const uint4& v, uint32_t* params) {
  const uint32_t a = least2(T{}, least2(T{}, v.x, v.y), least2(T{}, v.z, v.w));
  const uint32_t b = most2(T{}, most2(T{}, v.x, v.y), most2(T{}, v.z, v.w)) ^ 0x80008000u;
  uint32_t ends = least2(T{}, __byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
  ends = least2(T{}, ends, __shfl_xor_sync(0xffffffffu, ends, 1));
  ends = least2(T{}, ends, __shfl_xor_sync(0xffffffffu, ends, 2));
  float lo = unpack2(T{}, ends).x, hi = -unpack2(T{}, ends).y;
  if (!(fabsf(lo) < INFINITY && fabsf(hi) < INFINITY)) lo = hi = __int_as_float(0x7fffffff);
  const uint32_t p = pack2(T{}, (float)(((double)hi - (double)lo) * (1.0 / 15.0)), lo);
  *params = p;
  const float step = unpack2(T{}, p).x;
  if (!(step > 0.f)) return 0;   // 0 or NaN
  const float inv = rcp_fast(step);
  const float2 v0 = unpack2(T{}, v.x), v1 = unpack2(T{}, v.y), v2 = unpack2(T{}, v.z), v3 = unpack2(T{}, v.w);
  const float x[8] = {v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
  // (a step far below its type's normal ones can be so much less than a fifteenth that quotients
  // pass 15.5; and see end_codes)
  if (!((hi - lo) * inv < 15.4f && fabsf(lo * inv) < 1000.f))
    return end_codes(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), lo, step);
  constexpr float kHalf = 1.5f * 2048.f + 0.5f + 2.f / 4096.f;   // (below a border: 0 or 1 2^-12, on it or above: 2 or 3)
  const float from = fmaf(-lo, inv, kHalf);
  uint32_t at[4];   // elements i and i + 4
#pragma unroll
  for (int i = 0; i < 4; ++i)
    at[i] = __byte_perm(__float_as_uint(fmaf(x[i], inv, from)), __float_as_uint(fmaf(x[i + 4], inv, from)), 0x5410);
  uint32_t codes = (at[0] >> 12 & 0x000f000fu) | (at[1] >> 8 & 0x00f000f0u) | (at[2] >> 4 & 0x0f000f00u) | (at[3] & 0xf000f000u);
  uint32_t clear = 0x80008000u;   // bits 15: no quotient is near a border
#pragma unroll
  for (int i = 0; i < 4; ++i) clear &= (at[i] & 0x0ffc0ffcu) + 0x7fff7fffu;
  if (clear != 0x80008000u) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((at[i & 3] >> (i < 4 ? 0 : 16) & 0xffcu) == 0) {
        const float t = (x[i] - lo) * inv;
        codes = (codes & ~(15u << (4 * i))) | (uint32_t)exact_code(x[i], lo, step, t, rintf(t)) << (4 * i);
      }
  }
  return codes;
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
