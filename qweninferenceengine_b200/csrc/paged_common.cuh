// paged_common.cuh -- device helpers shared by the paged-cache kernels.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"
#include "paged_split.h"
#include "qwen_common.cuh"

namespace qwen {

// Two 16-bit values of either type in a word, and their fp32 values.
__device__ __forceinline__ float2 unpack2(__half, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 unpack2(__nv_bfloat16, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(__half, float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The same two values with infinities and NaN replaced by finite ones: +-65504, or +-2^96
// (and bf16 beyond that), whose products with up to 2^24 weights of up to 2^7 are finite.
__device__ __forceinline__ uint32_t finite2(__half, uint32_t w) {
  uint32_t r;   // the lesser magnitude, w's sign
  asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0x7bff7bffu));
  return r;
}
__device__ __forceinline__ uint32_t finite2(__nv_bfloat16, uint32_t w) {
  uint32_t r;
  asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0x6f806f80u));
  return r;
}
// D = A(16x16, row) * B(16x8, col) + D, fp32 accumulation.
__device__ __forceinline__ void mma_16816_t(__half, float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1) {
  mma_16816(d, a, b0, b1, d);
}
__device__ __forceinline__ void mma_16816_t(__nv_bfloat16, float (&d)[4], const uint32_t (&a)[4],
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {   // ex2.approx: 2 steps of fp32; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ unsigned long long global_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
constexpr unsigned long long kPagedWaitNs = 2000000000ull;
// Bounded parity wait: false once it ran out (2 s; recorded, *abort set) or,
// where `heed`, once another role of the CTA gave up.
static __device__ __noinline__ bool paged_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort,
                                             int* err, bool heed) {
  if (heed && *abort) return false;
  const unsigned long long t0 = global_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 0) {
      if (heed && *abort) return false;
      if (global_ns() - t0 > kPagedWaitNs) {
        *abort = 1;
        raise_error(err, kDevWaitTimeout);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool paged_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err,
                                           bool heed = true) {
  return mbar_try_wait(bar, parity) || paged_wait_slow(bar, parity, abort, err, heed);
}
// 5-D tile load (element, slot, half, head, page) of a cache's tensor map; the
// box is (64, rows, head_dim / 64, 1, 1), so it lands as [half][rows][128 B].
__device__ __forceinline__ void tma_load_pages(void* dst, const CUtensorMap* map, int slot, int head,
                                               int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(slot), "r"(0), "r"(head), "r"(page),
      "r"(smem_u32(bar))
      : "memory");
}

// One half (64 elements) of the same, box (64, rows, 1, 1, 1).
__device__ __forceinline__ void tma_load_half(void* dst, const CUtensorMap* map, int slot, int half, int head,
                                              int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(slot), "r"(half), "r"(head), "r"(page),
      "r"(smem_u32(bar))
      : "memory");
}

// 128 or 64 fp32 values of a row, D / 32 to a lane.
__device__ __forceinline__ void load_vec(float (&v)[4], const float* p) {
  const float4 x = __ldcg(reinterpret_cast<const float4*>(p));
  v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}
__device__ __forceinline__ void load_vec(float (&v)[2], const float* p) {
  const float2 x = __ldcg(reinterpret_cast<const float2*>(p));
  v[0] = x.x, v[1] = x.y;
}
// Output row and log-sum-exp from the unnormalised row v (this lane's D / 32 values
// of it), its maximum and sum.  rcp and lg2 approximate to 2 steps of fp32.
template <typename T, int D>
__device__ __forceinline__ void write_row(const PagedAttnArgs& a, int seq, int head, float4 v, float M, float sum,
                                          int lane) {
  const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
  T* dst = reinterpret_cast<T*>(a.out) + (long long)seq * a.out_stride + (long long)head * D + D / 32 * lane;
  const uint32_t lo = pack2(T{}, v.x * inv, v.y * inv);
  if constexpr (D == 128) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, pack2(T{}, v.z * inv, v.w * inv));
  else *reinterpret_cast<uint32_t*>(dst) = lo;
  if (a.lse && lane == 0)
    a.lse[(long long)seq * a.n_heads + head] = sum == 0.f ? -INFINITY : (M + __log2f(sum)) * kLn2;
}
__device__ __forceinline__ float4 as_float4(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ float4 as_float4(const float (&v)[2]) { return make_float4(v[0], v[1], 0.f, 0.f); }

// Positions of sequence s, or 0 with the status word set when the length does
// not fit its row of the page table (*ok false).
__device__ __forceinline__ uint32_t checked_len(const qwen_paged_kv& kv, const uint32_t* seq_len,
                                                int s, bool* ok) {
  const uint32_t L = seq_len[s];
  *ok = L <= kv.max_pages * kv.page_size;
  return *ok ? L : 0;
}

}  // namespace qwen
