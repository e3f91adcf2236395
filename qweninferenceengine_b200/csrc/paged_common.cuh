// paged_common.cuh -- device helpers shared by the paged-cache kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"
#include "qwen_common.cuh"

namespace qwen {

// fp16 / bf16 value types behind the 16-bit patterns of the C ABI.
template <typename T>
struct Half2Of;
template <>
struct Half2Of<__half> {
  using type = __half2;
};
template <>
struct Half2Of<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Positions of sequence s, or 0 with the status word set when the length does
// not fit its row of the page table (*ok false).
__device__ __forceinline__ uint32_t checked_len(const qwen_paged_kv& kv, const uint32_t* seq_len,
                                                int s, bool* ok) {
  const uint32_t L = seq_len[s];
  *ok = L <= kv.max_pages * kv.page_size;
  return *ok ? L : 0;
}

}  // namespace qwen
