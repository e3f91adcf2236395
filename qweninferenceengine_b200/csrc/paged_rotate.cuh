// paged_rotate.cuh -- rotation of 16-element chunks of a head, and the search for a row's
// sequence, for the kernels that append to 16-bit (paged_append.cu) and 4-bit caches.
#pragma once
#include "paged_common.cuh"

namespace qwen {
namespace {

__device__ __forceinline__ void sincos_of(float pos, float inv_freq, float* sn, float* cs) {
  const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;
  sincospif(2.0f * (float)(turns - rint(turns)), sn, cs);
}

// 16 elements: the words of two 16-byte halves.
struct Chunk {
  uint32_t w[8];
};
__device__ __forceinline__ Chunk load_chunk(const void* a, const void* b) {
  const uint4 x = *reinterpret_cast<const uint4*>(a), y = *reinterpret_cast<const uint4*>(b);
  return {{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}};
}
__device__ __forceinline__ void store_chunk(void* a, void* b, const Chunk& c) {
  *reinterpret_cast<uint4*>(a) = make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]);
  *reinterpret_cast<uint4*>(b) = make_uint4(c.w[4], c.w[5], c.w[6], c.w[7]);
}
// Where chunk c's halves lie in a head.
template <bool kInterleaved>
__device__ __forceinline__ void places(int c, int R, int* a, int* b) {
  const bool split = !kInterleaved && 16 * c < R;
  *a = split ? 8 * c : 16 * c;
  *b = split ? R / 2 + 8 * c : 16 * c + 8;
}
// rot: (cos, sin) of the chunk's eight pairs.
template <typename T, bool kInterleaved>
__device__ __forceinline__ void rotate_chunk(Chunk& x, const float2 (&rot)[8]) {
  if constexpr (kInterleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = unpack2(T{}, x.w[i]);
      x.w[i] = pack2(T{}, v.x * rot[i].x - v.y * rot[i].y, v.x * rot[i].y + v.y * rot[i].x);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = unpack2(T{}, x.w[i]), b = unpack2(T{}, x.w[4 + i]);
      const float2 r0 = rot[2 * i], r1 = rot[2 * i + 1];
      x.w[i] = pack2(T{}, a.x * r0.x - b.x * r0.y, a.y * r1.x - b.y * r1.y);
      x.w[4 + i] = pack2(T{}, a.x * r0.y + b.x * r0.x, a.y * r1.y + b.y * r1.x);
    }
  }
}

// First sequence s with base(s + 1) > x, base(s) = (cu[s] >> shift) + per_seq * s.
// A warp: x is the same for the lanes of each group of kLanes.
template <int kLanes>
__device__ __forceinline__ int seq_of(const int32_t* cu, int n_seq, int shift, int per_seq, int x, int lane) {
  if (n_seq <= 256) {   // the lanes read all starts at once and count those up to x
    int s = 0;
#pragma unroll 1
    for (int b = 0; b < n_seq; b += 32) {
      const int start = b + lane < n_seq ? (cu[b + lane + 1] >> shift) + per_seq * (b + lane + 1) : 0x7fffffff;
#pragma unroll
      for (int g = 0; g < 32; g += kLanes) {
        const int count = __popc(__ballot_sync(0xffffffffu, start <= __shfl_sync(0xffffffffu, x, g)));
        if (lane / kLanes == g / kLanes) s += count;
      }
    }
    return min(s, n_seq - 1);
  }
  int lo = 0, hi = n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((cu[mid + 1] >> shift) + per_seq * (mid + 1) > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

}  // namespace
}  // namespace qwen
