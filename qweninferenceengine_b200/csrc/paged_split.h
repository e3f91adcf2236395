// paged_split.h -- arithmetic of the paged kernels that the host can run too: where
// the warps of k_prefix put their rows in shared memory.  Plain C++, so that the tests
// check what the kernels use.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define QWEN_HD __host__ __device__ __forceinline__
#else
#define QWEN_HD inline
#endif

namespace qwen {

constexpr int kRows = 128;                 // rows of a stream of k_prefix (M)
constexpr int kWarpRows = 16;              // of them, those whose queries a softmax warp loads

// Byte of 16-byte chunk x of row r in a stream's query tile: [half][row][128 B], swizzled.
QWEN_HD int query_byte(int r, int x) { return (x >> 3) * kRows * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4); }
// Byte of 16-byte chunk x of row r < 32 (D / 16 chunks of fp32 a row) that the stream's
// softmax warp j stages in the same tile: the bytes that its own 16 rows of queries take,
// 2 KB of each half, since a warp goes on from one piece's output to the next piece's
// queries without waiting for the others.
QWEN_HD int stage_byte(int D, int j, int r, int x) {
  const int at = r * D;   // of the warp's 32 D bytes
  return (at >> 11) * kRows * 128 + j * kWarpRows * 128 + (at & 2047) + ((x ^ (r & (D / 16 - 1))) << 4);
}

}  // namespace qwen
