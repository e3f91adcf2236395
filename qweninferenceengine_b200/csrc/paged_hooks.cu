// paged_hooks.cu -- test hooks: the paged kernels' host arithmetic (paged_split.h), for
// tests without a GPU.
#include "paged_split.h"

using namespace qwen;

extern "C" {

// Bytes of the query tile that softmax warp j of a stream of k_prefix writes queries to
// (query: [8][16 rows][dim / 8]) and stages output rows in (stage: [8][32 rows][dim / 16]).
void qwen_paged_prefix_tile(int dim, int* query, int* stage) {
  for (int j = 0; j < 8; ++j) {
    for (int r = 0; r < kWarpRows; ++r)
      for (int x = 0; x < dim / 8; ++x) *query++ = query_byte(j * kWarpRows + r, x);
    for (int r = 0; r < 32; ++r)
      for (int x = 0; x < dim / 16; ++x) *stage++ = stage_byte(dim, j, r, x);
  }
}

}  // extern "C"
