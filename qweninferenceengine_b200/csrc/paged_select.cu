// paged_select.cu -- the pages whose bounds promise the highest scores.
//
//   score(page) = sum_h sum_d max(q_hd lo_d, q_hd hi_d)
//               = sum_d (Q+_d hi_d + Q-_d lo_d),  Q+-_d = sum_h max/min(q_hd, 0)
//
// over the query heads h of a kv head: one dot product of 2 head_dim elements a
// page whatever the number of heads, and never less than sum_h q_h . k for a key
// of the page.  Sums are held in 64 bits: the list is whole numbers, and in
// 32 bits two pages closer than ~1e-6 would change places with the order of a
// sum.
#include "paged_common.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kSelectThreads = 256;

// Ascending order of keys = ascending order of scores; NaN above everything.
__device__ __forceinline__ unsigned long long score_key(double x) {
  if (x != x) return ~0ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// One CTA per (kv head, sequence): scores, then each page's rank by counting.
template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads) k_select_pages(PagedSelectArgs a) {
  const int h = blockIdx.x, s = blockIdx.y, K = a.kv.n_kv_heads, G = a.n_heads / K;
  const int tid = threadIdx.x;
  __shared__ double qp[D], qn[D];
  __shared__ int count;
  bool ok;
  const int L = (int)checked_len(a.kv, a.seq_len, s, &ok);
  if (!ok) {
    if (tid == 0) raise_error(a.err, kDevBadArgument);
    return;
  }
  const int n = (L + a.kv.page_size - 1) >> a.page_shift;
  int32_t* list = a.pages + ((long long)s * K + h) * a.n_select;
  if (n <= a.n_select) {
    for (int i = tid; i < a.n_select; i += kSelectThreads) list[i] = i < n ? i : -1;
    return;
  }
  for (int d = tid; d < D; d += kSelectThreads) {
    double p = 0, m = 0;
    for (int g = 0; g < G; ++g) {
      const double x = to_f32(reinterpret_cast<const T*>(a.q)[s * a.q_stride + (h * G + g) * D + d]);
      p += x > 0 ? x : 0;
      m += x > 0 ? 0 : x;
    }
    qp[d] = p;
    qn[d] = m;
  }
  if (tid == 0) count = 0;
  __syncthreads();
  unsigned long long* keys =
      reinterpret_cast<unsigned long long*>(a.scores) + ((long long)s * K + h) * a.kv.max_pages;
  const int32_t* table = a.kv.page_table + (long long)s * a.kv.table_stride;
  for (int i = tid; i < n; i += kSelectThreads) {
    const int page = table[i];
    unsigned long long key = 0;
    if (page < 0 || (uint32_t)page >= a.kv.n_pages) {
      raise_error(a.err, kDevBadArgument);
    } else {
      const T* lo = reinterpret_cast<const T*>(a.kv.bounds) + ((long long)page * 2 * K + h) * D;
      const T* hi = lo + (long long)K * D;
      double x = 0;
      for (int d = 0; d < D; ++d)
        x += qp[d] * (double)to_f32(hi[d]) + qn[d] * (double)to_f32(lo[d]);
      if (x != x) {   // 0 times an infinite bound that no query reads adds nothing
        x = 0;
        for (int d = 0; d < D; ++d)
          x += (qp[d] != 0 ? qp[d] * (double)to_f32(hi[d]) : 0) + (qn[d] != 0 ? qn[d] * (double)to_f32(lo[d]) : 0);
      }
      key = score_key(x);
    }
    keys[i] = key;
  }
  __syncthreads();
  const int wanted = a.n_select - a.n_first - a.n_last, end = n - a.n_last;
  for (int i = tid; i < n; i += kSelectThreads) {
    bool take = i < a.n_first || i >= end;
    if (!take) {
      int better = 0;
      for (int j = a.n_first; j < end; ++j)
        better += keys[j] > keys[i] || (keys[j] == keys[i] && j < i);
      take = better < wanted;
    }
    if (take) list[atomicAdd(&count, 1)] = i;
  }
  __syncthreads();
  if (tid == 0)   // ascending
    for (int i = 1; i < a.n_select; ++i) {
      const int x = list[i];
      int j = i;
      for (; j > 0 && list[j - 1] > x; --j) list[j] = list[j - 1];
      list[j] = x;
    }
}

}  // namespace

int launch_select_pages(const PagedSelectArgs& a, cudaStream_t st) {
  const dim3 grid(a.kv.n_kv_heads, a.kv.n_seq);
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16)
    d64 ? k_select_pages<__half, 64><<<grid, kSelectThreads, 0, st>>>(a)
        : k_select_pages<__half, 128><<<grid, kSelectThreads, 0, st>>>(a);
  else
    d64 ? k_select_pages<__nv_bfloat16, 64><<<grid, kSelectThreads, 0, st>>>(a)
        : k_select_pages<__nv_bfloat16, 128><<<grid, kSelectThreads, 0, st>>>(a);
  return 0;
}

}  // namespace qwen
