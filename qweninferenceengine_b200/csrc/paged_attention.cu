// paged_attention.cu -- decode attention over a paged cache:
//   out = sum_t softmax(scale q . K_t) V_t
// over a sequence's own pages, the listed ones, or a shared prefix and its own.
//
// One warp per (query head, sequence): lane l holds elements l, l + 32, .. of
// the head; per position the dot product is one warp sum, and the running
// maximum and sum of the softmax and the weighted values are kept in fp32.
#include "paged_common.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

template <typename T, int D>
struct Running {
  float q[D / 32], o[D / 32];
  float m = -INFINITY, l = 0.f;
  __device__ void add(const T* k, const T* v, int lane) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) s += q[i] * to_f32(k[lane + 32 * i]);
    s = warp_sum(s);
    const float m_new = fmaxf(m, s);
    const float c = m == -INFINITY ? 0.f : expf(m - m_new), p = expf(s - m_new);
    l = l * c + p;
    m = m_new;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = o[i] * c + p * to_f32(v[lane + 32 * i]);
  }
  // Positions 0 .. n-1 of pool page `page`.
  __device__ void add_page(const PagedAttnArgs& a, int page, int h, int n, int lane) {
    if (page < 0 || (uint32_t)page >= a.kv.n_pages) {
      if (lane == 0) raise_error(a.err, kDevBadArgument);
      return;
    }
    const long long base = (long long)page * a.kv.page_stride + (long long)h * a.kv.head_stride;
    for (int i = 0; i < n; ++i)
      add(reinterpret_cast<const T*>(a.kv.k) + base + i * a.kv.pos_stride,
          reinterpret_cast<const T*>(a.kv.v) + base + i * a.kv.pos_stride, lane);
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(32) k_paged_attention(PagedAttnArgs a) {
  const int head = blockIdx.x, s = blockIdx.y, lane = threadIdx.x;
  const int h = head / (a.n_heads / (int)a.kv.n_kv_heads), P = a.kv.page_size;
  bool ok;
  const int L = (int)checked_len(a.kv, a.seq_len, s, &ok);
  if (!ok) {
    if (lane == 0) raise_error(a.err, kDevBadArgument);
    return;
  }
  Running<T, D> r;
  const T* q = reinterpret_cast<const T*>(a.q) + s * a.q_stride + head * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    r.q[i] = to_f32(q[lane + 32 * i]) * a.scale;
    r.o[i] = 0.f;
  }
  for (int p = 0; p < (int)a.prefix_len; p += P)
    r.add_page(a, a.prefix_pages[p >> a.page_shift], h, min(P, (int)a.prefix_len - p), lane);
  const int32_t* table = a.kv.page_table + (long long)s * a.kv.table_stride;
  if (a.list) {
    const int32_t* list = a.list + ((long long)s * a.kv.n_kv_heads + h) * a.n_list;
    for (int i = 0; i < a.n_list; ++i) {
      const int c = list[i];
      if (c == -1) continue;
      if (c < 0 || c >= (int)a.kv.max_pages) {
        if (lane == 0) raise_error(a.err, kDevBadArgument);
        continue;
      }
      if (c * P < L) r.add_page(a, table[c], h, min(P, L - c * P), lane);
    }
  } else {
    for (int p = 0; p < L; p += P) r.add_page(a, table[p >> a.page_shift], h, min(P, L - p), lane);
  }
  T* out = reinterpret_cast<T*>(a.out) + s * a.out_stride + head * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    out[lane + 32 * i] = from_f32<T>(r.l > 0.f ? r.o[i] / r.l : 0.f);
  if (a.lse && lane == 0) a.lse[(long long)s * a.n_heads + head] = r.m + logf(r.l);
}

}  // namespace

int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
  const dim3 grid(a.n_heads, a.kv.n_seq);
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16)
    d64 ? k_paged_attention<__half, 64><<<grid, 32, 0, st>>>(a)
        : k_paged_attention<__half, 128><<<grid, 32, 0, st>>>(a);
  else
    d64 ? k_paged_attention<__nv_bfloat16, 64><<<grid, 32, 0, st>>>(a)
        : k_paged_attention<__nv_bfloat16, 128><<<grid, 32, 0, st>>>(a);
  return 0;
}

}  // namespace qwen
