// paged_append.cu -- rotation of new queries and keys, and the keys' and values'
// way into a paged cache.
//
//   y1 = x1 cos a - x2 sin a,  y2 = x1 sin a + x2 cos a,  a = position * inv_freq[i]
//
// One CTA per (sequence, page that its new tokens touch): it rotates those
// tokens' rows, writes them, and takes the keys into the page's bounds -- no
// other CTA touches that page, so the bounds need no atomics.  With ragged
// tokens the CTAs are numbered so that sequence s begins at
// cu_tokens[s] / page_size + 2 s: n tokens touch at most n / page_size + 2 pages.
//
// The angle is formed exactly (24 + 24 bits fit a double) and reduced to turns
// in 64 bits: an fp32 product at position 100,000 is off by up to 0.004 rad.
#include "paged_common.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kAppendThreads = 256;

__device__ __forceinline__ void sincos_of(float pos, float inv_freq, float* sn, float* cs) {
  const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;
  sincospif(2.0f * (float)(turns - rint(turns)), sn, cs);
}

// First sequence s with base(s + 1) > slot, base(s) = cu[s] / P + 2 s.
__device__ __forceinline__ int seq_of_slot(const int32_t* cu, int n_seq, int shift, int slot) {
  int lo = 0, hi = n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((cu[mid + 1] >> shift) + 2 * (mid + 1) > slot) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) k_rope_append(PagedAppendArgs a) {
  const int P = a.kv.page_size, H = a.n_heads, K = a.kv.n_kv_heads, R = a.rot_dim;
  int s, row0, n_new, index;
  if (a.cu_tokens) {
    s = seq_of_slot(a.cu_tokens, a.kv.n_seq, a.page_shift, blockIdx.x);
    row0 = a.cu_tokens[s];
    const int row1 = a.cu_tokens[s + 1];
    if (row0 < 0 || row1 < row0 || row1 > a.n_tokens) {
      if (threadIdx.x == 0) raise_error(a.err, kDevBadArgument);
      return;
    }
    n_new = row1 - row0;
    index = blockIdx.x - ((row0 >> a.page_shift) + 2 * s);
  } else {
    s = blockIdx.x;
    row0 = s;
    n_new = a.seq_len[s] > 0 ? 1 : 0;
    index = 0;
  }
  if (n_new == 0 || index < 0) return;
  bool ok;
  const int L = (int)checked_len(a.kv, a.seq_len, s, &ok);
  if (!ok || L < n_new) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadArgument);
    return;
  }
  const int start = L - n_new;
  const int col = (start >> a.page_shift) + index;
  const int p0 = max(start, col * P), p1 = min(L, (col + 1) * P);   // positions of this CTA
  if (p0 >= p1) return;
  const int page = a.kv.page_table[(long long)s * a.kv.table_stride + col];
  const bool in_pool = page >= 0 && (uint32_t)page < a.kv.n_pages;
  if (!in_pool && threadIdx.x == 0) raise_error(a.err, kDevBadArgument);
  const int n = p1 - p0;
  const long long row = row0 + (p0 - start);
  T* kc = reinterpret_cast<T*>(a.kv.k) + (long long)page * a.kv.page_stride;
  T* vc = reinterpret_cast<T*>(a.kv.v) + (long long)page * a.kv.page_stride;
  // rotated pairs, then what passes through, then the values
  for (int i = threadIdx.x; i < n * (H + K) * (R / 2); i += kAppendThreads) {
    const int pair = i % (R / 2), head = i / (R / 2) % (H + K), r = i / (R / 2) / (H + K);
    const int d1 = a.interleaved ? 2 * pair : pair, d2 = a.interleaved ? d1 + 1 : d1 + R / 2;
    float sn, cs;
    sincos_of((float)(p0 + r), a.inv_freq[pair], &sn, &cs);
    const T* x;
    T* y;
    if (head < H) {
      x = reinterpret_cast<const T*>(a.q) + (row + r) * a.q_stride + head * D;
      y = reinterpret_cast<T*>(a.q_out) + (row + r) * a.q_out_stride + head * D;
    } else {
      if (!in_pool) continue;
      x = reinterpret_cast<const T*>(a.k) + (row + r) * a.k_stride + (head - H) * D;
      y = kc + ((p0 + r) & (P - 1)) * a.kv.pos_stride + (head - H) * a.kv.head_stride;
    }
    const float x1 = to_f32(x[d1]), x2 = to_f32(x[d2]);
    y[d1] = from_f32<T>(x1 * cs - x2 * sn);
    y[d2] = from_f32<T>(x1 * sn + x2 * cs);
  }
  for (int i = threadIdx.x; i < n * (H + K) * (D - R); i += kAppendThreads) {
    const int d = R + i % (D - R), head = i / (D - R) % (H + K), r = i / (D - R) / (H + K);
    if (head < H)
      reinterpret_cast<T*>(a.q_out)[(row + r) * a.q_out_stride + head * D + d] =
          reinterpret_cast<const T*>(a.q)[(row + r) * a.q_stride + head * D + d];
    else if (in_pool)
      kc[((p0 + r) & (P - 1)) * a.kv.pos_stride + (head - H) * a.kv.head_stride + d] =
          reinterpret_cast<const T*>(a.k)[(row + r) * a.k_stride + (head - H) * D + d];
  }
  if (!in_pool) return;
  for (int i = threadIdx.x; i < n * K * D; i += kAppendThreads) {
    const int d = i % D, h = i / D % K, r = i / D / K;
    vc[((p0 + r) & (P - 1)) * a.kv.pos_stride + h * a.kv.head_stride + d] =
        reinterpret_cast<const T*>(a.v)[(row + r) * a.v_stride + h * D + d];
  }
  if (!a.kv.bounds) return;
  __syncthreads();   // the keys just written are read back below
  const bool anew = (p0 & (P - 1)) == 0;
  T* bounds = reinterpret_cast<T*>(a.kv.bounds) + (long long)page * 2 * K * D;
  for (int i = threadIdx.x; i < K * D; i += kAppendThreads) {
    const T* x = kc + (p0 & (P - 1)) * a.kv.pos_stride + (i / D) * a.kv.head_stride + i % D;
    T lo = anew ? x[0] : bounds[i], hi = anew ? x[0] : bounds[K * D + i];
    for (int r = 0; r < n; ++r) {
      lo = __hmin_nan(lo, x[r * a.kv.pos_stride]);
      hi = __hmax_nan(hi, x[r * a.kv.pos_stride]);
    }
    bounds[i] = lo;
    bounds[K * D + i] = hi;
  }
}

}  // namespace

int launch_rope_append(const PagedAppendArgs& a, cudaStream_t st) {
  const int grid = a.cu_tokens ? (a.n_tokens >> a.page_shift) + 2 * (int)a.kv.n_seq : (int)a.kv.n_seq;
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16)
    d64 ? k_rope_append<__half, 64><<<grid, kAppendThreads, 0, st>>>(a)
        : k_rope_append<__half, 128><<<grid, kAppendThreads, 0, st>>>(a);
  else
    d64 ? k_rope_append<__nv_bfloat16, 64><<<grid, kAppendThreads, 0, st>>>(a)
        : k_rope_append<__nv_bfloat16, 128><<<grid, kAppendThreads, 0, st>>>(a);
  return 0;
}

}  // namespace qwen
