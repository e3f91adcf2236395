// paged_q4_append.cu -- rotation of new queries and keys at given positions, the keys'
// and values' way into a 4-bit paged cache, and its rows' way back into 16 bits.
#include "paged_q4.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kThreads = 128;

// Rows of sequence s and its length; false (reported) where they do not fit.
__device__ __forceinline__ bool rows_of(const qwen_paged_kv_q4& kv, const uint32_t* seq_len, const int32_t* cu,
                                        int n_rows, int* err, int s, int* row0, int* row1, int* L) {
  *row0 = cu[s];
  *row1 = cu[s + 1];
  *L = 0;
  bool ok = *row0 >= 0 && *row1 >= *row0 && *row1 <= n_rows;
  if (ok && *row1 > *row0) {
    const uint32_t len = seq_len[s];
    *L = (int)len;
    ok = len <= q4_capacity(kv) && *L >= *row1 - *row0;
  }
  if (!ok) raise_error(err, kDevBadArgument);
  return ok;
}
// Sequence and slot of a row (a token, or a row read back); false: the row is no one's.
__device__ __forceinline__ bool find_row(const qwen_paged_kv_q4& kv, const uint32_t* seq_len, const int32_t* cu,
                                         int n_rows, int* err, int row, int* seq, int* slot) {
  if (row >= n_rows) return false;
  if (!cu) {
    const uint32_t len = seq_len[row];
    if (len > q4_capacity(kv)) raise_error(err, kDevBadArgument);
    if (len == 0 || len > q4_capacity(kv)) return false;
    *seq = row;
    *slot = (int)len - 1;
    return true;
  }
  int lo = 0, hi = (int)kv.n_seq - 1;   // the first s with cu[s + 1] > row
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > row) hi = mid;
    else lo = mid + 1;
  }
  int row0, row1, L;
  if (!rows_of(kv, seq_len, cu, n_rows, err, lo, &row0, &row1, &L) || row < row0 || row >= row1) return false;
  *seq = lo;
  *slot = L - (row1 - row);
  return true;
}

struct Token {
  int seq, slot, page;   // seq -1: no one's row; page -1: outside the pool
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack2(T{}, w.x), b = unpack2(T{}, w.y), c = unpack2(T{}, w.z), d = unpack2(T{}, w.w);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2(T{}, x[0], x[1]), pack2(T{}, x[2], x[3]), pack2(T{}, x[4], x[5]), pack2(T{}, x[6], x[7]));
}
// x rounded to the cache's type.
template <typename T>
__device__ __forceinline__ void round8(float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 r = unpack2(T{}, pack2(T{}, x[i], x[i + 1]));
    x[i] = r.x;
    x[i + 1] = r.y;
  }
}

// kTile tokens a CTA; D / 8 lanes a head's row, 8 elements each.
template <typename T, int D, bool kInterleaved, int kTile>
__global__ void __launch_bounds__(kThreads) k_append_q4(const __grid_constant__ Q4AppendArgs a) {
  constexpr int NC = D / 8;
  __shared__ double2 rot[kTile][D / 2];   // cos, sin
  __shared__ Token tok[kTile];
  const int tid = threadIdx.x, H = a.n_heads, K = a.kv.n_kv_heads, R = a.rot_dim;
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();
  if (tid < kTile) {
    Token t;
    t.seq = t.slot = t.page = -1;
    int s, slot;
    if (find_row(a.kv, a.seq_len, a.cu_tokens, a.n_tokens, a.err, blockIdx.x * kTile + tid, &s, &slot)) {
      t.seq = s;
      t.slot = slot;
      t.page = q4_page(a.kv, a.err, s, slot >> a.page_shift);
    }
    tok[tid] = t;
  }
  __syncthreads();
  for (int i = tid; i < kTile * (R / 2); i += kThreads) {
    const int t = i / (R / 2), pair = i - t * (R / 2);
    if (tok[t].seq < 0) continue;
    int axis = a.pair_axis ? a.pair_axis[pair] : 0;
    if (axis >= a.n_axes) {
      raise_error(a.err, kDevBadArgument);
      axis = 0;
    }
    const int pos = a.positions ? a.positions[axis * a.position_stride + blockIdx.x * kTile + t] : tok[t].slot;
    double sn, cs;
    sincos((double)pos * (double)a.inv_freq[pair], &sn, &cs);
    rot[t][pair] = make_double2(cs, sn);
  }
  __syncthreads();
  const int rows = kTile * (H + 2 * K), c = tid % NC;
  const int first = tid / NC;
  for (int base = 0; base < rows; base += kThreads / NC) {   // (the warp's lanes stay together)
    const int i = base + first, t = min(i / (H + 2 * K), kTile - 1), head = i - t * (H + 2 * K);
    const bool live = i < rows && tok[t].seq >= 0;
    const long long row = (long long)blockIdx.x * kTile + t;
    const bool is_q = head < H, is_k = !is_q && head < H + K;
    float x[8] = {};
    if (live) {
      const T* src = is_q ? reinterpret_cast<const T*>(a.q) + row * a.q_stride + head * D
                     : is_k ? reinterpret_cast<const T*>(a.k) + row * a.k_stride + (head - H) * D
                            : reinterpret_cast<const T*>(a.v) + row * a.v_stride + (head - H - K) * D;
      load8(src + 8 * c, x);
      if ((is_q || is_k) && 8 * c < R) {
        float y[8];
        const bool second = !kInterleaved && 8 * c >= R / 2;
        const int first_pair = kInterleaved ? 4 * c : 8 * c - (second ? R / 2 : 0);
        if constexpr (!kInterleaved) load8(src + (second ? 8 * c - R / 2 : 8 * c + R / 2), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double2 r = rot[t][first_pair + (kInterleaved ? e / 2 : e)];
          const bool two = kInterleaved ? e & 1 : second;
          const float mate = kInterleaved ? x[e ^ 1] : y[e];
          float z;
          if (is_k) z = (float)(two ? (double)mate * r.y + (double)x[e] * r.x : (double)x[e] * r.x - (double)mate * r.y);
          else z = two ? mate * (float)r.y + x[e] * (float)r.x : x[e] * (float)r.x - mate * (float)r.y;
          if constexpr (kInterleaved) {
            y[e] = z;
          } else {
            x[e] = z;
          }
        }
        if constexpr (kInterleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = y[e];
        }
        if (is_k) round8<T>(x);
      }
    }
    if (live && is_q) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.q_out) + row * a.q_out_stride + head * D + 8 * c) = pack8<T>(x);
    if (!__any_sync(0xffffffffu, live && !is_q)) continue;
    uint32_t params;
    const uint32_t codes = quantise_group<T>(x, &params);
    if (!live || is_q || tok[t].page < 0) continue;
    const int h = is_k ? head - H : head - H - K, slot = tok[t].slot, in_page = slot & ((int)a.kv.page_size - 1);
    uint8_t* block = q4_block<D>(a.kv, tok[t].page, h, in_page);
    const int g = c / 4, r = in_page & 15;
    *reinterpret_cast<uint32_t*>(block + (is_k ? 0 : Q4Block<D>::kValues) + g * 256 + r * 16 + (c & 3) * 4) = codes;
    if ((c & 3) == 0)
      *reinterpret_cast<uint32_t*>(block + (is_k ? Q4Block<D>::kKeySteps : Q4Block<D>::kValueSteps) + g * 64 + r * 4) = params;
    if (is_k && c == 0) {
      const long long at = ((long long)tok[t].seq * K + h) * q4_capacity(a.kv) + slot;
      if (a.kv.weights) a.kv.weights[at] = 0.f;
      if (a.kv.positions) a.kv.positions[at] = a.positions ? a.positions[row] : slot;
    }
  }
}

template <typename T, int D, bool kInterleaved>
int launch(const Q4AppendArgs& a, cudaStream_t st) {
  if (!a.cu_tokens) k_append_q4<T, D, kInterleaved, 1><<<a.n_tokens, kThreads, 0, st>>>(a);
  else k_append_q4<T, D, kInterleaved, 8><<<(a.n_tokens + 7) / 8, kThreads, 0, st>>>(a);
  return 0;
}
template <typename T, int D>
int launch(const Q4AppendArgs& a, cudaStream_t st) {
  return a.interleaved ? launch<T, D, true>(a, st) : launch<T, D, false>(a, st);
}

// A CTA per row; D / 8 lanes a head's row of k or of v.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) k_expand_q4(const __grid_constant__ Q4ExpandArgs a) {
  constexpr int NC = D / 8;
  const int row = blockIdx.x, K = a.kv.n_kv_heads, c = threadIdx.x % NC;
  int s, slot;
  if (!find_row(a.kv, a.seq_len, a.cu_rows, a.n_rows, a.err, row, &s, &slot)) return;
  const int page = q4_page(a.kv, a.err, s, slot >> a.page_shift);
  if (page < 0) return;
  const int in_page = slot & ((int)a.kv.page_size - 1), g = c / 4, r = in_page & 15;
  for (int i = threadIdx.x / NC; i < 2 * K; i += kThreads / NC) {
    const bool is_k = i < K;
    const int h = is_k ? i : i - K;
    const uint8_t* block = q4_block<D>(a.kv, page, h, in_page);
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(block + (is_k ? 0 : Q4Block<D>::kValues) + g * 256 + r * 16 + (c & 3) * 4);
    const uint32_t params = *reinterpret_cast<const uint32_t*>(block + (is_k ? Q4Block<D>::kKeySteps : Q4Block<D>::kValueSteps) + g * 64 + r * 4);
    float x[8];
    expand_word<T>(codes, params, x);
    T* dst = reinterpret_cast<T*>(is_k ? a.k : a.v) + (long long)row * (is_k ? a.k_stride : a.v_stride) + h * D + 8 * c;
    *reinterpret_cast<uint4*>(dst) = pack8<T>(x);
  }
}

}  // namespace

int launch_rope_append_q4(const Q4AppendArgs& a, cudaStream_t st) {
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) return d64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return d64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}

int launch_expand_q4(const Q4ExpandArgs& a, cudaStream_t st) {
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) {
    if (d64) k_expand_q4<__half, 64><<<a.n_rows, kThreads, 0, st>>>(a);
    else k_expand_q4<__half, 128><<<a.n_rows, kThreads, 0, st>>>(a);
  } else {
    if (d64) k_expand_q4<__nv_bfloat16, 64><<<a.n_rows, kThreads, 0, st>>>(a);
    else k_expand_q4<__nv_bfloat16, 128><<<a.n_rows, kThreads, 0, st>>>(a);
  }
  return 0;
}

}  // namespace qwen
