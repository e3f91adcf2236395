// paged_q4_append.cu -- rotation of new queries and keys at given positions, the keys'
// and values' way into a 4-bit paged cache, and its rows' way back into 16 bits.
//
//   y1 = x1 cos a - x2 sin a,  y2 = x1 sin a + x2 cos a,  a = position[axis of i] inv_freq[i]
//   low = min, step = (max - min) / 15, code = (x - low) / step of 32 elements each
//
// Keys are turned in 64 bits and rounded once, so that their codes are those of the formula;
// queries, which keep 16 bits, in fp32 from angles formed in 64.  A decode step's tokens are
// bound by latency (2.4 us for one, 3.1 for 64), prompts by instructions more than by HBM:
// 52,600 tokens of 12 and 2 heads, fp16, take 93 us where their bytes take 60, 9600 of 32 and 8
// heads, bf16, 48 for 32.
#include <algorithm>

#include "paged_q4.cuh"
#include "paged_rotate.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

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
struct Token {
  int seq, slot;    // seq -1: no one's row
  uint8_t* block;   // the slot's, of head 0; null: its page is outside the pool
};
template <int D>
__device__ __forceinline__ uint8_t* block_of(const qwen_paged_kv_q4& kv, int page, int slot) {
  return page < 0 ? nullptr : q4_block<D>(kv, page, 0, slot & ((int)kv.page_size - 1));
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2(T{}, x[0], x[1]), pack2(T{}, x[2], x[3]), pack2(T{}, x[4], x[5]), pack2(T{}, x[6], x[7]));
}
// 8 elements of a row, and of a key the 8 that theirs are turned with.
struct Raw {
  uint4 own, mate;
};
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const float2 a = unpack2(T{}, w.x), b = unpack2(T{}, w.y), c = unpack2(T{}, w.z), d = unpack2(T{}, w.w);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}
// Lane c of a row: elements 8 c .. 8 c + 7; turned: whether they are rotated.
template <typename T, bool kInterleaved>
__device__ __forceinline__ Raw load_raw(const T* row, int c, int R, bool turned) {
  Raw r;
  r.own = *reinterpret_cast<const uint4*>(row + 8 * c);
  if (!kInterleaved && turned) r.mate = *reinterpret_cast<const uint4*>(row + (8 * c >= R / 2 ? 8 * c - R / 2 : 8 * c + R / 2));
  return r;
}
// Where a pair's (cos, sin) stands in shared memory: lanes side by side read adjacent ones.
template <int D, bool kInterleaved>
__device__ __forceinline__ int rot_at(int pair) {
  constexpr int kOf = kInterleaved ? 4 : 8;   // pairs of a lane
  return pair % kOf * (D / 2 / kOf) + pair / kOf;
}
// Rotates in the arithmetic of A (double for keys, float for queries).
template <typename A, typename T, int D, bool kInterleaved>
__device__ __forceinline__ uint4 rotate_raw(const Raw& r, const double2* rot, int c, int R) {
  float own[8], mate[8], x[8];
  unpack8<T>(r.own, own);
  if constexpr (!kInterleaved) unpack8<T>(r.mate, mate);
  const bool second = !kInterleaved && 8 * c >= R / 2;
  const double2* at = rot + (kInterleaved ? c : c - (second ? R / 16 : 0));
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double2 cs = at[rot_at<D, kInterleaved>(kInterleaved ? e / 2 : e)];
    const bool two = kInterleaved ? e & 1 : second;
    const A a = (A)own[e], b = (A)(kInterleaved ? own[e ^ 1] : mate[e]), s = (A)(two ? cs.y : -cs.y);
    x[e] = (float)(a * (A)cs.x + b * s);
  }
  return pack8<T>(x);
}
// Rotates 16 elements of a key, chunk c, in 64 bits.  Interleaved: elements 8 c .. 8 c + 7 and D / 2
// + 8 c ..; else pairs 8 c .. 8 c + 7, the first of each in words 0 .. 3.
template <typename T, int D, bool kInterleaved>
__device__ __forceinline__ void rotate_key(Chunk& x, const double2* rot, int c, int R) {
  if constexpr (kInterleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = 8 * c + (i < 4 ? 0 : D / 2);
      if (at >= R) continue;
      const double2 cs = rot[rot_at<D, true>(at / 2 + i % 4)];
      const float2 v = unpack2(T{}, x.w[i]);
      const double a = v.x, b = v.y;
      x.w[i] = pack2(T{}, (float)(a * cs.x + b * -cs.y), (float)(b * cs.x + a * cs.y));
    }
  } else if (16 * c < R) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double2 r0 = rot[rot_at<D, false>(8 * c + 2 * i)], r1 = rot[rot_at<D, false>(8 * c + 2 * i + 1)];
      const float2 v = unpack2(T{}, x.w[i]), u = unpack2(T{}, x.w[4 + i]);
      const double a0 = v.x, a1 = v.y, b0 = u.x, b1 = u.y;
      x.w[i] = pack2(T{}, (float)(a0 * r0.x + b0 * -r0.y), (float)(a1 * r1.x + b1 * -r1.y));
      x.w[4 + i] = pack2(T{}, (float)(b0 * r0.x + a0 * r0.y), (float)(b1 * r1.x + a1 * r1.y));
    }
  }
}
// Quantises 8 values, a quarter of a group, whose others its neighbours have, and stores the codes
// and (once a group) the parameters (all 32 lanes; of those that are live, and not of others).
template <typename T>
__device__ __forceinline__ void store_quantised(const uint4& x, uint8_t* codes_at, uint8_t* params_at, int quarter, bool live) {
  uint32_t params;
  const uint32_t codes = quantise_group<T>(x, &params);
  if (!live) return;
  *reinterpret_cast<uint32_t*>(codes_at) = codes;
  if (quarter == 0) *reinterpret_cast<uint32_t*>(params_at) = params;
}
// Where a head's row of keys or values has the codes of lane c's 8 elements (of group c / 4),
// and that group's parameters, in slot 0 of a block of head 0.
template <int D>
__device__ __forceinline__ long long codes_from(const Q4AppendArgs& a, int h, bool is_k, int c) {
  return h * a.kv.head_stride + (is_k ? 0 : Q4Block<D>::kValues) + c / 4 * 256 + c % 4 * 4;
}
template <int D>
__device__ __forceinline__ long long params_from(const Q4AppendArgs& a, int h, bool is_k, int c) {
  return h * a.kv.head_stride + (is_k ? Q4Block<D>::kKeySteps : Q4Block<D>::kValueSteps) + c / 4 * 64;
}
__device__ __forceinline__ int axis_of(const Q4AppendArgs& a, int pair) {
  if (!a.pair_axis) return 0;
  const int axis = a.pair_axis[pair];
  if (axis < a.n_axes) return axis;
  raise_error(a.err, kDevBadArgument);
  return 0;
}
__device__ __forceinline__ int position_of(const Q4AppendArgs& a, int pair, int row, int slot) {
  return a.positions ? a.positions[axis_of(a, pair) * a.position_stride + row] : slot;
}
// What the cache keeps of the slot beside its key and value.
__device__ __forceinline__ void keep_slot(const Q4AppendArgs& a, const Token& t, int h, int row) {
  const long long at = ((long long)t.seq * a.kv.n_kv_heads + h) * q4_capacity(a.kv) + t.slot;
  if (a.kv.weights) a.kv.weights[at] = 0.f;
  if (a.kv.positions) a.kv.positions[at] = a.positions ? a.positions[row] : t.slot;
}

// One token per sequence: a CTA per token, D / 8 lanes a row.  A row's elements are on their
// way while length, page and angles are found.
constexpr int kTokenThreads = 256;
template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kTokenThreads) k_append_token_q4(const __grid_constant__ Q4AppendArgs a) {
  constexpr int NC = D / 8, kRows = kTokenThreads / NC;
  __shared__ double2 rot[D / 2];   // cos, sin
  const int tid = threadIdx.x, H = a.n_heads, K = a.kv.n_kv_heads, R = a.rot_dim, c = tid % NC, row = blockIdx.x;
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();
  auto source = [&](int head) {
    return head < H ? reinterpret_cast<const T*>(a.q) + row * a.q_stride + head * D
           : head < H + K ? reinterpret_cast<const T*>(a.k) + row * a.k_stride + (head - H) * D
                          : reinterpret_cast<const T*>(a.v) + row * a.v_stride + (head - H - K) * D;
  };
  int head = tid / NC;
  Raw next{};
  if (head < H + 2 * K) next = load_raw<T, kInterleaved>(source(head), c, R, 8 * c < R && head < H + K);
  Token t;
  t.seq = row;
  const uint32_t len = a.seq_len[row];
  if (len == 0 || len > q4_capacity(a.kv)) {
    if (len != 0 && tid == 0) raise_error(a.err, kDevBadArgument);
    return;
  }
  t.slot = (int)len - 1;
  const int entry = a.kv.page_table[(long long)row * a.kv.table_stride + (t.slot >> a.page_shift)];
  for (int pair = tid; pair < R / 2; pair += kTokenThreads) {
    double sn, cs;
    sincos((double)position_of(a, pair, row, t.slot) * (double)a.inv_freq[pair], &sn, &cs);
    rot[rot_at<D, kInterleaved>(pair)] = make_double2(cs, sn);
  }
  const bool there = entry >= 0 && (uint32_t)entry < a.kv.n_pages;
  t.block = block_of<D>(a.kv, there ? entry : -1, t.slot);
  if (!there && tid == 0) raise_error(a.err, kDevBadArgument);
  if (tid < K) keep_slot(a, t, tid, row);
  for (int h = tid + kTokenThreads; h < K; h += kTokenThreads) keep_slot(a, t, h, row);
  __syncthreads();
  for (int base = 0; base < H + 2 * K; base += kRows, head += kRows) {   // (the warp's lanes stay together)
    const bool live = head < H + 2 * K, is_q = head < H, is_k = !is_q && head < H + K;
    const Raw r = next;
    __syncwarp();   // q_out may be q: every lane has its mates before a row is written
    if (head + kRows < H + 2 * K)
      next = load_raw<T, kInterleaved>(source(head + kRows), c, R, 8 * c < R && head + kRows < H + K);
    uint4 x = r.own;
    if ((is_q || is_k) && 8 * c < R) {
      if (is_q) x = rotate_raw<float, T, D, kInterleaved>(r, rot, c, R);
      else x = rotate_raw<double, T, D, kInterleaved>(r, rot, c, R);
    }
    if (is_q) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.q_out) + row * a.q_out_stride + head * D + 8 * c) = x;
    if (__any_sync(0xffffffffu, live && !is_q)) {
      const int h = is_k ? head - H : head - H - K, r = t.slot & 15;
      store_quantised<T>(x, t.block + codes_from<D>(a, h, is_k, c) + r * 16, t.block + params_from<D>(a, h, is_k, c) + r * 4,
                         c & 3, live && !is_q && t.block);
    }
  }
}

// Ragged tokens.  CTAs 0 .. kv_ctas - 1: keys and values of up to 4 kv heads of 8 tokens, D / 16
// lanes a row; the rest: 4 query heads of 16 tokens (32 with head_dim 64), a thread 16
// elements of a token's heads, as in k_append_rows.  Both wait for memory and for one another's
// steps more than they compute, so that CTAs on an SM count for more than what a thread has in
// flight: 9632 tokens, 32 and 8 heads, pairs half a head apart: 8 CTAs with one row of a kv
// CTA's thread and 4 query heads at a time 56 us, 4 CTAs with 4 and 8 79 us.  Sixteen elements
// a thread share what a row's address, token and place cost (8: 56 us, 16: 50; with quotients in
// fixed point 46.5; 4 tokens a CTA, whose angles fill fewer lanes, 50; 16 tokens 51).
constexpr int kRowThreads = 128, kRowCtasPerSm = 8, kQHeads = 4, kKvTokens = 8, kKvHeads = 4;
template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kRowThreads, kRowCtasPerSm) k_append_rows_q4(const __grid_constant__ Q4AppendArgs a, int kv_ctas) {
  __shared__ double2 rot[kKvTokens][D / 2];   // cos, sin
  __shared__ Token tok[kKvTokens];
  __shared__ __align__(16) uint16_t stage[kRowThreads / (D / 16)][kInterleaved ? 8 : D];
  const int tid = threadIdx.x, lane = tid & 31, H = a.n_heads, K = a.kv.n_kv_heads, R = a.rot_dim, n_seq = a.kv.n_seq;
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();
  if ((int)blockIdx.x >= kv_ctas) {
    constexpr int NC = D / 16;
    const int parts = (H + kQHeads - 1) / kQHeads, cta = (int)blockIdx.x - kv_ctas, tile = cta / parts;
    const int first = (cta - tile * parts) * kQHeads, count = min(kQHeads, H - first);
    const int row = tile * (kRowThreads / NC) + tid / NC, c = tid % NC;
    const bool there = row < a.n_tokens;
    int pa, pb;
    places<kInterleaved>(c, R, &pa, &pb);
    const T* src = reinterpret_cast<const T*>(a.q) + row * a.q_stride + first * D;
    Chunk x[kQHeads];
#pragma unroll
    for (int j = 0; j < kQHeads; ++j)
      if (there && j < count) x[j] = load_chunk(src + j * D + pa, src + j * D + pb);
    const int s = seq_of<NC>(a.cu_tokens, n_seq, 0, 0, row, lane);
    int row0, row1, L;
    if (!there || !rows_of(a.kv, a.seq_len, a.cu_tokens, a.n_tokens, a.err, s, &row0, &row1, &L) || row < row0 || row >= row1)
      return;
    T* dst = reinterpret_cast<T*>(a.q_out) + row * a.q_out_stride + first * D;
    float2 turn[8];
    const bool turns = 16 * c < R;
    if (turns) {
      const int slot = L - (row1 - row), one = a.positions && !a.pair_axis ? a.positions[row] : slot;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float sn, cs;
        const int at = a.pair_axis ? position_of(a, 8 * c + i, row, slot) : one;
        const double turns = (double)at * (double)a.inv_freq[8 * c + i] * 0.15915494309189533577;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        turn[i] = make_float2(cs, sn);
      }
    }
#pragma unroll
    for (int j = 0; j < kQHeads; ++j)
      if (j < count) {
        if (turns) rotate_chunk<T, kInterleaved>(x[j], turn);
        store_chunk(dst + j * D + pa, dst + j * D + pb, x[j]);
      }
    return;
  }
  // A thread takes 16 elements of the rows of one kv head's keys or values, of every dt-th token.
  constexpr int NC = D / 16, kStep = kRowThreads / NC;   // rows at once
  const int parts = (K + kKvHeads - 1) / kKvHeads, tile = blockIdx.x / parts;
  const int first = ((int)blockIdx.x - tile * parts) * kKvHeads, heads = min(kKvHeads, K - first);
  const int c = tid % NC, row0 = tile * kKvTokens, tokens = min(kKvTokens, a.n_tokens - row0);
  const int lg = heads > 2 ? 2 : heads - 1, x = tid / NC & ((2 << lg) - 1), h = x & ((1 << lg) - 1), dt = kStep >> (lg + 1);
  const bool is_k = x >> lg == 0, live = h < heads, staged = !kInterleaved && R != D;
  int t = tid / NC >> (lg + 1), pa = 8 * c, pb = D / 2 + 8 * c;
  if (staged && is_k) places<false>(c, R, &pa, &pb);
  const long long stride = is_k ? a.k_stride : a.v_stride;
  const T* src = reinterpret_cast<const T*>(is_k ? a.k : a.v) + (row0 + t) * stride + (first + h) * D;
  const long long codes_at = codes_from<D>(a, first + h, is_k, c), params_at = params_from<D>(a, first + h, is_k, c);
  Chunk next{};
  if (live && t < tokens) next = load_chunk(src + pa, src + pb);
  if (tid < 32) {
    const int t = lane / (32 / kKvTokens), row = row0 + t;
    const int s = seq_of<32 / kKvTokens>(a.cu_tokens, n_seq, 0, 0, row, lane);
    Token x;
    x.seq = x.slot = -1;
    x.block = nullptr;
    int r0, r1, L;
    if (row < a.n_tokens && lane % (32 / kKvTokens) == 0 &&
        rows_of(a.kv, a.seq_len, a.cu_tokens, a.n_tokens, a.err, s, &r0, &r1, &L) && row >= r0 && row < r1) {
      x.seq = s;
      x.slot = L - (r1 - row);
      x.block = block_of<D>(a.kv, q4_page(a.kv, a.err, s, x.slot >> a.page_shift), x.slot);
    }
    if (lane % (32 / kKvTokens) == 0) tok[t] = x;
  }
  __syncthreads();
  const int pair = tid % (D / 2);
  if (pair < R / 2)
    for (int i = tid / (D / 2); i < tokens; i += kRowThreads / (D / 2)) {
      if (tok[i].seq < 0) continue;
      double sn, cs;
      sincos((double)position_of(a, pair, row0 + i, tok[i].slot) * (double)a.inv_freq[pair], &sn, &cs);
      rot[i][rot_at<D, kInterleaved>(pair)] = make_double2(cs, sn);
    }
  for (int i = tid; i < tokens * heads; i += kRowThreads)
    if (tok[i / heads].seq >= 0) keep_slot(a, tok[i / heads], first + i % heads, row0 + i / heads);
  __syncthreads();
#pragma unroll 1
  for (int base = 0; base < tokens; base += dt, t += dt) {   // (the warp's lanes stay together)
    Chunk now = next;
    src += dt * stride;
    if (live && t + dt < tokens) next = load_chunk(src + pa, src + pb);
    const Token& token = tok[min(t, tokens - 1)];
    const bool there = live && t < tokens;
    if (is_k && there && token.seq >= 0) rotate_key<T, D, kInterleaved>(now, rot[t], c, R);
    if (staged) {   // pairs R / 2 apart: to where the others have theirs
      T* row = reinterpret_cast<T*>(stage[tid / NC]);
      store_chunk(row + pa, row + pb, now);
      __syncwarp();
      now = load_chunk(row + 8 * c, row + D / 2 + 8 * c);
      __syncwarp();
    }
    uint8_t *codes = token.block + codes_at + (token.slot & 15) * 16, *params = token.block + params_at + (token.slot & 15) * 4;
    const bool stored = there && token.block;
    store_quantised<T>(make_uint4(now.w[0], now.w[1], now.w[2], now.w[3]), codes, params, c & 3, stored);
    store_quantised<T>(make_uint4(now.w[4], now.w[5], now.w[6], now.w[7]), codes + D / 64 * 256, params + D / 64 * 64, c & 3, stored);
  }
}

template <typename T, int D, bool kInterleaved>
int launch(const Q4AppendArgs& a, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!a.cu_tokens) {
    cfg.gridDim = dim3(a.n_tokens);
    cfg.blockDim = dim3(kTokenThreads);
    return cudaLaunchKernelEx(&cfg, k_append_token_q4<T, D, kInterleaved>, a) == cudaSuccess ? 0 : -1;
  }
  constexpr int kTileRows = kRowThreads / (D / 16);
  const int q_ctas = (a.n_tokens + kTileRows - 1) / kTileRows * ((a.n_heads + kQHeads - 1) / kQHeads);
  const int kv_ctas = (a.n_tokens + kKvTokens - 1) / kKvTokens * (((int)a.kv.n_kv_heads + kKvHeads - 1) / kKvHeads);
  cfg.gridDim = dim3(q_ctas + kv_ctas);
  cfg.blockDim = dim3(kRowThreads);
  return cudaLaunchKernelEx(&cfg, k_append_rows_q4<T, D, kInterleaved>, a, kv_ctas) == cudaSuccess ? 0 : -1;
}
template <typename T, int D>
int launch(const Q4AppendArgs& a, cudaStream_t st) {
  return a.interleaved ? launch<T, D, true>(a, st) : launch<T, D, false>(a, st);
}

// Rows back in 16 bits.  Bound: HBM, 160 B in and 512 out a row of K and V of 128.  A CTA has a
// run of rows, up to 64 of which it looks up at once, each in a thread (a lookup is a chain
// of four round trips: with 8 rows a CTA its warps spent most of their time behind it); then
// D / 8 lanes take a head's row of k or of v.
constexpr int kExpandRows = 64, kExpandThreads = 256, kExpandCtasPerSm = 8, kExpandLeast = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kExpandThreads, kExpandCtasPerSm) k_expand_q4(const __grid_constant__ Q4ExpandArgs a) {
  constexpr int NC = D / 8, kStep = kExpandThreads / NC, kAtOnce = 4;   // rows of a thread in flight
  struct Row {
    const uint8_t *codes, *params;   // of head 0; null: no one's row
  };
  __shared__ Row row_at[kExpandRows];
  const int tid = threadIdx.x, K = a.kv.n_kv_heads, n_seq = a.kv.n_seq;
  const int begin = (int)((long long)a.n_rows * blockIdx.x / gridDim.x);
  const int end = (int)((long long)a.n_rows * (blockIdx.x + 1) / gridDim.x);
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();
  int s0 = 0;   // sequence of the first row
  if (a.cu_rows)
    for (int base = 0; base < n_seq - 1; base += kExpandThreads)
      s0 += __syncthreads_count(base + tid < n_seq - 1 && a.cu_rows[base + tid + 1] <= begin);
  const int c = tid % NC, per = 2 * K, add_t = kStep / per, add_x = kStep - add_t * per;
  const int first_t = tid / NC / per, first_x = tid / NC - first_t * per;
#pragma unroll 1
  for (int row0 = begin; row0 < end; row0 += kExpandRows) {
    const int tokens = min(kExpandRows, end - row0);
    if (tid < tokens) {
      const int row = row0 + tid;
      int r0 = row, r1 = row + 1, L = 0, s = row;
      bool mine;
      if (a.cu_rows) {
        int hi = n_seq - 1;   // the first s with cu[s + 1] > row
        s = s0;
        if (s < hi && a.cu_rows[s + 1] > row) hi = s;
        while (s < hi) {
          const int mid = (s + hi) >> 1;
          if (a.cu_rows[mid + 1] > row) hi = mid;
          else s = mid + 1;
        }
        mine = rows_of(a.kv, a.seq_len, a.cu_rows, a.n_rows, a.err, s, &r0, &r1, &L) && row >= r0 && row < r1;
      } else {
        const uint32_t len = a.seq_len[row];
        mine = len != 0 && len <= q4_capacity(a.kv);
        if (len > q4_capacity(a.kv)) raise_error(a.err, kDevBadArgument);
        L = (int)len;
      }
      Row at = {nullptr, nullptr};
      if (mine) {
        const int slot = L - (r1 - row), page = q4_page(a.kv, a.err, s, slot >> a.page_shift);
        if (page >= 0) {
          const uint8_t* block = block_of<D>(a.kv, page, slot);
          at.codes = block + (slot & 15) * 16;
          at.params = block + Q4Block<D>::kKeySteps + (slot & 15) * 4;
        }
      }
      row_at[tid] = at;
    }
    __syncthreads();
    int t = first_t, x = first_x;   // row of the tile, key (x < K) or value of a head
#pragma unroll 1
    while (t < tokens) {
      uint32_t codes[kAtOnce], params[kAtOnce];
      T* to[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        to[j] = nullptr;
        if (t < tokens && row_at[t].codes) {
          const bool is_k = x < K;
          const int h = is_k ? x : x - K;
          const long long off = (long long)h * a.kv.head_stride + (c / 4) * 64;
          codes[j] = __ldg(reinterpret_cast<const uint32_t*>(row_at[t].codes + off + (is_k ? 0 : Q4Block<D>::kValues) + (c / 4) * 192 + (c & 3) * 4));
          params[j] = __ldg(reinterpret_cast<const uint32_t*>(row_at[t].params + off + (is_k ? 0 : Q4Block<D>::kValueSteps - Q4Block<D>::kKeySteps)));
          to[j] = reinterpret_cast<T*>(is_k ? a.k : a.v) + (long long)(row0 + t) * (is_k ? a.k_stride : a.v_stride) + h * D + 8 * c;
        }
        t += add_t;
        x += add_x;
        if (x >= per) {
          x -= per;
          ++t;
        }
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (to[j]) *reinterpret_cast<uint4*>(to[j]) = expand_word(T{}, codes[j], params[j]);
    }
    __syncthreads();
  }
}

template <typename T, int D>
int launch(const Q4ExpandArgs& a, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::min((a.n_rows + kExpandLeast - 1) / kExpandLeast, kExpandCtasPerSm * paged_sm_count()));
  cfg.blockDim = dim3(kExpandThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_expand_q4<T, D>, a) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_rope_append_q4(const Q4AppendArgs& a, cudaStream_t st) {
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) return d64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return d64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}

int launch_expand_q4(const Q4ExpandArgs& a, cudaStream_t st) {
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) return d64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return d64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}

}  // namespace qwen
