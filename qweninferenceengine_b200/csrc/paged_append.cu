// paged_append.cu -- rotation of new queries and keys, and the keys' and values'
// way into a paged cache, in one launch.
//
//   y1 = x1 cos a - x2 sin a,  y2 = x1 sin a + x2 cos a,  a = position * inv_freq[i]
//
// Bound: HBM for prompts (each row read and written once), latency for a decode
// step.  9627 tokens of two prompts, 32 query and 8 kv heads of 128, bf16: 43.5 us,
// 5.4 TB/s; 256 single tokens 3.2 us.  A thread moves 16 elements of a head as two 16-byte loads and stores:
// chunk c is elements 8c.. and R/2 + 8c.. (the two sides of 8 pairs), or with
// interleaved pairs, and behind the rotated part of a head, elements 16c .. 16c+15.
//
// The angle is formed exactly (24 + 24 bits fit a double) and reduced to turns
// in 64 bits: an fp32 product at position 100,000 is off by up to 0.004 rad.  Its
// sine and cosine cost as much as rotating six heads by it, so prompts compute each
// once or a few times: k_append_rows' query CTAs keep eight of a thread's angles in
// registers for eight heads (sixteen took 18 us where eight took 15: it is the number of
// CTAs that hides the memory's latency), its key CTAs a page's in shared memory for four.
//
// Bounds: a key CTA owns two chunks of one page's new keys (all kv heads), so the
// least and greatest are reduced inside it: no atomics, and a page begun anew
// starts from its own keys.  The new rows of a sequence touch at most
// n / page_size + 2 pages; the key CTAs of sequence s are numbered from
// cu_tokens[s] / page_size + 2 s on.
#include "paged_common.cuh"
#include "paged_rotate.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kTokenThreads = 128;    // decode: a CTA per token
constexpr int kRowThreads = 128;      // prompts
constexpr int kHeads = 8;             // query or value heads of a CTA, in flight together
constexpr int kKeyHeads = 4;          // kv heads of a key CTA

__device__ __forceinline__ void rotation_of(const PagedAppendArgs& a, int pos, int c, float2 (&rot)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float sn, cs;
    sincos_of((float)pos, a.inv_freq[8 * c + i], &sn, &cs);
    rot[i] = make_float2(cs, sn);
  }
}

__device__ __forceinline__ uint32_t min2(__half, uint32_t a, uint32_t b) {
  const __half2 r = __hmin2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2(__half, uint32_t a, uint32_t b) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t min2(__nv_bfloat16, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2(__nv_bfloat16, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t inf2(__half) { return 0x7c007c00u; }
__device__ __forceinline__ uint32_t inf2(__nv_bfloat16) { return 0x7f807f80u; }

// The pool page of a table entry, or -1 with the status word set.
__device__ __forceinline__ int pool_page(const PagedAppendArgs& a, int s, int col) {
  const int page = a.kv.page_table[(long long)s * a.kv.table_stride + col];
  if (page >= 0 && (uint32_t)page < a.kv.n_pages) return page;
  raise_error(a.err, kDevBadArgument);
  return -1;
}

// One token per sequence: a CTA per token, a thread per (head, chunk).
template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kTokenThreads) k_append_token(const __grid_constant__ PagedAppendArgs a) {
  constexpr int NC = D / 16;
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int s = blockIdx.x, H = a.n_heads, K = a.kv.n_kv_heads, R = a.rot_dim;
  bool ok;
  const int L = (int)checked_len(a.kv, a.seq_len, s, &ok);
  if (L == 0) {
    if (!ok && threadIdx.x == 0) raise_error(a.err, kDevBadArgument);
    return;
  }
  const int pos = L - 1, slot = pos & (a.kv.page_size - 1);
  const int c = threadIdx.x % NC;   // the same for all of a thread's heads
  int pa, pb;
  places<kInterleaved>(c, R, &pa, &pb);
  float2 rot[8];
  const bool turns = 16 * c < R;
  if (turns) rotation_of(a, pos, c, rot);
  const int page = pool_page(a, s, pos >> a.page_shift);
  for (int head = threadIdx.x / NC; head < H + 2 * K; head += kTokenThreads / NC) {
    const T* src = head < H ? reinterpret_cast<const T*>(a.q) + s * a.q_stride + head * D
                   : head < H + K ? reinterpret_cast<const T*>(a.k) + s * a.k_stride + (head - H) * D
                                  : reinterpret_cast<const T*>(a.v) + s * a.v_stride + (head - H - K) * D;
    Chunk x = load_chunk(src + pa, src + pb);
    if (turns && head < H + K) rotate_chunk<T, kInterleaved>(x, rot);
    if (head < H) {
      T* dst = reinterpret_cast<T*>(a.q_out) + s * a.q_out_stride + head * D;
      store_chunk(dst + pa, dst + pb, x);
      continue;
    }
    if (page < 0) continue;
    const int h = head < H + K ? head - H : head - H - K;
    T* dst = reinterpret_cast<T*>(head < H + K ? a.kv.k : a.kv.v) + page * a.kv.page_stride + slot * a.kv.pos_stride +
             h * a.kv.head_stride;
    store_chunk(dst + pa, dst + pb, x);
    if (a.kv.bounds && head < H + K) {
      T* lo = reinterpret_cast<T*>(a.kv.bounds) + ((long long)page * 2 * K + h) * D;
      T* hi = lo + (long long)K * D;
      Chunk least = x, most = x;
      if (slot != 0) {
        const Chunk l0 = load_chunk(lo + pa, lo + pb), m0 = load_chunk(hi + pa, hi + pb);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          least.w[i] = min2(T{}, l0.w[i], x.w[i]);
          most.w[i] = max2(T{}, m0.w[i], x.w[i]);
        }
      }
      store_chunk(lo + pa, lo + pb, least);
      store_chunk(hi + pa, hi + pb, most);
    }
  }
}

// Rows of sequence s and its length; false (reported if `report`) where they do not fit.
__device__ __forceinline__ bool rows_of(const PagedAppendArgs& a, int s, bool report, int* row0, int* row1, int* L) {
  *row0 = a.cu_tokens[s];
  *row1 = a.cu_tokens[s + 1];
  bool ok = *row0 >= 0 && *row1 >= *row0 && *row1 <= a.n_tokens;
  if (ok && *row1 > *row0) {
    bool fits;
    *L = (int)checked_len(a.kv, a.seq_len, s, &fits);
    ok = fits && *L >= *row1 - *row0;
  }
  if (!ok && report) raise_error(a.err, kDevBadArgument);
  return ok;
}

// Ragged tokens.  CTAs 0 .. key_ctas - 1: chunks 2j, 2j+1 of the new keys of one page,
// or of the two or four whose rows make up 64; the rest: 8 query or value heads of
// kRowThreads / (D / 16) tokens.
template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kRowThreads, 4) k_append_rows(const __grid_constant__ PagedAppendArgs a, int key_ctas) {
  constexpr int NC = D / 16, kWarps = kRowThreads / 32;
  extern __shared__ float2 page_rot[];   // key CTA: [max(page_size, 64)][16]
  __shared__ uint32_t part[kKeyHeads][kWarps][32];
  const int H = a.n_heads, K = a.kv.n_kv_heads, R = a.rot_dim, P = a.kv.page_size, tid = threadIdx.x;
  const int n_seq = a.kv.n_seq, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();

  if ((int)blockIdx.x >= key_ctas) {
    // ------------------------------------------------------------- q and v --
    // The rows' elements are on their way while their sequence is looked up.
    const int q_parts = (H + kHeads - 1) / kHeads, parts = q_parts + (K + kHeads - 1) / kHeads;
    const int tile = ((int)blockIdx.x - key_ctas) / parts, part_no = (int)blockIdx.x - key_ctas - tile * parts;
    const bool is_q = part_no < q_parts;
    const int first = (is_q ? part_no : part_no - q_parts) * kHeads, count = min(kHeads, (is_q ? H : K) - first);
    const int row = tile * (kRowThreads / NC) + tid / NC, c = tid % NC;
    const bool there = row < a.n_tokens, turns = is_q && 16 * c < R;
    int pa = 16 * c, pb = 16 * c + 8;
    if (is_q) places<kInterleaved>(c, R, &pa, &pb);
    const T* src = (is_q ? reinterpret_cast<const T*>(a.q) + row * a.q_stride : reinterpret_cast<const T*>(a.v) + row * a.v_stride) + first * D;
    Chunk x[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j)
      if (there && j < count) x[j] = load_chunk(src + j * D + pa, src + j * D + pb);
    const int s = seq_of<NC>(a.cu_tokens, n_seq, 0, 0, row, lane);
    int row0, row1, L;
    if (!there || !rows_of(a, s, false, &row0, &row1, &L) || row < row0 || row >= row1) return;
    const int pos = L - (row1 - row);
    T* dst;
    long long stride = D;
    if (is_q) {
      dst = reinterpret_cast<T*>(a.q_out) + row * a.q_out_stride + first * D;
    } else {
      const int page = pool_page(a, s, pos >> a.page_shift);
      if (page < 0) return;
      stride = a.kv.head_stride;
      dst = reinterpret_cast<T*>(a.kv.v) + page * a.kv.page_stride + (pos & (P - 1)) * a.kv.pos_stride + first * stride;
    }
    float2 rot[8];
    if (turns) rotation_of(a, pos, c, rot);
#pragma unroll
    for (int j = 0; j < kHeads; ++j)
      if (j < count) {
        if (turns) rotate_chunk<T, kInterleaved>(x[j], rot);
        store_chunk(dst + j * stride + pa, dst + j * stride + pb, x[j]);
      }
    return;
  }

  // ------------------------------------------------------------------ keys --
  // A warp has 16 rows of one page; page_warps warps share a page of up to 64 rows, and
  // go on in steps of 64 through a larger one.
  const int page_warps = min(P / 16, kWarps), sub = warp / page_warps;
  const int splits = (K + kKeyHeads - 1) / kKeyHeads;   // CTAs by kv heads
  const int pair = blockIdx.x % (D / 32), rest = blockIdx.x / (D / 32);
  const int slot = rest / splits * (kWarps / page_warps) + sub;
  const int hb = rest % splits * kKeyHeads, he = min(K, hb + kKeyHeads);
  const int s = seq_of<32>(a.cu_tokens, n_seq, a.page_shift, 2, slot, lane);
  int row0 = 0, row1 = 0, L = 0, n = 0, p0 = 0, start = 0, page = -1;   // positions p0 .. p0 + n - 1
  if (rows_of(a, s, lane == 0, &row0, &row1, &L) && row1 > row0) {
    const int index = slot - ((row0 >> a.page_shift) + 2 * s);
    start = L - (row1 - row0);
    const int col = (start >> a.page_shift) + index;
    p0 = max(start, col * P);
    if (index >= 0) n = max(0, min(L, (col + 1) * P) - p0);
    if (n > 0) page = pool_page(a, s, col);
    if (page < 0) n = 0;
  }
  const int c = 2 * pair + (lane & 1), group_tid = tid - sub * page_warps * 32, r0 = group_tid >> 1;
  int pa, pb;
  places<kInterleaved>(c, R, &pa, &pb);
  const bool turns = 16 * c < R;
  float2* my_rot = page_rot + sub * P * 16;   // the angles of the page's chunks: 16 a row
#pragma unroll 4
  for (int i = group_tid; i < n * 16; i += page_warps * 32) {
    const int f = 16 * pair + (i & 15);
    if (f < R / 2) {
      float sn, cs;
      sincos_of((float)(p0 + (i >> 4)), a.inv_freq[f], &sn, &cs);
      my_rot[i] = make_float2(cs, sn);
    }
  }
  __syncthreads();
  const bool anew = (p0 & (P - 1)) == 0;
  const T* k = reinterpret_cast<const T*>(a.k) + (long long)(row0 + (p0 - start)) * a.k_stride;
  T* dst = reinterpret_cast<T*>(a.kv.k) + (long long)max(page, 0) * a.kv.page_stride + (p0 & (P - 1)) * a.kv.pos_stride;
  {
#pragma unroll 1
    for (int h = hb; h < he; ++h) {
      uint32_t least[8], most[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        least[i] = inf2(T{});
        most[i] = inf2(T{}) | 0x80008000u;
      }
      constexpr int kAtOnce = 4, kStep = kRowThreads / 2;   // rows of a thread in flight, and between them
#pragma unroll 1
      for (int r = r0; r < n; r += kAtOnce * kStep) {
        Chunk x[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
          if (r + j * kStep < n) {
            const T* src = k + (r + j * kStep) * a.k_stride + h * D;
            x[j] = load_chunk(src + pa, src + pb);
          }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int row = r + j * kStep;
          if (row >= n) break;
          if (turns) {
            float2 rot[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 v = reinterpret_cast<const float4*>(my_rot + 16 * row + 8 * (c & 1))[i];
              rot[2 * i] = make_float2(v.x, v.y);
              rot[2 * i + 1] = make_float2(v.z, v.w);
            }
            rotate_chunk<T, kInterleaved>(x[j], rot);
          }
          T* y = dst + row * a.kv.pos_stride + h * a.kv.head_stride;
          store_chunk(y + pa, y + pb, x[j]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            least[i] = min2(T{}, least[i], x[j].w[i]);
            most[i] = max2(T{}, most[i], x[j].w[i]);
          }
        }
      }
      if (!a.kv.bounds) continue;
      // Over the warp's 16 rows, halving what a lane keeps at each exchange: in the end
      // bit 4 of the lane says least or most, bits 3, 2, 1 which word, bit 0 the chunk.
      uint32_t v[8];
      const bool up = lane & 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, up ? least[i] : most[i], 16);
        v[i] = up ? max2(T{}, most[i], other) : min2(T{}, least[i], other);
      }
#pragma unroll
      for (int o = 8; o >= 2; o >>= 1) {
        const int keep = o / 2;
#pragma unroll
        for (int i = 0; i < keep; ++i) {
          const bool odd = lane & o;
          const uint32_t mine = odd ? v[keep + i] : v[i];
          const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[keep + i], o);
          v[i] = up ? max2(T{}, mine, other) : min2(T{}, mine, other);
        }
      }
      part[h - hb][warp][lane] = v[0];
    }
    if (!a.kv.bounds) return;
    __syncthreads();
    // A page's warps take its heads in turn.
    for (int h = hb + warp % page_warps; h < he && n > 0; h += page_warps) {
      const bool up = lane & 16;
      const int word = (lane >> 1) & 7;   // of the chunk's eight
      uint32_t v = part[h - hb][sub * page_warps][lane];
#pragma unroll 1
      for (int w = 1; w < page_warps; ++w) {
        const uint32_t other = part[h - hb][sub * page_warps + w][lane];
        v = up ? max2(T{}, v, other) : min2(T{}, v, other);
      }
      T* at = reinterpret_cast<T*>(a.kv.bounds) + (((long long)page * 2 + (up ? 1 : 0)) * K + h) * D +
              (word < 4 ? pa + 2 * word : pb + 2 * (word - 4));
      if (!anew) {
        const uint32_t old = *reinterpret_cast<const uint32_t*>(at);
        v = up ? max2(T{}, v, old) : min2(T{}, v, old);
      }
      *reinterpret_cast<uint32_t*>(at) = v;
    }
  }
}

template <typename T, int D, bool kInterleaved>
int launch(const PagedAppendArgs& a, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!a.cu_tokens) {
    cfg.gridDim = dim3(a.kv.n_seq);
    cfg.blockDim = dim3(kTokenThreads);
    return cudaLaunchKernelEx(&cfg, k_append_token<T, D, kInterleaved>, a) == cudaSuccess ? 0 : -1;
  }
  const int per_cta = a.kv.page_size >= 64 ? 1 : 64 / (int)a.kv.page_size;   // pages
  const int slots = (a.n_tokens >> a.page_shift) + 2 * (int)a.kv.n_seq;
  const int key_ctas = (slots + per_cta - 1) / per_cta * (D / 32) * (((int)a.kv.n_kv_heads + kKeyHeads - 1) / kKeyHeads);
  constexpr int kTileRows = kRowThreads / (D / 16);
  const int parts = (a.n_heads + kHeads - 1) / kHeads + ((int)a.kv.n_kv_heads + kHeads - 1) / kHeads;
  cfg.gridDim = dim3(key_ctas + (a.n_tokens + kTileRows - 1) / kTileRows * parts);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = (size_t)(a.kv.page_size < 64 ? 64 : a.kv.page_size) * 16 * sizeof(float2);
  return cudaLaunchKernelEx(&cfg, k_append_rows<T, D, kInterleaved>, a, key_ctas) == cudaSuccess ? 0 : -1;
}

template <typename T, int D>
int launch(const PagedAppendArgs& a, cudaStream_t st) {
  return a.interleaved ? launch<T, D, true>(a, st) : launch<T, D, false>(a, st);
}

}  // namespace

int launch_rope_append(const PagedAppendArgs& a, cudaStream_t st) {
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) return d64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return d64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}

}  // namespace qwen
