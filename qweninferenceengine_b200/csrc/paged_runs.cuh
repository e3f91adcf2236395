// paged_runs.cuh -- runs of tiles and the join of the pieces they cut, for the decode
// kernels over 16-bit (paged_decode.cu, which explains the protocol) and 4-bit pages.
#pragma once
#include "paged_common.cuh"

namespace qwen {
namespace {

constexpr int kJoin = 16;                     // partials joined at once

// A piece that a run leaves of a unit it shares with others.
struct CutUnit : CutPiece {
  int seq, head, heads;
  int unit;   // number in the launch
};

struct DecodeArgs {
  PagedAttnArgs a;
  int units_per_seq;        // kv heads x chunks of query heads (of a partial slot's number at most, S)
  int chunks;               // chunks per kv head
  int group;                // query heads per kv head
  int list_tiles;           // tiles of a listed unit
  int tile_shift;           // positions of a tile: 1 << tile_shift
  float scale_log2;
  float* part_o;            // [2 G][S][D], S the kernel's query heads of a unit: 16 (16-bit pages), 8 (4-bit)
  float* part_ml;           // [2 G][S][2]
  unsigned long long* arrived;   // [2 G] by partial slot, then [units]: tag << 16 | arrivals
  unsigned long long tag;
  float* own_o;             // if set: unnormalised rows [n_seq][n_heads][D] and their (max,
  float2* own_ml;           //   sum) go here instead of outputs, for the shared-prefix join
  uint32_t few_tiles = 0;   // up to so many tiles are divided among `few` CTAs only (no tiles at all: a call
  int few = 1;              // of lengths beyond the table alone; the number of runs is divided by)
};

__device__ __forceinline__ uint32_t seq_tiles(const DecodeArgs& p, uint32_t L) {
  if (p.a.list) return p.list_tiles;
  if (L > p.a.kv.max_pages * p.a.kv.page_size) return 0;
  return L ? ((L - 1) >> p.tile_shift) + 1 : 1;   // an empty sequence still has its zeros written
}

// Total number of tiles, the number G of runs, and the sequence that holds tile
// run_start(total, c) with its length and the number of tiles before it (one warp).
__device__ __forceinline__ uint32_t find_run(const DecodeArgs& p, uint32_t c, uint32_t& G, int lane, int* seq,
                                             uint32_t* before, uint32_t* length) {
  const int n_seq = p.a.kv.n_seq;
  const uint32_t u = p.units_per_seq;
  if (p.a.list) {
    const uint32_t total = u * p.list_tiles * n_seq;
    *seq = min((int)(run_start(total, c, G) / (u * p.list_tiles)), n_seq - 1);
    *before = (uint32_t)*seq * u * p.list_tiles;
    *length = p.a.seq_len[*seq];
    return total;
  }
  const int per = (n_seq + 31) / 32, s0 = min(n_seq, lane * per), s1 = min(n_seq, s0 + per);
  uint32_t sum = 0, L = 0;
  bool bad = false;
  if (per == 1) {
    if (lane < n_seq) {
      L = p.a.seq_len[lane];
      sum = seq_tiles(p, L);
      bad = sum == 0;
    }
  } else {
#pragma unroll 1
    for (int s = s0; s < s1; s += 4) {   // four lengths a round trip
      uint32_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = p.a.seq_len[min(s + j, s1 - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t t = seq_tiles(p, x[j]);
        if (s + j < s1) sum += t;
        bad |= t == 0;
      }
    }
  }
  if (bad && c == 0) raise_error(p.a.err, kDevBadArgument);   // (by both producers)
  uint32_t inc = sum * u;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  const uint32_t total = __shfl_sync(0xffffffffu, inc, 31);
  if (total <= p.few_tiles) G = p.few;
  const uint32_t target = run_start(total, c, G);
  uint32_t at = inc - sum * u;
  const uint32_t mine = __ballot_sync(0xffffffffu, target >= at && target < inc);
  int s = s0;
  if (per > 1 && mine >> lane & 1) {
#pragma unroll 1
    for (;; ++s) {
      L = p.a.seq_len[s];
      const uint32_t t = seq_tiles(p, L) * u;
      if (target < at + t) break;
      at += t;
    }
  }
  const int from = mine ? __ffs(mine) - 1 : 0;   // none: the run is empty
  *seq = __shfl_sync(0xffffffffu, s, from);
  *before = __shfl_sync(0xffffffffu, at, from);
  *length = __shfl_sync(0xffffffffu, L, from);
  return total;
}

// A finished row: output and log-sum-exp, or for the shared-prefix join what they
// are made of.
template <typename T, int D, bool kOwn>
__device__ __forceinline__ void finish_row(const DecodeArgs& p, int seq, int head, float4 v, float M, float sum, int lane) {
  if constexpr (!kOwn) {
    write_row<T, D>(p.a, seq, head, v, M, sum, lane);
    return;
  }
  const long long row = (long long)seq * p.a.n_heads + head;
  if constexpr (D == 128) reinterpret_cast<float4*>(p.own_o)[row * 32 + lane] = v;
  else reinterpret_cast<float2*>(p.own_o)[row * 32 + lane] = make_float2(v.x, v.y);
  if (lane == 0) p.own_ml[row] = make_float2(M, sum);
}
// The same into a partial slot (in units of heads).
template <int D>
__device__ __forceinline__ void store_partial(const DecodeArgs& p, int at, float4 v, float M, float sum, int lane) {
  if constexpr (D == 128) reinterpret_cast<float4*>(p.part_o)[(long long)at * 32 + lane] = v;
  else reinterpret_cast<float2*>(p.part_o)[(long long)at * 32 + lane] = make_float2(v.x, v.y);
  if (lane == 0) reinterpret_cast<float2*>(p.part_ml)[at] = make_float2(M, sum);
}
// Joins n <= 32 partials of every head of a unit, pieces first, first + step, .. (kWarps
// warps, two heads of each at a time so that their loads are one round trip; eight
// pieces at a time instead of four: single sequences -0.2 us, batches +0.6): into the
// output rows, or into the first piece's slot.
template <typename T, int D, bool kOwn, int kSlotHeads, int kWarps>
__device__ __forceinline__ void join_pieces(const DecodeArgs& p, const CutUnit& u, int G, int first, int step, int n, bool final,
                            int warp, int lane) {
  constexpr int V = D / 32, HB = 2;
  const int slot = lane < n ? piece_slot(u, first + lane * step, G) * kSlotHeads : 0;
#pragma unroll 1
  for (int h0 = warp; h0 < u.heads; h0 += HB * kWarps) {
    float2 ml[HB];
    float v[HB][V], f[HB], M[HB], sum[HB];
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int hh = min(h0 + b * kWarps, u.heads - 1);
      ml[b] = make_float2(-INFINITY, 0.f);
      if (lane < n) ml[b] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot + hh);
#pragma unroll
      for (int k = 0; k < V; ++k) v[b][k] = 0.f;
    }
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 4) {
      float x[4][HB][V];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long at = __shfl_sync(0xffffffffu, slot, min(i0 + i, n - 1));
#pragma unroll
        for (int b = 0; b < HB; ++b)
          load_vec(x[i][b], p.part_o + (at + min(h0 + b * kWarps, u.heads - 1)) * D + V * lane);
      }
      if (i0 == 0) {
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          M[b] = warp_max(ml[b].x);
          f[b] = ml[b].x == -INFINITY ? 0.f : exp2_fast(ml[b].x - M[b]);
          sum[b] = warp_sum(ml[b].y * f[b]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          const float fi = __shfl_sync(0xffffffffu, f[b], (i0 + i) & 31);
          if (i0 + i < n) {
#pragma unroll
            for (int k = 0; k < V; ++k) v[b][k] += x[i][b][k] * fi;
          }
        }
    }
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int hh = h0 + b * kWarps;
      if (hh >= u.heads) continue;
      if (final) finish_row<T, D, kOwn>(p, u.seq, u.head + hh, as_float4(v[b]), M[b], sum[b], lane);
      else store_partial<D>(p, __shfl_sync(0xffffffffu, slot, 0) + hh, as_float4(v[b]), M[b], sum[b], lane);
    }
  }
}
// Makes a count this call's, at 0, unless another CTA did.
__device__ __noinline__ void open_count(unsigned long long* count, unsigned long long tag) {
  const unsigned long long old = *(volatile unsigned long long*)count;
  if (old >> 16 != tag) atomicCAS(count, old, tag << 16);
}
__device__ __forceinline__ unsigned long long add_acq_rel(unsigned long long* p, unsigned long long x) {
  unsigned long long old;
  asm volatile("atom.add.acq_rel.gpu.global.u64 %0, [%1], %2;" : "=l"(old) : "l"(p), "l"(x) : "memory");
  return old;
}
__device__ __forceinline__ unsigned long long cas_acq_rel(unsigned long long* p, unsigned long long was,
                                                          unsigned long long x) {
  unsigned long long old;
  asm volatile("atom.cas.acq_rel.gpu.global.b64 %0, [%1], %2, %3;" : "=l"(old) : "l"(p), "l"(was), "l"(x) : "memory");
  return old;
}
// Counts an arrival; true for the last of `expected`, which leaves the count at 0.  What
// the CTA wrote before its last barrier is released, what the others wrote acquired, by
// the addition itself (fences around it, and one behind the store of the 0, took 0.3 to
// 0.8 us more of a call).
__device__ __noinline__ bool arrive_last(unsigned long long* count, unsigned long long tag, int expected) {
  unsigned long long now = add_acq_rel(count, 1ull) + 1;
  while (now >> 16 != tag) {   // not opened yet: what was there is another call's
    const unsigned long long seen = cas_acq_rel(count, now, tag << 16 | 1);
    if (seen == now) now = tag << 16 | 1;
    else now = seen >> 16 == tag ? add_acq_rel(count, 1ull) + 1 : seen;
  }
  const bool last = (int)(now & 0xffff) == expected;
  if (last) *(volatile unsigned long long*)count = tag << 16;
  return last;
}

// Arrival of a piece at the first level of its join.
__device__ __forceinline__ int arrive_first(const DecodeArgs& p, const CutUnit& u, int G) {
  const int first = u.piece / kJoin * kJoin;
  return arrive_last(u.pieces <= kJoin ? p.arrived + 2 * G + u.unit : p.arrived + piece_slot(u, first, G), p.tag,
                     min(kJoin, u.pieces - first));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}

}  // namespace
}  // namespace qwen
