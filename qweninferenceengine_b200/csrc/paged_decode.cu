// paged_decode.cu -- decode attention over a paged cache, one query token per
// sequence, over all of a sequence's pages or over listed ones:
//   out = sum_t softmax(scale q . K_t) V_t
//
// Bound: HBM, each key and value read once (512 B a position and kv head of 128;
// group flops a byte).  So the kernel is a stream of pages through shared
// memory with just enough arithmetic beside it.  32 sequences of 16384 positions, 32
// query and 8 kv heads of 128: 325 us, 6.6 TB/s; of 64 sequences of 512 .. 2048
// positions and 2 kv heads the 79 MB take 12 us and the rest of its 22.6 us is latency:
// launch, lengths, page numbers, first tile, join, one after another (9 us in a call
// of 512 positions).
//
// Work: a unit is one (sequence, kv head, up to 16 query heads), a tile 64 positions
// of a unit (128 with head_dim 64).  All tiles of all units stand in one row, and CTA
// c of G (two per SM) takes an equal run of them, start(c) = c T / G, wherever units
// begin and end: a ragged batch, one long sequence and a batch of short ones all divide
// evenly.  A unit within one CTA is finished there; a unit cut by a run's end
// leaves fp32 partials (max, sum, unnormalised output), which are joined in run
// order whoever joins them, so results do not depend on timing.  A CTA counts in its
// pieces (two at most): the one its run began with while its last tiles are on their
// way, the one its run ends with at the end; the last to arrive at a unit joins up
// to 16 of them; of more, the last of each 16 joins those, and the last of the
// joined ones the rest (one CTA reading 148 partials of six heads would take as
// long as streaming 128K positions).  Nothing waits for another CTA, and a call's
// counts carry its own tag, so the workspace needs no zeroing.
//
// CTA: 4 consumer warps and two producer warps, one for K and one for V (a lane's TMA
// issue takes ~75 cycles and lanes take turns, so one warp with pages of 16 could not
// keep up).  Per tile a producer's lanes read list and page table (32 entries at a
// time) and issue one TMA load per box of 16 or 32 positions (a 5-D map over the
// pool, so any stride order; the 128-byte swizzle keeps fragment loads free of bank
// conflicts); K's also writes how many of each warp's 16 positions count.  Positions
// past a sequence's end and pages outside the pool are never loaded or, inside a box,
// masked in registers.
// Consumer warp w takes positions 16w..16w+15 (and 64 behind) of a tile on its own:
//   S^T[16 pos x 8 heads] = K q^T, the softmax, o^T[d x 8] += V^T P^T
// with m16n8k16 MMAs (8 = the heads that share the kv head; tcgen05's smallest
// M of 64 would be nine tenths padding), P^T turned by movmatrix.
// The running maximum moves only when a score passes it by 2^15 (a vote, no
// shuffles, in most tiles): weights are formed as 2^(s - r), r = max - 7 when last
// moved, which keeps them within fp16's normal range from 2^15 down to 2^-21 of
// the largest.  For the MMA a weight is two values of the cache's type, itself rounded
// and what that left (relative 2^-22 or 2^-16, as k_attention_decode's fp16 pair; the
// second product takes V without infinities, which the first has: 0 times one would be
// NaN); sums, maxima and outputs are fp32.  One value alone: 64 x 2048 22.6 us against
// 22.7, 64 x 4096 with 32 query heads of 64 a kv head, where the MMAs count most, 47.4
// against 51.9.  Beside a shared prefix, whose weights are one value, own positions' are too
// (64 x 8704: 34.5 us against 35.9).
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
#include <mutex>

#include "paged_common.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kWarps = 4;                      // consumer warps
// 16-position slices of a tile that a warp takes, and positions of a tile: 32 KB of K
// and V either way (a tile costs the producers ~500 cycles whatever its size).
constexpr int slices_of(int D) { return D == 64 ? 2 : 1; }
constexpr int tile_of(int D) { return 16 * kWarps * slices_of(D); }
constexpr int kThreads = (kWarps + 2) * 32;
constexpr int kCtasPerSm = 2;
constexpr int kMaxSlotHeads = 16;             // query heads of a unit
constexpr int kJoin = 16;                     // partials joined at once

enum StageFlags { kFirst = 1, kLast = 2, kEnd = 4 };

struct StageMeta {
  int valid[8];        // positions of each 16 that count
  int flags;
  int seq, head, heads;   // the unit: sequence, first query head, query heads
  int dest;            // partial slot, or -1: the whole unit, or -2: nothing is written
};

// A piece that a run leaves of a unit it shares with others.
struct CutUnit : CutPiece {
  int seq, head, heads;
  int unit;   // number in the launch
};

constexpr int kStages = 3;

// Queries in flight: of 16 heads two units', of 8 four.
template <int NT>
constexpr int query_slots() {
  return 4 / NT;
}

template <int D, int NT>
struct __align__(1024) DecodeSmem {
  uint8_t kv[kStages][2][tile_of(D) * D * 2];
  uint16_t q[query_slots<NT>()][8 * NT * D];
  float2 ml[2][kWarps][kMaxSlotHeads];   // by piece parity: maximum and sum of each warp
  StageMeta meta[kStages];
  uint64_t full[kStages], empty[kStages], qfull[query_slots<NT>()], qempty[query_slots<NT>()], joined, early;
  CutUnit cut[2];
  int n_cut, n_early;   // cut pieces; of those counted in before the end
  int runs;
  int last[2];
  int abort;
};

struct DecodeArgs {
  PagedAttnArgs a;
  int units_per_seq;        // kv heads x chunks of at most 16 query heads
  int chunks;               // chunks per kv head
  int group;                // query heads per kv head
  int list_tiles;           // tiles of a listed unit
  int tile_shift;           // positions of a tile: 1 << tile_shift
  float scale_log2;
  float* part_o;            // [2 G][16][D]
  float* part_ml;           // [2 G][16][2]
  unsigned long long* arrived;   // [2 G] by partial slot, then [units]: tag << 16 | arrivals
  unsigned long long tag;
  float* own_o;             // if set: unnormalised rows [n_seq][n_heads][D] and their (max,
  float2* own_ml;           //   sum) go here instead of outputs, for the shared-prefix join
  uint32_t few_tiles;       // up to so many tiles are divided among `few` CTAs only
  int few;
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
// Joins n <= 32 partials of every head of a unit, pieces first, first + step, .. (four
// warps, two heads of each at a time so that their loads are one round trip; eight
// pieces at a time instead of four: single sequences -0.2 us, batches +0.6): into the
// output rows, or into the first piece's slot.
template <typename T, int D, bool kOwn>
__device__ __forceinline__ void join_pieces(const DecodeArgs& p, const CutUnit& u, int G, int first, int step, int n, bool final,
                            int warp, int lane) {
  constexpr int V = D / 32, HB = 2;
  const int slot = lane < n ? piece_slot(u, first + lane * step, G) * kMaxSlotHeads : 0;
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

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
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

// NT: 8-head MMA columns of a unit (1 or 2).  kOwn: beside a kernel that reads a shared
// prefix (PagedOwn), and like it with weights rounded once.
template <typename T, int D, int NT, bool kOwn>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    k_paged_decode(const __grid_constant__ DecodeArgs p, int box_rows,
                   const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
  constexpr int ST = kStages, SL = slices_of(D), kTile = tile_of(D), QS = query_slots<NT>();
  extern __shared__ uint8_t smem_raw[];
  DecodeSmem<D, NT>& s = *reinterpret_cast<DecodeSmem<D, NT>*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const PagedAttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&s.full[i], 2);   // both producers
      mbar_init(&s.empty[i], kWarps);
    }
    for (int i = 0; i < QS; ++i) {
      mbar_init(&s.qfull[i], 1);
      mbar_init(&s.qempty[i], kWarps);
    }
    mbar_init(&s.joined, kWarps);
    mbar_init(&s.early, kWarps);
    s.abort = 0;
    fence_mbar_init();
    prefetch_map(&tmk);
    prefetch_map(&tmv);
  }
  __syncthreads();
  // (Behind a shared prefix the kernel before is k_prefix, which this one runs beside: it
  // lets this one start only once all that came before is there.)
  if (!kOwn) pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int c = blockIdx.x;

  if (warp >= kWarps) {
    // ------------------------------------------------------------ producer --
    // What a CTA does before its first load is on the path of every call: 32-bit
    // arithmetic, lengths handed on by shuffles, pieces described only after their loads.
    const int P = a.kv.page_size;
    const uint32_t box_bytes = (uint32_t)box_rows * D * 2, capacity = a.kv.max_pages * a.kv.page_size;
    // lane l < 4 (8): 16-position slice l of a tile; it loads the box that begins with it
    const bool is_k = warp == kWarps;   // K's also writes what the consumers read, V's what the join reads
    const int slice = lane & (kWarps * SL - 1), per_box = box_rows / 16;
    const bool loads = lane < kWarps * SL && slice % per_box == 0;
    const uint32_t box_at = (uint32_t)slice / per_box * box_bytes;
    uint32_t it = 0, pieces = 0;
    int seq, n_cut = 0;
    uint32_t before, L, G = gridDim.x;
    const uint32_t total = find_run(p, c, G, lane, &seq, &before, &L);
    const uint32_t t1 = c < (int)G ? run_start(total, c + 1, G) : 0;
    uint32_t t = run_start(total, c, G), ts = seq_tiles(p, L);   // (c >= G: no run)
    int cached_unit = -1, cached_base = 0, page = -1, left = 0, next_page = -1;   // lane i: entry cached_base + i
    bool alive = true, cut_first = false;
#pragma unroll 1
    while (t < t1 && alive) {
#pragma unroll 1
      while (t >= before + ts * p.units_per_seq) {
        before += ts * p.units_per_seq;
        L = a.seq_len[++seq];
        ts = seq_tiles(p, L);
      }
      const uint32_t unit = (t - before) / ts, begin = before + unit * ts, tile0 = t - begin;
      const uint32_t tile1 = min(ts, tile0 + (t1 - t));
      t += tile1 - tile0;
      const int h = p.chunks == 1 ? (int)unit : (int)unit / p.chunks, chunk = (int)unit - h * p.chunks;
      const int head = h * p.group + chunk * kMaxSlotHeads, heads = min(kMaxSlotHeads, p.group - chunk * kMaxSlotHeads);
      const bool fits = L <= capacity;
      if (!fits && lane == 0) raise_error(a.err, kDevBadArgument);
      const int dest = !fits ? -2 : tile0 == 0 && tile1 == ts ? -1 : 2 * c + (tile0 == 0 ? 1 : 0);
      const int32_t* table = a.kv.page_table + (long long)seq * a.kv.table_stride;
      const int32_t* list = a.list ? a.list + ((long long)seq * a.kv.n_kv_heads + h) * a.n_list : nullptr;
      const int n_entries = a.list ? a.n_list : (int)((L + P - 1) >> a.page_shift);
      const int unit_id = a.list ? seq * (int)a.kv.n_kv_heads + h : seq;   // one table row serves all heads
      bool first = true;
#pragma unroll 1
      for (uint32_t tile = tile0; tile < tile1; ++tile) {
        const int first_entry = ((int)tile * kTile) >> a.page_shift;
        if (cached_unit != unit_id || first_entry < cached_base ||
            ((int)tile * kTile + kTile - 1) >> a.page_shift >= cached_base + 32) {
          // page of the pool, and how many of the sequence's positions begin with it
          const int e = first_entry + lane;
          const bool ahead = cached_unit == unit_id && !list && first_entry == cached_base + 32;
          const int col = e < n_entries ? (list ? list[e] : e) : -1;
          page = -1;
          left = 0;
          if (fits && col != -1) {
            bool bad = col < 0 || col >= (int)a.kv.max_pages;
            if (!bad && (uint32_t)col * P < L) {
              page = ahead ? next_page : table[col];
              bad = page < 0 || (uint32_t)page >= a.kv.n_pages;
              if (!bad) left = (int)(L - (uint32_t)col * P);
            }
            if (bad) raise_error(a.err, kDevBadArgument);
          }
          cached_unit = unit_id;
          cached_base = first_entry;
          // the next 32 of the table row, asked for now
          if (!list && e + 32 < n_entries) next_page = table[e + 32];
        }
        const int pos = (int)tile * kTile + 16 * slice, from = (pos >> a.page_shift) - cached_base;
        const int off = pos & (P - 1);
        const int valid = min(max(__shfl_sync(0xffffffffu, left, from) - off, 0), 16);   // of this slice's positions
        const int my_page = __shfl_sync(0xffffffffu, page, from);
        const uint32_t any = __ballot_sync(0xffffffffu, loads && valid > 0);
        const bool last = tile + 1 == tile1;
        if (!any && !last) continue;   // nothing of the tile is listed
        const int st = it % ST;
        if (it >= ST &&
            !__all_sync(0xffffffffu, paged_wait(&s.empty[st], ((it / ST) - 1) & 1, &s.abort, a.err))) {
          alive = false;
          break;
        }
        StageMeta& meta = s.meta[st];
        if (is_k && lane < kWarps * SL) meta.valid[lane] = valid;
        if (is_k && lane == 0) {
          meta.flags = (first ? kFirst : 0) | (last ? kLast : 0);
          meta.heads = heads;
          if (last) {
            meta.seq = seq;
            meta.head = head;
            meta.dest = dest;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&s.full[st], box_bytes * __popc(any));
        __syncwarp();
        if (any >> lane & 1)
          tma_load_pages(s.kv[st][is_k ? 0 : 1] + box_at, is_k ? &tmk : &tmv, off, h, my_page, &s.full[st]);
        ++it;
        if (first && !is_k) {   // the unit's queries, behind its first tile
          const int qs = pieces % QS;
          if (pieces >= QS &&
              !__all_sync(0xffffffffu, paged_wait(&s.qempty[qs], (pieces / QS - 1) & 1, &s.abort, a.err))) {
            alive = false;
            break;
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&s.qfull[qs], (uint32_t)heads * D * 2);
            bulk_g2s(s.q[qs], a.q + (long long)seq * a.q_stride + (long long)head * D, (uint32_t)heads * D * 2,
                     &s.qfull[qs]);
          }
          ++pieces;
        }
        first = false;
      }
      if (dest >= 0 && !is_k) {
        CutUnit u;
        static_cast<CutPiece&>(u) = cut_piece(total, begin, ts, tile0, c, G);
        u.seq = seq;
        u.head = head;
        u.heads = heads;
        u.unit = seq * p.units_per_seq + (int)unit;
        if (lane == 0) s.cut[n_cut] = u;
        if (pieces == 1) cut_first = true;
        ++n_cut;
      }
    }
    __syncwarp();
    if (!is_k) {
      // While the last tiles are on their way: the counts of the units it shares, and
      // the arrival of a piece that is not the run's last.
      if (lane < n_cut) {
        const CutUnit& u = s.cut[lane];
        open_count(p.arrived + 2 * G + u.unit, p.tag);
        if (u.pieces > kJoin) open_count(p.arrived + piece_slot(u, u.piece / kJoin * kJoin, G), p.tag);
      }
      const int n_early = alive && n_cut > 0 && pieces > 1 && cut_first ? 1 : 0;
      if (n_early) {
        alive = __all_sync(0xffffffffu, paged_wait(&s.early, 0, &s.abort, a.err));
        if (alive && lane == 0) s.last[0] = arrive_first(p, s.cut[0], G);
      }
      if (lane == 0) {
        s.n_cut = n_cut;
        s.runs = (int)G;
        s.n_early = n_early;
      }
      __syncwarp();
    }
    uint32_t drained = it >= (uint32_t)ST ? it - ST : 0;
    if (alive) {   // the end of the run, in a stage whose last copy was consumed
      const int st = it % ST;
      alive = it < ST || __all_sync(0xffffffffu, paged_wait(&s.empty[st], ((it / ST) - 1) & 1, &s.abort, a.err));
      if (alive) {
        if (it >= ST) ++drained;
        if (lane == 0) {
          if (is_k) s.meta[st].flags = kEnd;
          mbar_arrive(&s.full[st]);
        }
      }
    }
    __syncwarp();
    // Every issued copy lands before the CTA may exit.
#pragma unroll 1
    for (uint32_t j = drained; j < it; ++j)
      paged_wait(&s.full[j % ST], (j / ST) & 1, &s.abort, a.err, false);
#pragma unroll 1
    for (uint32_t j = pieces > (uint32_t)QS ? pieces - QS : 0; j < pieces; ++j)
      paged_wait(&s.qfull[j % QS], (j / QS) & 1, &s.abort, a.err, false);
    if (kOwn && is_k && c == (int)gridDim.x - 1) pdl_wait();   // so that whoever waits for this kernel finds k_prefix done too
    return;
  }

  // -------------------------------------------------------------- consumers --
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t half_bytes = (uint32_t)box_rows * 128;   // [half][rows][128 B] of a box
  uint32_t qf[NT][D / 8];
  float o[NT][D / 16][4], m[NT][2], l[NT][2];
  uint32_t pieces = 0, joins = 0;
  auto join = [&]() {   // the consumer warps' barrier
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.joined);
    return __all_sync(0xffffffffu, paged_wait(&s.joined, joins++ & 1, &s.abort, a.err));
  };
#pragma unroll 1
  for (uint32_t it = 0;; ++it) {
    const int st = it % ST;
    if (!__all_sync(0xffffffffu, paged_wait(&s.full[st], (it / ST) & 1, &s.abort, a.err))) return;
    const StageMeta& meta = s.meta[st];
    const int flags = meta.flags;
    if (flags & kEnd) break;
    if (flags & kFirst) {
      const int qs = pieces % QS;
      if (!__all_sync(0xffffffffu, paged_wait(&s.qfull[qs], (pieces / QS) & 1, &s.abort, a.err))) return;
      ++pieces;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint4 v = 8 * n + g < meta.heads
                              ? *reinterpret_cast<const uint4*>(s.q[qs] + (8 * n + g) * D + (j >> 1) * 64 +
                                                                (2 * t4 + (j & 1)) * 8)
                              : make_uint4(0, 0, 0, 0);
          qf[n][4 * j] = v.x;
          qf[n][4 * j + 1] = v.y;
          qf[n][4 * j + 2] = v.z;
          qf[n][4 * j + 3] = v.w;
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.qempty[qs]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      }
    }
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
      const int valid = meta.valid[warp + kWarps * sl];
      if (valid <= 0) continue;
      const int first_row = 16 * (warp + kWarps * sl), row0 = first_row % box_rows;
      const uint32_t box_off = (uint32_t)(first_row / box_rows) * box_rows * D * 2;
      const uint8_t* kb = s.kv[st][0] + box_off;
      const uint8_t* vb = s.kv[st][1] + box_off;
      // ---- S^T = K q^T.  Lane (g, t) holds 16-byte chunks 2t, 2t+1 of each half of
      // rows g and g+8 (with the swizzle, eight lanes touch eight bank groups); the
      // MMA's k order is the lanes' order, the same for q.
      float sv[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) sv[n][0] = sv[n][1] = sv[n][2] = sv[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint8_t* p0 = kb + (j >> 1) * half_bytes + (row0 + g) * 128 + (((2 * t4 + (j & 1)) ^ g) << 4);
        const uint4 x = *reinterpret_cast<const uint4*>(p0), y = *reinterpret_cast<const uint4*>(p0 + 8 * 128);
        const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_16816_t(T{}, sv[n], a0, qf[n][4 * j], qf[n][4 * j + 1]);
          mma_16816_t(T{}, sv[n], a1, qf[n][4 * j + 2], qf[n][4 * j + 3]);
        }
      }
      // sv: (pos g, heads 2t, 2t+1), (pos g+8, heads 2t, 2t+1)
      bool grown = false;
      float mx[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sv[n][e] *= p.scale_log2;
        if (g >= valid) sv[n][0] = sv[n][1] = -INFINITY;
        if (g + 8 >= valid) sv[n][2] = sv[n][3] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[n][e] = fmaxf(sv[n][e], sv[n][2 + e]);
          grown |= mx[n][e] > m[n][e] + 15.f;
        }
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = mx[n][e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float r = fmaxf(m[n][e], x - 7.f);
            const float f = r == -INFINITY ? 1.f : exp2_fast(m[n][e] - r);
            m[n][e] = r;
            l[n][e] *= f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[n][i][e] *= f;
              o[n][i][2 + e] *= f;
            }
          }
      }
      uint32_t b0[NT], b1[NT], c0[NT], c1[NT];   // weights: rounded, and what that left
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float r = m[n][e] == -INFINITY ? 0.f : m[n][e];
          sv[n][e] = exp2_fast(sv[n][e] - r);
          sv[n][2 + e] = exp2_fast(sv[n][2 + e] - r);
          l[n][e] += sv[n][e] + sv[n][2 + e];
        }
        const uint32_t x0 = pack2(T{}, sv[n][0], sv[n][1]), x1 = pack2(T{}, sv[n][2], sv[n][3]);
        const float2 y0 = unpack2(T{}, x0), y1 = unpack2(T{}, x1);
        b0[n] = movmatrix(x0);   // (head g; pos 2t, 2t+1)
        b1[n] = movmatrix(x1);   // (head g; pos 2t+8, 2t+9)
        c0[n] = movmatrix(pack2(T{}, sv[n][0] - y0.x, sv[n][1] - y0.y));
        c1[n] = movmatrix(pack2(T{}, sv[n][2] - y1.x, sv[n][3] - y1.y));
      }
      // ---- o^T += V^T P^T: A = V^T[16 d x 16 pos] by ldmatrix.trans.
      const int vrow = row0 + (lane & 7) + ((lane >> 4) << 3);
      const uint8_t* vp = vb + vrow * 128;
      const int vchunk = (lane >> 3) & 1;
      if (valid == 16) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t av[4];
          ldmatrix_x4_t(av, vp + (i >> 2) * half_bytes + (((2 * (i & 3) + vchunk) ^ (lane & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816_t(T{}, o[n][i], av, b0[n], b1[n]);
          if constexpr (!kOwn) {
#pragma unroll
            for (int k = 0; k < 4; ++k) av[k] = finite2(T{}, av[k]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816_t(T{}, o[n][i], av, c0[n], c1[n]);
          }
        }
      } else {   // what lies past the end may be anything: 0 weight times NaN would be NaN
        const uint32_t k0 = (2 * t4 < valid ? 0xffffu : 0u) | (2 * t4 + 1 < valid ? 0xffff0000u : 0u);
        const uint32_t k1 = (2 * t4 + 8 < valid ? 0xffffu : 0u) | (2 * t4 + 9 < valid ? 0xffff0000u : 0u);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t av[4];
          ldmatrix_x4_t(av, vp + (i >> 2) * half_bytes + (((2 * (i & 3) + vchunk) ^ (lane & 7)) << 4));
          av[0] &= k0;
          av[1] &= k0;
          av[2] &= k1;
          av[3] &= k1;
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816_t(T{}, o[n][i], av, b0[n], b1[n]);
          if constexpr (!kOwn) {
#pragma unroll
            for (int k = 0; k < 4; ++k) av[k] = finite2(T{}, av[k]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816_t(T{}, o[n][i], av, c0[n], c1[n]);
          }
        }
      }
    }
    if (!(flags & kLast)) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[st]);
      continue;
    }

    // ---- the end of a piece.  Join the warps: o[n][i][e]: (d 16i+g, head 8n+2t+e),
    // [2+e]: (d 16i+g+8, ..).  The piece's last stage, which every warp is done with
    // after the first join, holds their rows: [warp][head][d ^ 8 (head / 2 % 4)].
    const StageMeta u = meta;
    float2(*ml)[kMaxSlotHeads] = s.ml[(pieces - 1) & 1];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[n][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) ml[warp][8 * n + 2 * t4 + e] = make_float2(m[n][e], x);
      }
    if (!join()) return;
    float* rows = reinterpret_cast<float*>(s.kv[st][0]);
    static_assert(kWarps * 8 * NT * D * 4 <= 2 * tile_of(D) * D * 2, "the warps' rows exceed a stage");
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int head = 8 * n + 2 * t4 + e;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w][head].x);
        const float f = m[n][e] == -INFINITY ? 0.f : exp2_fast(m[n][e] - M);
        float* row = rows + (warp * 8 * NT + head) * D;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          row[(16 * i + g) ^ (8 * t4)] = o[n][i][e] * f;
          row[(16 * i + g + 8) ^ (8 * t4)] = o[n][i][2 + e] * f;
        }
      }
    if (!join()) return;
#pragma unroll 1
    for (int head = warp; head < u.heads && u.dest != -2; head += kWarps) {
      constexpr int V = D / 32;   // elements of this lane
      float M = -INFINITY, sum = 0.f, v[V];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w][head].x);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // (a warp without a maximum has the sum 0, or NaN, which stays)
        sum += ml[w][head].y * (ml[w][head].x == -INFINITY ? 0.f : exp2_fast(ml[w][head].x - M));
        const float* row = rows + (w * 8 * NT + head) * D + ((V * lane) ^ (8 * (head / 2 % 4)));
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] += row[k];
      }
      if (u.dest == -1) finish_row<T, D, kOwn>(p, u.seq, u.head + head, as_float4(v), M, sum, lane);
      else store_partial<D>(p, u.dest * kMaxSlotHeads + head, as_float4(v), M, sum, lane);
    }
    fence_proxy_async();   // the rows before the next TMA write
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&s.empty[st]);
      if (pieces == 1) mbar_arrive(&s.early);   // the run's first piece is written
    }
  }

  // ---- the last pieces to arrive join the others'
  const int n_cut = s.n_cut, n_early = s.n_early, G = s.runs;
  if (n_cut == 0) return;
  if (!join()) return;   // every warp's partials are written
  if (threadIdx.x == 0 && n_early < n_cut) s.last[n_early] = arrive_first(p, s.cut[n_early], G);
  if (!join()) return;
#pragma unroll 1
  for (int k = 0; k < n_cut; ++k) {
    if (!s.last[k]) continue;
    const CutUnit& u = s.cut[k];
    const int groups = (u.pieces + kJoin - 1) / kJoin, first = u.piece / kJoin * kJoin;
    int from = first, step = 1, n = min(kJoin, u.pieces - first);
    bool final = groups == 1;
#pragma unroll 1
    for (;;) {   // its sixteen, then the unit's sixteens
      join_pieces<T, D, kOwn>(p, u, G, from, step, n, final, warp, lane);
      if (final) break;
      if (!join()) return;
      if (threadIdx.x == 0) s.last[k] = arrive_last(p.arrived + 2 * G + u.unit, p.tag, groups);
      if (!join()) return;
      if (!s.last[k]) break;
      from = 0;
      step = kJoin;
      n = groups;
      final = true;
    }
  }
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// A call's tag: an odd number of 48 bits, spread so that stale memory does not hold it
// but by a chance of 2^-47 a word.  Two calls may get the same one, as replays of one
// captured call do: a call leaves its counts at 0, which is what opening them would do.
unsigned long long next_tag() {
  static std::atomic<uint64_t> calls{splitmix64((uint64_t)std::chrono::steady_clock::now().time_since_epoch().count())};
  return (splitmix64(calls.fetch_add(1, std::memory_order_relaxed)) >> 16) | 1;
}

template <typename T, int D, int NT, bool kOwn>
int launch(const DecodeArgs& p, int G, const CUtensorMap& tmk, const CUtensorMap& tmv, int box_rows,
           cudaStream_t st) {
  auto kern = k_paged_decode<T, D, NT, kOwn>;
  const int smem = (int)sizeof(DecodeSmem<D, NT>) + 1024;
  static_assert((sizeof(DecodeSmem<D, NT>) + 2048) * kCtasPerSm <= 228 * 1024, "CTAs per SM");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(G);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static OncePerDevice once;
  return once.launch(reinterpret_cast<const void*>(kern), smem, [&] {
           return cudaLaunchKernelEx(&cfg, kern, p, box_rows, tmk, tmv);
         }) == cudaSuccess
             ? 0
             : -1;
}

template <typename T, int D>
int launch(const DecodeArgs& p, int G, const CUtensorMap& tmk, const CUtensorMap& tmv, int box_rows, cudaStream_t st) {
  if (p.group > 8)
    return p.own_o ? launch<T, D, 2, true>(p, G, tmk, tmv, box_rows, st)
                   : launch<T, D, 2, false>(p, G, tmk, tmv, box_rows, st);
  return p.own_o ? launch<T, D, 1, true>(p, G, tmk, tmv, box_rows, st)
                 : launch<T, D, 1, false>(p, G, tmk, tmv, box_rows, st);
}

int units_per_head(const qwen_paged_kv& kv, int n_heads) {
  return (n_heads / (int)kv.n_kv_heads + kMaxSlotHeads - 1) / kMaxSlotHeads;
}

}  // namespace

int paged_sm_count() {
  static std::mutex mu;
  static int counts[DeviceSymbolCache::kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= DeviceSymbolCache::kMaxDevices) return 148;
  std::lock_guard<std::mutex> lk(mu);
  if (!counts[dev] && cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return counts[dev];
}

// Rows = positions of the pool, innermost 64 elements: (element, slot, half, head, page).
// L2 fetches no more than a head's row at once, 128 or 256 B: with 64-element heads side
// by side, 256 B would bring the next head's along (64 x 16384 positions of 8 heads:
// 4400 GB/s so, 5550 GB/s with 128; in head-major pages 6550 GB/s either way).
int encode_pages_map(CUtensorMap* map, const qwen_paged_kv& kv, const uint16_t* base, int box_rows, int box_halves) {
  auto enc = tensor_map_encoder();
  if (!enc) return -1;
  const int halves = (int)kv.head_dim / 64;
  const cuuint64_t dims[5] = {64, kv.page_size, (cuuint64_t)halves, kv.n_kv_heads, kv.n_pages};
  const cuuint64_t strides[4] = {(cuuint64_t)kv.pos_stride * 2, 128, (cuuint64_t)kv.head_stride * 2,
                                 (cuuint64_t)kv.page_stride * 2};
  const cuuint32_t box[5] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_halves, 1, 1};
  const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
  return enc(map, kv.dtype == QWEN_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
             const_cast<uint16_t*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, halves == 1 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : -1;
}

bool paged_decode_fits(const qwen_paged_kv& kv, int n_heads, int n_list) {
  const double units = (double)kv.n_seq * kv.n_kv_heads * units_per_head(kv, n_heads);
  const double tiles = std::ceil((n_list ? n_list : (double)kv.max_pages) * kv.page_size / tile_of((int)kv.head_dim));
  return units * std::max(tiles, 1.0) < 2147483648.0;
}

size_t paged_decode_workspace(const qwen_paged_kv& kv, int n_heads) {
  const size_t G = kCtasPerSm * paged_sm_count(), units = (size_t)kv.n_seq * kv.n_kv_heads * units_per_head(kv, n_heads);
  return 2 * G * kMaxSlotHeads * (kv.head_dim + 2) * sizeof(float) + (2 * G + units) * sizeof(unsigned long long);
}

int launch_paged_decode(const PagedAttnArgs& a, cudaStream_t st, const PagedOwn& own) {
  DecodeArgs p{};
  p.a = a;
  p.chunks = units_per_head(a.kv, a.n_heads);
  p.group = a.n_heads / (int)a.kv.n_kv_heads;
  p.units_per_seq = (int)a.kv.n_kv_heads * p.chunks;
  p.tile_shift = a.kv.head_dim == 64 ? 7 : 6;
  static_assert(tile_of(64) == 128 && tile_of(128) == 64, "tile_shift");
  p.list_tiles = (int)(((long long)a.n_list * a.kv.page_size + (1 << p.tile_shift) - 1) >> p.tile_shift);
  p.scale_log2 = a.scale * kLog2e;
  const int G = kCtasPerSm * paged_sm_count();
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = p.part_o + (size_t)2 * G * kMaxSlotHeads * a.kv.head_dim;
  p.arrived = reinterpret_cast<unsigned long long*>(p.part_ml + (size_t)2 * G * kMaxSlotHeads * 2);
  p.tag = next_tag();
  p.own_o = own.o;
  p.own_ml = own.ml;
  p.few = own.few;
  p.few_tiles = own.few_tiles;
  // Boxes of 32 positions, or 16 where a page holds no more: a sequence's last
  // page costs at most 31 positions of traffic that do not count.
  const int box_rows = a.kv.page_size < 32 ? 16 : 32;
  CUtensorMap tmk, tmv;
  const int halves = (int)a.kv.head_dim / 64;
  if (encode_pages_map(&tmk, a.kv, a.kv.k, box_rows, halves) || encode_pages_map(&tmv, a.kv, a.kv.v, box_rows, halves))
    return -1;
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16)
    return d64 ? launch<__half, 64>(p, G, tmk, tmv, box_rows, st) : launch<__half, 128>(p, G, tmk, tmv, box_rows, st);
  return d64 ? launch<__nv_bfloat16, 64>(p, G, tmk, tmv, box_rows, st)
             : launch<__nv_bfloat16, 128>(p, G, tmk, tmv, box_rows, st);
}

}  // namespace qwen
