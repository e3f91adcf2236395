// paged_q4_evict.cu -- cuts the sequences of a 4-bit paged cache to a budget: of each
// (sequence, kv head) the n_keep slots stay that come first by (guarded, weight, slot).
//
// Two launches.  k_evict_select, a CTA per (sequence, kv head): weights and positions are
// read once into registers (up to 32 slots a thread; longer rows are read again from L2), the
// n_keep-th weight is found digit by digit (11, 11 and 10 bits of an order-preserving key, a
// histogram in shared memory each), and the slots that go and those that come are numbered
// in slot order.  k_evict_move copies the rows, as many CTAs as fill the GPU.  Nothing a row
// is copied from is written, so the copies need no order, and what stays below n_keep is not
// touched: a sequence one token over its budget moves one row.
#include <algorithm>
#include <climits>

#include "paged_q4.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kBins = 2048;

// A weight as a number that grows with it: NaN greatest, -0 like 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}

// What the first kernel leaves for the second, per (sequence, kv head): pairs of slots,
// (where to, where from), and their number; per sequence its new length or -1.
struct Moves {
  int2* pairs;    // [units][n_keep]
  int* count;
  int* length;
};
__host__ __device__ inline Moves moves_of(const Q4EvictArgs& a) {
  const size_t units = (size_t)a.kv.n_seq * a.kv.n_kv_heads;
  Moves m;
  m.pairs = static_cast<int2*>(a.workspace);
  m.count = reinterpret_cast<int*>(m.pairs + units * a.n_keep);
  m.length = m.count + units;
  return m;
}

constexpr int kTileSteps = 32, kTile = kTileSteps * kThreads;   // slots numbered at once

struct SelectSmem {
  int bins[kBins];
  uint32_t words[kTile / 32];   // a bit a slot
  int before[kTile / 32];       // bits set in the words before
  int sums[2][kWarps];
  int digit, left, in_bin;
};

// Sum of x over the CTA, and (before) over the threads before this one.  `turn` alternates
// from call to call, so that one barrier is enough.
__device__ __forceinline__ int block_sum(int x, SelectSmem& s, int turn, int* before = nullptr) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) s.sums[turn & 1][warp] = inc;
  __syncthreads();
  int all = s.sums[turn & 1][lane];
  if (before) *before = inc - x + __reduce_add_sync(0xffffffffu, lane < warp ? all : 0);
  return __reduce_add_sync(0xffffffffu, all);
}

// One (sequence, kv head).  kE: slots a thread keeps in registers, slot e * kThreads + tid; 0:
// any number, read again each time.
template <int kE>
struct Row {
  const float* weights;
  const int32_t* positions;
  int L, n_first;
  long long recent;
  uint32_t keys[kE ? kE : 1];
  uint32_t guards[kE ? (kE + 31) / 32 : 1];

  __device__ __forceinline__ int steps() const { return kE ? kE : (L + kThreads - 1) / kThreads; }
  __device__ __forceinline__ bool guarded(int e) const {
    if constexpr (kE != 0) {
      return guards[e / 32] >> (e % 32) & 1;
    } else {
      const int p = positions[e * kThreads + threadIdx.x];
      return p < n_first || (long long)p > recent;
    }
  }
  __device__ __forceinline__ uint32_t key(int e) const {
    if constexpr (kE != 0) return keys[e];
    else return weight_key(weights[e * kThreads + threadIdx.x]);
  }
  __device__ __forceinline__ bool there(int e) const { return e * kThreads + (int)threadIdx.x < L; }
};

template <int kE>
__device__ __forceinline__ void select_row(const Q4EvictArgs& a, int unit, int L, SelectSmem& s) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t capacity = q4_capacity(a.kv);
  Row<kE> row;
  row.weights = a.kv.weights + (long long)unit * capacity;
  row.positions = a.kv.positions + (long long)unit * capacity;
  row.L = L;
  row.n_first = a.n_first;
  int turn = 0;
  // ---- the newest position, and how many are guarded
  constexpr bool kHold = kE != 0 && kE <= 8;   // positions in registers (more would not fit: read again)
  int newest = INT_MIN, pos[kHold ? kE : 1];
  if constexpr (kE != 0) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int p = row.there(e) ? row.positions[e * kThreads + tid] : INT_MIN;
      if constexpr (kHold) pos[e] = p;
      newest = max(newest, p);
    }
#pragma unroll
    for (int e = 0; e < kE; ++e) row.keys[e] = row.there(e) ? __float_as_uint(row.weights[e * kThreads + tid]) : 0;
  } else {
    for (int i = tid; i < L; i += kThreads) newest = max(newest, row.positions[i]);
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) s.sums[1][warp] = newest;
  for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
  __syncthreads();
  newest = __reduce_max_sync(0xffffffffu, s.sums[1][lane]);
  row.recent = (long long)newest - a.n_recent;
  int n = 0;
  if constexpr (kE != 0) {
#pragma unroll
    for (int i = 0; i < (kE + 31) / 32; ++i) row.guards[i] = 0;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      row.keys[e] = weight_key(__uint_as_float(row.keys[e]));
      int p = 0;
      if constexpr (kHold) p = pos[e];
      else if (row.there(e)) p = row.positions[e * kThreads + tid];
      const bool g = row.there(e) && (p < a.n_first || (long long)p > row.recent);
      row.guards[e / 32] |= (uint32_t)g << (e % 32);
      n += g;
    }
  } else {
    for (int e = 0; row.there(e); ++e) n += row.guarded(e);
  }
  const int n_guarded = block_sum(n, s, turn++);
  // ---- of the class that is cut (the guarded, if there are more than n_keep, else the
  // others) the rank-th greatest key; of those equal to it, the first `rank` slots stay
  const bool cut = n_guarded > a.n_keep;
  int rank = cut ? a.n_keep : a.n_keep - n_guarded, equal = 0;
  uint32_t key = 0xffffffffu, mask = 0xffffffffu;   // rank 0: none of the others stays
  if (rank > 0) {
    key = mask = 0;
#pragma unroll 1
    for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift - 10) {
      const uint32_t digits = shift == 0 ? 1023 : 2047;
#pragma unroll
      for (int e = 0; e < row.steps(); ++e)
        if (row.there(e) && row.guarded(e) == cut && (row.key(e) & mask) == key)
          atomicAdd(&s.bins[row.key(e) >> shift & digits], 1);
      __syncthreads();
      // thread i has bins 2047 - 2i and 2046 - 2i: the greatest first
      const int b0 = s.bins[kBins - 1 - 2 * tid], b1 = s.bins[kBins - 2 - 2 * tid];
      int before;
      block_sum(b0 + b1, s, turn++, &before);
      if (before < rank && before + b0 + b1 >= rank) {
        const bool second = before + b0 < rank;
        s.digit = kBins - 1 - 2 * tid - second;
        s.left = rank - before - (second ? b0 : 0);
        s.in_bin = second ? b1 : b0;
      }
      s.bins[kBins - 1 - 2 * tid] = s.bins[kBins - 2 - 2 * tid] = 0;
      __syncthreads();
      key |= (uint32_t)s.digit << shift;
      mask |= digits << shift;
      rank = s.left;
      equal = s.in_bin;
      if (equal == rank) break;   // all that begin like this stay
    }
  }
  // ---- which stay, and in slot order the holes below n_keep and what comes into them
  int2* pairs = moves_of(a).pairs + (long long)unit * a.n_keep;
  // Numbers the set bits of a tile: s.before[] for s.words[], after `seen` before the tile.
  auto number = [&](int& seen) {
    __syncthreads();
    const uint32_t w = s.words[tid];
    int before;
    const int total = block_sum(__popc(w), s, turn++, &before);
    s.before[tid] = seen + before;
    seen += total;
    __syncthreads();
  };
  s.words[tid] = 0;   // (of steps that the row does not have)
  __syncthreads();
  const uint32_t below = (1u << lane) - 1;
  auto rank_of = [&](int e) { return s.before[e * kWarps + warp] + __popc(s.words[e * kWarps + warp] & below); };
  int seen = 0, kept = 0, kept_below = 0;   // equal ones, those that stay, and of them below n_keep
#pragma unroll 1
  for (int base = 0; base < L; base += kTile) {
    const int e_base = base / kThreads;   // (0 where registers hold the row)
    uint32_t stays = 0;                   // bit e: this thread's slot of step e
    auto each = [&](auto&& f) {   // f(step of the tile, step of the row)
      if constexpr (kE != 0) {
#pragma unroll
        for (int e = 0; e < kE; ++e) f(e, e);
      } else {
#pragma unroll 1
        for (int e = 0; e < kTileSteps; ++e) f(e, e_base + e);
      }
    };
    auto same_as_key = [&](int row_e) {
      return row.there(row_e) && row.guarded(row_e) == cut && (row.key(row_e) & mask) == key;
    };
    if (equal > rank) {   // ties: of those the first stay
      each([&](int e, int row_e) {
        const uint32_t w = __ballot_sync(0xffffffffu, same_as_key(row_e));
        if (lane == 0) s.words[e * kWarps + warp] = w;
      });
      number(seen);
      each([&](int e, int row_e) { stays |= (uint32_t)(same_as_key(row_e) && rank_of(e) < rank) << e; });
      __syncthreads();
    } else if (rank > 0) {
      each([&](int e, int row_e) { stays |= (uint32_t)same_as_key(row_e) << e; });
    }
    each([&](int e, int row_e) {
      const bool in = row.there(row_e);
      stays |= (uint32_t)(in && (row.guarded(row_e) == cut ? (row.key(row_e) & mask) > key : !cut)) << e;
      const uint32_t w = __ballot_sync(0xffffffffu, stays >> e & 1);
      if (lane == 0) s.words[e * kWarps + warp] = w;
    });
    number(kept);
    if (base <= a.n_keep && a.n_keep < base + kTile) {
      const int i = a.n_keep - base;   // slots that stay before slot n_keep
      kept_below = s.before[i / 32] + __popc(s.words[i / 32] & ((1u << (i % 32)) - 1));
    }
    each([&](int e, int row_e) {
      const int i = row_e * kThreads + tid, r = rank_of(e);
      const bool stay = stays >> e & 1;
      if (i < a.n_keep ? !stay : stay) {   // (i < L: n_keep is less)
        if (stay) pairs[r - kept_below].y = i;
        else pairs[i - r].x = i;
      }
    });
    __syncthreads();
  }
  if (tid == 0) moves_of(a).count[unit] = a.n_keep - kept_below;
}

__global__ void __launch_bounds__(kThreads) k_evict_select(const __grid_constant__ Q4EvictArgs a) {
  __shared__ SelectSmem s;
  const int K = a.kv.n_kv_heads, unit = blockIdx.x, seq = unit / K, tid = threadIdx.x;
  const Moves out = moves_of(a);
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();
  const uint32_t len = a.seq_len[seq];
  const bool fits = len <= q4_capacity(a.kv);
  if (tid == 0) {
    if (!fits) raise_error(a.err, kDevBadArgument);
    if (unit % K == 0) out.length[seq] = fits ? min((int)len, a.n_keep) : -1;
  }
  if (!fits || (int)len <= a.n_keep) {
    if (tid == 0) out.count[unit] = 0;
    return;
  }
  if (len <= 2 * kThreads) select_row<2>(a, unit, (int)len, s);
  else if (len <= 8 * kThreads) select_row<8>(a, unit, (int)len, s);
  else if (len <= 32 * kThreads) select_row<32>(a, unit, (int)len, s);
  else select_row<0>(a, unit, (int)len, s);
}

// D / 8 lanes a pair: 16 bytes of codes of each group of K and of V, then their parameters.
constexpr int kMoveThreads = 256;
template <int D>
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(const __grid_constant__ Q4EvictArgs a) {
  constexpr int G = D / 32, NC = 4 * G, kPairs = kMoveThreads / NC;
  const int K = a.kv.n_kv_heads, unit = blockIdx.x, s = unit / K, h = unit - s * K, c = threadIdx.x % NC, P = a.kv.page_size;
  const Moves in = moves_of(a);
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  if (blockIdx.y == 0 && threadIdx.x == 0 && h == 0 && in.length[s] >= 0) a.new_len[s] = (uint32_t)in.length[s];
  const int n = in.count[unit];
  const long long row = (long long)unit * q4_capacity(a.kv);
  for (int i = blockIdx.y * kPairs + threadIdx.x / NC; i < n; i += gridDim.y * kPairs) {
    const int2 p = in.pairs[(long long)unit * a.n_keep + i];
    const int to = q4_page(a.kv, a.err, s, p.x >> a.page_shift), from = q4_page(a.kv, a.err, s, p.y >> a.page_shift);
    if (c == 0) a.kv.weights[row + p.x] = a.kv.weights[row + p.y];
    if (c == 1) a.kv.positions[row + p.x] = a.kv.positions[row + p.y];
    if (to < 0 || from < 0) continue;
    uint8_t* dst = q4_block<D>(a.kv, to, h, p.x & (P - 1));
    const uint8_t* src = q4_block<D>(a.kv, from, h, p.y & (P - 1));
    const int rd = p.x & 15, rs = p.y & 15;
    if (c < 2 * G) {
      *reinterpret_cast<uint4*>(dst + c * 256 + rd * 16) = *reinterpret_cast<const uint4*>(src + c * 256 + rs * 16);
    } else {
      const int g = c - 2 * G;
      *reinterpret_cast<uint32_t*>(dst + Q4Block<D>::kKeySteps + g * 64 + rd * 4) =
          *reinterpret_cast<const uint32_t*>(src + Q4Block<D>::kKeySteps + g * 64 + rs * 4);
    }
  }
}

}  // namespace

size_t evict_q4_workspace(const qwen_paged_kv_q4& kv, uint32_t n_keep) {
  const size_t units = (size_t)kv.n_seq * kv.n_kv_heads;
  return units * n_keep * sizeof(int2) + (units + kv.n_seq) * sizeof(int);
}

int launch_evict_q4(const Q4EvictArgs& a, cudaStream_t st) {
  const int units = (int)(a.kv.n_seq * a.kv.n_kv_heads);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, k_evict_select, a) != cudaSuccess) return -1;
  const int per_cta = kMoveThreads / ((int)a.kv.head_dim / 8);
  cfg.gridDim = dim3(units, std::max(1, std::min((a.n_keep + per_cta - 1) / per_cta, 8 * paged_sm_count() / units)));
  cfg.blockDim = dim3(kMoveThreads);
  return cudaLaunchKernelEx(&cfg, a.kv.head_dim == 64 ? k_evict_move<64> : k_evict_move<128>, a) == cudaSuccess ? 0 : -1;
}

}  // namespace qwen
