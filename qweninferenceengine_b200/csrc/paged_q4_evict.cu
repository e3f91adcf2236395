// paged_q4_evict.cu -- cuts the sequences of a 4-bit paged cache to a budget: of each
// (sequence, kv head) the n_keep slots stay that come first by (guarded, weight, slot).
//
// Two launches.  k_evict_select, a CTA or a cluster per (sequence, kv head): weights and
// positions are read into shared memory as ordered keys (up to 16384 slots a CTA; longer rows
// are read again from L2), the n_keep-th weight is found digit by digit (11, 11 and 10 bits, a
// histogram in shared memory each), and the slots that go and those that come are numbered in
// slot order.
// Few long rows are divided among the CTAs of a cluster, which add up their histograms.
// k_evict_move copies the rows, as many CTAs as fill the GPU.  Nothing a row is copied from is
// written, so the copies need no order, and what stays below n_keep is not touched: a sequence
// one token over its budget moves one row.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "paged_q4.cuh"
#include "qwen_internal.h"

namespace cg = cooperative_groups;

namespace qwen {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2048;

// A weight as a number that grows with it: NaN greatest, -0 like 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}

// What the first kernel leaves for the second, per (sequence, kv head): pairs of slots,
// (where to, where from), and their number; per sequence its new length or -1.
struct Moves {
  int2* pairs;     // [units][most]
  int* count;
  int* length;
  long long most;  // of a unit: as many as are kept or as are not, whichever are fewer
};
__host__ __device__ inline long long most_moves(const qwen_paged_kv_q4& kv, long long n_keep) {
  const long long rest = (long long)kv.max_pages * kv.page_size - n_keep;
  return rest < 0 ? 0 : rest < n_keep ? rest : n_keep;
}
__host__ __device__ inline Moves moves_of(const Q4EvictArgs& a) {
  const size_t units = (size_t)a.kv.n_seq * a.kv.n_kv_heads;
  Moves m;
  m.most = most_moves(a.kv, a.n_keep);
  m.pairs = static_cast<int2*>(a.workspace);
  m.count = reinterpret_cast<int*>(m.pairs + units * m.most);
  m.length = m.count + units;
  return m;
}

constexpr int kMaxHeld = 16384;              // slots whose keys a CTA holds in shared memory at most
constexpr int kTile = 32 * kThreads;         // slots numbered at once: a word of bits a thread
constexpr int kMaxCluster = 8;
constexpr int kAllBins = 2 * kBins + kBins / 2;   // of digits of 11, 11 and 10 bits

// Bits of a tile's slots, and how many are set in the words before.
struct Bits {
  uint32_t words[kTile / 32];
  int before[kTile / 32];
  __device__ __forceinline__ int rank_of(int i) const {   // (of slot i, in the tile)
    return before[i / 32] + __popc(words[i / 32] & ((1u << (i & 31)) - 1));
  }
};
struct __align__(16) SelectSmem {
  union {
    struct {
      int bins[kAllBins];   // a histogram for each digit
      int all[kAllBins];    // the cluster's, in its first CTA
    };
    int32_t positions[2 * kAllBins];   // before
  };
  Bits equal, stay;
  int sums[2][kWarps];
  int digit, left, in_bin;
  int newest, guarded, n_equal, kept, kept_below;   // of this CTA's slots, for the cluster
  uint32_t keys[1];   // as many as the launch has room for
};

// Sum of x over the CTA, and (before) over the threads before this one.  `turn` alternates
// from call to call, so that one barrier is enough.
__device__ __noinline__ int block_sum(int x, int (&sums)[2][kWarps], int turn, int* before) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) sums[turn & 1][warp] = inc;
  __syncthreads();
  const int all = lane < kWarps ? sums[turn & 1][lane] : 0;
  *before = inc - x + __reduce_add_sync(0xffffffffu, lane < warp ? all : 0);
  return __reduce_add_sync(0xffffffffu, all);
}

// One (sequence, kv head) by the CTAs of a cluster, or by one.  Latency throughout: for two
// rows of 32768 slots over eight CTAs each 15 us, of which the six cluster barriers take half;
// for 128 rows of 1060 slots 6 us, of 16384 slots 21.  Loops are rolled, with their loads in
// flight together: code that runs once is waited for line by line.
__device__ __forceinline__ void select_row(const Q4EvictArgs& a, int unit, int first, int n, int room, bool wide, SelectSmem& s) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int me = wide ? (int)cluster.block_rank() : 0, ctas = wide ? (int)cluster.num_blocks() : 1;
  // Lane i's: what CTA i left in x (`none` beyond the last).
  auto of_cluster = [&](int* x, int none) { return lane >= ctas ? none : wide ? *cluster.map_shared_rank(x, lane) : *x; };
  auto sum_of = [&](int* x, int upto) { return __reduce_add_sync(0xffffffffu, lane < upto ? of_cluster(x, 0) : 0); };
  const long long at = (long long)unit * q4_capacity(a.kv) + first;
  const float* weights = a.kv.weights + at;
  const int32_t* positions = a.kv.positions + at;
  const bool held = n <= room, held_positions = n <= 2 * kAllBins;
  int turn = 0, before;
  // ---- keys, and the newest position.  NaN is the greatest weight: 0xfffffffe.
  auto raw_key = [&](int i) { return min(weight_key(__ldg(weights + i)), 0xfffffffeu); };
  int newest = INT_MIN;
  constexpr int kAtOnce = 8;   // loads in flight
  for (int i0 = tid; i0 < n; i0 += kAtOnce * kThreads) {
    int p[kAtOnce];
    float w[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = i0 + j * kThreads;
      p[j] = i < n ? __ldg(positions + i) : INT_MIN;
      w[j] = i < n ? __ldg(weights + i) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      newest = max(newest, p[j]);
      const int i = i0 + j * kThreads;
      if (held && i < n) s.keys[i] = min(weight_key(w[j]), 0xfffffffeu);
      if (held_positions && i < n) s.positions[i] = p[j];
    }
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) s.sums[1][warp] = newest;
  __syncthreads();
  newest = __reduce_max_sync(0xffffffffu, s.sums[1][lane % kWarps]);
  if (wide) {
    if (tid == 0) s.newest = newest;
    cluster.sync();
    newest = __reduce_max_sync(0xffffffffu, of_cluster(&s.newest, INT_MIN));
  }
  const long long recent = (long long)newest - a.n_recent;
  // ---- how many are guarded; their key is all ones
  auto guards = [&](int p) { return p < a.n_first || (long long)p > recent; };
  auto guarded = [&](int i) { return guards(__ldg(positions + i)); };
  int count = 0;
  for (int i0 = tid; i0 < n; i0 += kAtOnce * kThreads) {
    int p[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = min(i0 + j * kThreads, n - 1);
      p[j] = held_positions ? s.positions[i] : __ldg(positions + i);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const bool g = i0 + j * kThreads < n && guards(p[j]);
      count += g;
      if (held && g) s.keys[i0 + j * kThreads] = 0xffffffffu;
    }
  }
  count = block_sum(count, s.sums, turn++, &before);
  for (int i = tid; i < 2 * kAllBins / 4; i += kThreads) reinterpret_cast<int4*>(s.bins)[i] = make_int4(0, 0, 0, 0);
  if (wide) {
    if (tid == 0) s.guarded = count;
    cluster.sync();
    count = sum_of(&s.guarded, ctas);
  } else {
    __syncthreads();
  }
  // Of the class that is cut (the guarded, if there are more than n_keep, else the others) the
  // rank-th greatest key is looked for; `pass_over` is the key of the other class.
  const bool cut = count > a.n_keep;
  const uint32_t pass_over = cut ? 0 : 0xffffffffu;
  if (cut && held) {
    for (int i = tid; i < n; i += kThreads) s.keys[i] = s.keys[i] == 0xffffffffu ? raw_key(i) : 0;
    __syncthreads();
  }
  auto key_of = [&](int i) { return held ? s.keys[i] : guarded(i) == cut ? raw_key(i) : pass_over; };
  int rank = cut ? a.n_keep : a.n_keep - count, equal = 0;
  uint32_t key = 0xffffffffu, mask = 0xffffffffu;   // rank 0: the guarded alone stay
  if (rank > 0) {
    key = mask = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023 : 2047;
      int* bins = s.bins + pass * kBins;
#pragma unroll 4
      for (int i = tid; i < n; i += kThreads) {
        const uint32_t k = key_of(i);
        if (k != pass_over && (k & mask) == key) atomicAdd(&bins[k >> shift & digits], 1);
      }
      __syncthreads();
      // thread i has bins 4i .. 4i + 3 from the greatest down; the first CTA adds up all's
      const int top = kBins - 4 - 4 * tid - (pass == 2 ? kBins / 2 : 0);   // (below 0: none)
      int4 b = make_int4(0, 0, 0, 0);
      if (top >= 0) b = *reinterpret_cast<const int4*>(bins + top);
      if (wide) {
        int* to = cluster.map_shared_rank(s.all + pass * kBins, 0) + top;
        if (b.x) atomicAdd(to, b.x);
        if (b.y) atomicAdd(to + 1, b.y);
        if (b.z) atomicAdd(to + 2, b.z);
        if (b.w) atomicAdd(to + 3, b.w);
        cluster.sync();
        if (top >= 0) b = *reinterpret_cast<const int4*>(to);
      }
      const int here = b.x + b.y + b.z + b.w;
      block_sum(here, s.sums, turn++, &before);
      if (before < rank && before + here >= rank) {
        const int in[4] = {b.w, b.z, b.y, b.x};
        int left = rank - before, j = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (j == i && left > in[i]) {
            left -= in[i];
            ++j;
          }
        s.digit = top + 3 - j;
        s.left = left;
        s.in_bin = in[j];
      }
      __syncthreads();
      key |= (uint32_t)s.digit << shift;
      mask |= digits << shift;
      rank = s.left;
      equal = s.in_bin;
      if (equal == rank) break;   // all that begin like this stay
    }
  }
  // ---- which stay: keys above, and of those equal to it (but the other class) the first `rank`
  const bool ties = equal > rank, some = rank > 0;
  auto same = [&](uint32_t k) { return some && k != pass_over && (k & mask) == key; };
  // Marks and numbers a tile's bits, after `seen`.
  auto number = [&](Bits& b, int base, int& seen, auto&& bit) {
    const int words = min(kTile, n - base + 31) / 32;
#pragma unroll 2
    for (int w = warp; w < words; w += kWarps) {
      const int i = base + 32 * w + lane;
      const uint32_t x = __ballot_sync(0xffffffffu, i < n && bit(i));
      if (lane == 0) b.words[w] = x;
    }
    __syncthreads();
    const int total = block_sum(tid < words ? __popc(b.words[tid]) : 0, s.sums, turn++, &before);
    b.before[tid] = seen + before;
    seen += total;
    __syncthreads();
  };
  int equal_before = 0;   // of the CTAs before
  if (ties && wide) {
    int mine = 0;
    for (int i = tid; i < n; i += kThreads) mine += same(key_of(i));
    mine = block_sum(mine, s.sums, turn++, &before);
    if (tid == 0) s.n_equal = mine;
    cluster.sync();
    equal_before = sum_of(&s.n_equal, me);
  }
  int seen = equal_before, kept = 0, kept_below = 0;   // of this CTA: that stay, of them below n_keep
  auto decide = [&](int base) {
    if (ties) number(s.equal, base, seen, [&](int i) { return same(key_of(i)); });
    number(s.stay, base, kept, [&](int i) {
      const uint32_t k = key_of(i);
      return same(k) ? !ties || s.equal.rank_of(i - base) < rank
                     : k == pass_over ? !cut : (k & mask) > key;
    });
    const int i = a.n_keep - first - base;   // (of this tile, or the last before n_keep)
    if (i > 0) kept_below = i >= min(kTile, n - base) ? kept : s.stay.rank_of(i);
    if (n > kTile) __syncthreads();   // every thread has read the tile's bits: the next one's take their place
  };
#pragma unroll 1
  for (int base = 0; base < n; base += kTile) decide(base);
  int offset = 0;   // that stay in the CTAs before
  if (wide) {
    if (tid == 0) {
      s.kept = kept;
      s.kept_below = kept_below;
    }
    cluster.sync();
    kept_below = sum_of(&s.kept_below, ctas);
    offset = sum_of(&s.kept, me);
  }
  // ---- in slot order the holes below n_keep and what comes into them
  int2* pairs = moves_of(a).pairs + unit * moves_of(a).most;
  const int below = kept_below;
  seen = equal_before;
  kept = 0;
#pragma unroll 1
  for (int base = 0; base < n; base += kTile) {
    if (n > kTile) decide(base);   // (else it stands there)
    const int end = min(kTile, n - base);
    for (int i = tid; i < end; i += kThreads) {
      const int slot = first + base + i;
      const bool stays = s.stay.words[i / 32] >> (i & 31) & 1;
      if (slot < a.n_keep ? stays : !stays) continue;
      const int r = offset + s.stay.rank_of(i);   // that stay before it
      if (stays) pairs[r - below].y = slot;
      else pairs[slot - r].x = slot;
    }
    __syncthreads();
  }
  if (tid == 0 && me == 0) moves_of(a).count[unit] = a.n_keep - below;
  if (wide) cluster.sync();   // what others may still read is there until then
}

__global__ void __launch_bounds__(kThreads, 2) k_evict_select(const __grid_constant__ Q4EvictArgs a, int ctas, int room) {
  extern __shared__ __align__(16) uint8_t smem[];
  SelectSmem& s = *reinterpret_cast<SelectSmem*>(smem);
  const int K = a.kv.n_kv_heads, unit = blockIdx.x / ctas, me = blockIdx.x - unit * ctas, seq = unit / K, tid = threadIdx.x;
  const Moves out = moves_of(a);
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();
  const uint32_t len = a.seq_len[seq];
  const bool fits = len <= q4_capacity(a.kv);
  if (tid == 0 && me == 0) {
    if (!fits) raise_error(a.err, kDevBadArgument);
    if (unit % K == 0) out.length[seq] = fits ? min((int)len, a.n_keep) : -1;
  }
  if (!fits || (int)len <= a.n_keep) {
    if (tid == 0 && me == 0) out.count[unit] = 0;
    return;
  }
  // whole words of bits to each CTA
  const int share = (((int)len + ctas - 1) / ctas + 31) / 32 * 32, first = me * share;
  select_row(a, unit, first, max(0, min(share, (int)len - first)), room, ctas > 1, s);
}

// D / 8 lanes a pair: 16 bytes of codes of each group of K and of V, then their parameters.
// A row is 1.25 D bytes in D / 8 sectors of 32, so that scattered ones cost three times that:
// 229,000 pairs of 64-element heads 19 us.
constexpr int kMoveThreads = 256;
template <int D>
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(const __grid_constant__ Q4EvictArgs a) {
  constexpr int G = D / 32, NC = 4 * G, kPairs = kMoveThreads / NC, kAtOnce = 4;   // pairs of a thread in flight
  const int K = a.kv.n_kv_heads, unit = blockIdx.x, s = unit / K, h = unit - s * K, c = threadIdx.x % NC, P = a.kv.page_size;
  const Moves in = moves_of(a);
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  if (blockIdx.y == 0 && threadIdx.x == 0 && h == 0 && in.length[s] >= 0) a.new_len[s] = (uint32_t)in.length[s];
  const int n = in.count[unit];
  const long long row = (long long)unit * q4_capacity(a.kv);
  // this lane's part of a slot in its block
  const int part = c < 2 * G ? c * 256 : Q4Block<D>::kKeySteps + (c - 2 * G) * 64, step = c < 2 * G ? 16 : 4;
  const int2* pairs = in.pairs + unit * in.most;
  for (int i0 = blockIdx.y * kPairs * kAtOnce + threadIdx.x / NC; i0 < n; i0 += gridDim.y * kPairs * kAtOnce) {
    int2 p[kAtOnce];
    int to[kAtOnce], from[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) p[j] = pairs[min(i0 + j * kPairs, n - 1)];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      to[j] = q4_page(a.kv, a.err, s, p[j].x >> a.page_shift);
      from[j] = q4_page(a.kv, a.err, s, p[j].y >> a.page_shift);
    }
    uint4 x[kAtOnce];
    uint32_t kept[kAtOnce];
    const uint32_t* slots = reinterpret_cast<const uint32_t*>(c ? (const void*)a.kv.positions : (const void*)a.kv.weights) + row;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (i0 + j * kPairs >= n) to[j] = -2;
      if (c < 2) kept[j] = slots[p[j].y];
      if (to[j] >= 0 && from[j] >= 0) {
        const uint8_t* src = q4_block<D>(a.kv, from[j], h, p[j].y & (P - 1)) + part + (p[j].y & 15) * step;
        if (c < 2 * G) x[j] = *reinterpret_cast<const uint4*>(src);
        else x[j].x = *reinterpret_cast<const uint32_t*>(src);
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (to[j] == -2) continue;
      if (c < 2) const_cast<uint32_t*>(slots)[p[j].x] = kept[j];
      if (to[j] < 0 || from[j] < 0) continue;
      uint8_t* dst = q4_block<D>(a.kv, to[j], h, p[j].x & (P - 1)) + part + (p[j].x & 15) * step;
      if (c < 2 * G) *reinterpret_cast<uint4*>(dst) = x[j];
      else *reinterpret_cast<uint32_t*>(dst) = x[j].x;
    }
  }
}

}  // namespace

size_t evict_q4_workspace(const qwen_paged_kv_q4& kv, uint32_t n_keep) {
  const size_t units = (size_t)kv.n_seq * kv.n_kv_heads;
  return units * most_moves(kv, n_keep) * sizeof(int2) + (units + kv.n_seq) * sizeof(int);
}

int launch_evict_q4(const Q4EvictArgs& a, cudaStream_t st) {
  const int units = (int)(a.kv.n_seq * a.kv.n_kv_heads);
  // CTAs of a row: as many as find room at once (two an SM), where rows can be long enough
  int cluster = 1;
  while (cluster < kMaxCluster && 2 * cluster * units <= 2 * paged_sm_count() &&
         (long long)a.kv.max_pages * a.kv.page_size > 4096 * cluster)
    cluster *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * cluster);
  cfg.blockDim = dim3(kThreads);
  const long long share = ((long long)a.kv.max_pages * a.kv.page_size + cluster - 1) / cluster + 31;
  const int room = (int)std::min<long long>(kMaxHeld, share);
  const int smem = (int)sizeof(SelectSmem) + 4 * room;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  static_assert(2 * (sizeof(SelectSmem) + 4 * kMaxHeld + 1024) <= 228 * 1024, "two CTAs an SM");
  static OncePerDevice once;
  if (once.launch(reinterpret_cast<const void*>(k_evict_select), (int)sizeof(SelectSmem) + 4 * kMaxHeld,
                  [&] { return cudaLaunchKernelEx(&cfg, k_evict_select, a, cluster, room); }) != cudaSuccess)
    return -1;
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  // (a round of pairs a CTA where there may be many, one pair a thread where few CTAs suffice)
  const int per_cta = kMoveThreads / ((int)a.kv.head_dim / 8);
  cfg.gridDim = dim3(units, std::max(1, std::min((a.n_keep + per_cta - 1) / per_cta, 8 * paged_sm_count() / units)));
  cfg.blockDim = dim3(kMoveThreads);
  return cudaLaunchKernelEx(&cfg, a.kv.head_dim == 64 ? k_evict_move<64> : k_evict_move<128>, a) == cudaSuccess ? 0 : -1;
}

}  // namespace qwen
