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
//
// k_page_scores streams the bounds (HBM: 512 B a page and kv head of 128) into one
// 64-bit key a page whose order is the scores'.  16 x 2048 pages of 8 heads, 134 MB:
// 34 us, 4.0 TB/s; 29 us without the conversions to 64 bits (16 a clock and SM).  Its SMs
// are busy for four fifths of it: launch, lengths, first bounds and the last run's end are
// the rest.
// k_page_list picks, a CTA per kv head and sequence: bins the keys linearly between
// their least and greatest (2048 bins), finds the bin that the last place falls
// in, and goes on inside it -- one round where scores are spread, and a round per 11
// bits at worst -- until the bin is taken whole, small enough to rank directly, or
// one value.  Bound by latency: 10 us for 2048 pages, a dozen barriers and round trips.
#include <algorithm>

#include "paged_common.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kScoreWarps = 8, kScoreCtas = 2;   // of an SM
constexpr int kBatch = 8;             // pages a warp has in flight
constexpr int kListThreads = 512;
constexpr int kBins = 2048;
constexpr int kRank = 128;            // keys ranked directly
constexpr int kCached = 8192;         // keys held in shared memory

typedef unsigned long long u64;

// Ascending order of keys = ascending order of scores; NaN above everything.
__device__ __forceinline__ u64 score_key(double x) {
  if (x != x) return ~0ull;
  const u64 b = (u64)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// Pages of a sequence of length L that compete for a place on its list (0: all are
// on it, or the length is refused).
__device__ __forceinline__ uint32_t scored_pages(const PagedSelectArgs& a, uint32_t L) {
  if (L > a.kv.max_pages * a.kv.page_size) return 0;
  const uint32_t n = (L + a.kv.page_size - 1) >> a.page_shift;
  return n > (uint32_t)a.n_select ? n : 0;
}

// Pages [begin, end) of sequence s, all kv heads, by the CTA's warps.  A warp keeps one
// kv head's Q+- in registers; a group of D / 4 lanes reads a page's bounds, lower half
// lo and upper half hi, 8 elements a lane.
template <typename T, int D>
__device__ __forceinline__ void score_pages(const PagedSelectArgs& a, int s, int begin, int end, int warp, int lane,
                                            uint4 (&held)[2][kBatch][32]) {
  constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;   // lanes of a page, pages of a load
  const int K = a.kv.n_kv_heads, G = a.n_heads / K;
  // warps per head, where there are fewer heads than warps
  const int share = K >= kScoreWarps ? 1 : kScoreWarps / K;
  const int part = lane & (kLanes - 1), sub = lane / kLanes;
  const bool upper = part >= kLanes / 2;
  const int d0 = 8 * (part & (kLanes / 2 - 1));
  const int32_t* table = a.kv.page_table + (long long)s * a.kv.table_stride;
#pragma unroll 1
  for (int h = warp / share; h < K; h += kScoreWarps / share) {
    u64* keys = reinterpret_cast<u64*>(a.scores) + ((long long)s * K + h) * a.kv.max_pages;
    const T* bounds = reinterpret_cast<const T*>(a.kv.bounds) + (upper ? (long long)K * D : 0) + (long long)h * D + d0;
    constexpr int kPages = kBatch * kAtOnce;
    // One batch's bounds are on their way while the one before is summed, and the page
    // numbers of the one after.
    const int step = share * kPages, p_first = begin + (warp % share) * kPages;
    auto page_of = [&](int p0) {   // lane i: page p0 + i of the sequence, or -1
      int page = 0;
      if (lane < kPages && p0 + lane < end) {
        page = table[p0 + lane];
        if (page < 0 || (uint32_t)page >= a.kv.n_pages) {
          raise_error(a.err, kDevBadArgument);
          page = -1;
        }
      }
      return page;
    };
    // A lane copies what it reads itself, so that no one else waits for it.
    auto fetch = [&](int page, int stage) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const long long at = max(__shfl_sync(0xffffffffu, page, i * kAtOnce + sub), 0);
        cp_async16(&held[stage][i][lane], bounds + at * 2 * K * D);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int page0 = page_of(p_first), page1 = page_of(p_first + step), stage = 0;
    fetch(page0, 0);
    double w[8];
    uint32_t used[4];   // bounds that no query multiplies read as 0 (they may be infinite)
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
    for (int g = 0; g < G; ++g) {
      const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + s * a.q_stride +
                                                      (long long)(h * G + g) * D + d0);
      const uint32_t b[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2(T{}, b[i]);
        w[2 * i] += (v.x > 0.f) == upper ? v.x : 0.f;   // NaN goes to the lower half
        w[2 * i + 1] += (v.y > 0.f) == upper ? v.y : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) used[i] = (w[2 * i] != 0 ? 0xffffu : 0u) | (w[2 * i + 1] != 0 ? 0xffff0000u : 0u);
    auto score = [&](int p0, int page, const uint4 (&x)[kBatch][32]) {
      const uint32_t bads = __ballot_sync(0xffffffffu, page < 0);
      double sum[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint4 y = x[i][lane];
        const uint32_t b[4] = {y.x & used[0], y.y & used[1], y.z & used[2], y.w & used[3]};
        sum[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = unpack2(T{}, b[j]);
          sum[i] = fma(w[2 * j], (double)v.x, sum[i]);
          sum[i] = fma(w[2 * j + 1], (double)v.y, sum[i]);
        }
      }
      // Eight sums over kLanes lanes: halve the sums while exchanging, so that lane
      // part = 4 x (its page in reading order, bits swapped) holds one.
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const int keep = kBatch / (2 * o);
#pragma unroll
        for (int i = 0; i < keep; ++i) {
          const bool odd = lane & o;
          const double mine = odd ? sum[keep + i] : sum[i], other = odd ? sum[i] : sum[keep + i];
          sum[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
      }
#pragma unroll
      for (int o = 8; o < kLanes; o <<= 1) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], o);
      const int i = ((lane & 1) << 2) | (lane & 2) | ((lane & 4) >> 2);   // of the batch
      const int at = i * kAtOnce + sub;
      if (part < 8 && p0 + at < end) keys[p0 + at] = bads >> at & 1 ? 0 : score_key(sum[0]);
    };
#pragma unroll 1
    for (int p0 = p_first; p0 < end; p0 += step) {
      fetch(page1, stage ^ 1);
      const int next = page_of(p0 + 2 * step);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      score(p0, page0, held[stage]);
      page0 = page1;
      page1 = next;
      stage ^= 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
}

// The scored pages of all sequences stand in one row, and each CTA takes an equal run
// of it.  (A CTA for 64 pages of a sequence, with the batches on their way in registers:
// 51 us for both kernels at the size above, 44.5 us so.)
template <typename T, int D>
__global__ void __launch_bounds__(kScoreWarps * 32, kScoreCtas) k_page_scores(const __grid_constant__ PagedSelectArgs a) {
  extern __shared__ uint4 smem[];   // [warp][stage][load][lane]
  auto held = reinterpret_cast<uint4(*)[2][kBatch][32]>(smem);
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_seq = a.kv.n_seq;
  // The run [x, x1), the sequence that holds x and the pages before it: each warp scans
  // the lengths.
  const int per_lane = (n_seq + 31) / 32, s0 = min(n_seq, lane * per_lane), s1 = min(n_seq, s0 + per_lane);
  u64 sum = 0;
  bool bad = false;
#pragma unroll 4
  for (int i = s0; i < s1; ++i) {
    const uint32_t L = a.seq_len[i];
    bad |= L > a.kv.max_pages * a.kv.page_size;
    sum += scored_pages(a, L);
  }
  if (bad && blockIdx.x == 0) raise_error(a.err, kDevBadArgument);
  u64 inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  const u64 total = __shfl_sync(0xffffffffu, inc, 31), per = divide(total + gridDim.x - 1, gridDim.x);
  u64 x = blockIdx.x * per;
  const u64 x1 = min(total, x + per);
  if (x >= x1) return;
  const int from = __ffs(__ballot_sync(0xffffffffu, x < inc)) - 1;   // the lane whose sequences hold x
  u64 before = __shfl_sync(0xffffffffu, inc - sum, from);
#pragma unroll 1
  for (int s = __shfl_sync(0xffffffffu, s0, from); x < x1; ++s) {
    const uint32_t n = scored_pages(a, a.seq_len[s]);
    if (x < before + n) {
      const u64 end = min((u64)n, x1 - before);
      score_pages<T, D>(a, s, (int)(x - before), (int)end, warp, lane, held[warp]);
      x = before + end;
    }
    before += n;
  }
}

struct ListSmem {
  uint32_t bins[kBins];
  u64 rank_key[kRank];
  int rank_at[kRank];
  u64 red[2][kListThreads / 32];
  uint32_t warp_sum[kListThreads / 32];
  u64 warp_pair[kListThreads / 32];
  uint32_t count, found_bin, found_above;
  u64 key;
};

// Exclusive sum over the CTA's threads of v (and the total), packed or not.  Small
// code throughout this kernel: it runs once, from a cold instruction cache.
template <typename V>
__device__ __forceinline__ V exclusive_sum(V v, V* warp_sums, V* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kW = kListThreads / 32;
  V inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  V ws = lane < kW ? warp_sums[lane] : 0;   // every warp adds up the warps' sums
#pragma unroll
  for (int o = 1; o < kW; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, ws, o);
    if (lane >= o) ws += x;
  }
  *total = __shfl_sync(0xffffffffu, ws, kW - 1);
  const V before = __shfl_sync(0xffffffffu, ws, (warp - 1) & 31);
  return inc - v + (warp ? before : 0);
}

__global__ void __launch_bounds__(kListThreads) k_page_list(const __grid_constant__ PagedSelectArgs a) {
  extern __shared__ u64 cached[];
  __shared__ ListSmem sm;
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int h = blockIdx.x, s = blockIdx.y, K = a.kv.n_kv_heads, tid = threadIdx.x;
  bool ok;
  const int L = (int)checked_len(a.kv, a.seq_len, s, &ok);
  if (!ok) return;   // reported by k_page_scores
  const int n = (L + a.kv.page_size - 1) >> a.page_shift;
  int32_t* list = a.pages + ((long long)s * K + h) * a.n_select;
  if (n <= a.n_select) {
    for (int i = tid; i < a.n_select; i += kListThreads) list[i] = i < n ? i : -1;
    return;
  }
  // The pages that compete: [first, end); `wanted` of them are taken.
  const int first = a.n_first, end = n - a.n_last, m = end - first;
  uint32_t wanted = a.n_select - a.n_first - a.n_last;
  const u64* global = reinterpret_cast<const u64*>(a.scores) + ((long long)s * K + h) * a.kv.max_pages + first;
  const u64* keys = global;
  u64 lo = ~0ull, hi = 0;
#pragma unroll 4
  for (int i = tid; i < m; i += kListThreads) {
    const u64 x = __ldcg(global + i);
    if (m <= kCached) cached[i] = x;
    lo = min(lo, x);
    hi = max(hi, x);
  }
  if (m <= kCached) keys = cached;
  auto extremes = [&]() {
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) {
      lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  };
  extremes();
  if ((tid & 31) == 0) {
    sm.red[0][tid >> 5] = lo;
    sm.red[1][tid >> 5] = hi;
  }
  __syncthreads();
  lo = sm.red[0][tid & (kListThreads / 32 - 1)];
  hi = sm.red[1][tid & (kListThreads / 32 - 1)];
  extremes();
  // Taken: keys above `cut`, and of those equal to it the first `ties`.
  u64 cut = ~0ull;
  uint32_t ties = 0;
  if (wanted == 0) {
    cut = ~0ull;
  } else {
    for (;;) {
      if (lo == hi) {
        cut = lo;
        ties = wanted;
        break;
      }
      const int shift = max(0, 64 - __clzll(hi - lo) - 11);
      for (int i = tid; i < kBins; i += kListThreads) sm.bins[i] = 0;
      if (tid == 0) sm.count = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = tid; i < m; i += kListThreads) {
        const u64 x = keys[i];
        if (x >= lo && x <= hi) atomicAdd(&sm.bins[(x - lo) >> shift], 1u);
      }
      __syncthreads();
      // From the top: the bin where the count reaches `wanted`.
      constexpr int kPer = kBins / kListThreads;
      uint32_t c[kPer], sum = 0, total;
#pragma unroll
      for (int j = 0; j < kPer; ++j) sum += c[j] = sm.bins[kBins - 1 - (tid * kPer + j)];
      uint32_t above = exclusive_sum(sum, sm.warp_sum, &total);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (above < wanted && above + c[j] >= wanted) {
          sm.found_bin = kBins - 1 - (tid * kPer + j);
          sm.found_above = above;
        }
        above += c[j];
      }
      __syncthreads();
      const uint32_t bin = sm.found_bin, held = sm.bins[bin];
      wanted -= sm.found_above;
      lo += (u64)bin << shift;
      hi = lo + min(hi - lo, ((u64)1 << shift) - 1);
      if (held == wanted) {   // the whole bin
        cut = lo - 1;         // lo > 0: a bin below the top one, or lo == hi above
        if (lo == 0) {
          cut = 0;
          ties = 0xffffffffu;
        }
        break;
      }
      if (held <= kRank) {    // rank them: higher key first, then lower page
#pragma unroll 1
        for (int i = tid; i < m; i += kListThreads) {
          const u64 x = keys[i];
          if (x >= lo && x <= hi) {
            const uint32_t at = atomicAdd(&sm.count, 1u);
            sm.rank_key[at] = x;
            sm.rank_at[at] = i;
          }
        }
        __syncthreads();
        // (a warp for each of them: a thread for each took 10 us for 128)
        for (uint32_t k = tid / 32; k < held; k += kListThreads / 32) {
          const u64 x = sm.rank_key[k];
          const int at = sm.rank_at[k];
          uint32_t rank = 0, same = 0;
#pragma unroll 1
          for (uint32_t j = tid & 31; j < held; j += 32) {
            const u64 y = sm.rank_key[j];
            const int there = sm.rank_at[j];
            rank += y > x || (y == x && there < at);
            same += y == x && there <= at;
          }
          rank = __reduce_add_sync(0xffffffffu, rank);
          same = __reduce_add_sync(0xffffffffu, same);
          if (rank == wanted - 1 && (tid & 31) == 0) {
            sm.key = x;
            sm.count = same;
          }
        }
        __syncthreads();
        cut = sm.key;
        ties = sm.count;
        break;
      }
      __syncthreads();
    }
  }
  // Ascending list: each thread a run of pages; places from one sum over the CTA of
  // (keys above the cut, keys equal to it).
  const int per = (m + kListThreads - 1) / kListThreads, i0 = min(m, tid * per), i1 = min(m, i0 + per);
  u64 mine = 0, total;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) mine += keys[i] > cut ? 1ull << 32 : keys[i] == cut ? 1ull : 0ull;
  const u64 before = exclusive_sum(mine, sm.warp_pair, &total);
  uint32_t equal = (uint32_t)before;
  int at = a.n_first + (int)(before >> 32) + (int)min(equal, ties);
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    const bool take = keys[i] > cut || (keys[i] == cut && equal++ < ties);
    if (take) list[at++] = first + i;
  }
#pragma unroll 1
  for (int i = tid; i < a.n_first; i += kListThreads) list[i] = i;
#pragma unroll 1
  for (int i = tid; i < a.n_last; i += kListThreads) list[a.n_select - a.n_last + i] = end + i;
}

template <typename T, int D>
int launch(const PagedSelectArgs& a, cudaStream_t st) {
  // As many CTAs as run at once, fewer where that would leave a warp less than a batch of pages.
  const int share = std::max(1, kScoreWarps / (int)a.kv.n_kv_heads), least = share * kBatch * 32 / (D / 4);
  const long long pages = (long long)a.kv.max_pages * a.kv.n_seq;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min((long long)kScoreCtas * paged_sm_count(), (pages + least - 1) / least));
  cfg.blockDim = dim3(kScoreWarps * 32);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  constexpr int kSmem = kScoreWarps * 2 * kBatch * 32 * (int)sizeof(uint4);
  cfg.dynamicSmemBytes = kSmem;
  static OncePerDevice scores;
  if (scores.launch(reinterpret_cast<const void*>(k_page_scores<T, D>), kSmem,
                    [&] { return cudaLaunchKernelEx(&cfg, k_page_scores<T, D>, a); }) != cudaSuccess)
    return -1;
  cfg.gridDim = dim3(a.kv.n_kv_heads, a.kv.n_seq);
  cfg.blockDim = dim3(kListThreads);
  cfg.dynamicSmemBytes = (size_t)(a.kv.max_pages < (uint32_t)kCached ? a.kv.max_pages : kCached) * sizeof(u64);
  static OncePerDevice once;
  return once.launch(reinterpret_cast<const void*>(k_page_list), kCached * (int)sizeof(u64), [&] {
           return cudaLaunchKernelEx(&cfg, k_page_list, a);
         }) == cudaSuccess
             ? 0
             : -1;
}

}  // namespace

int launch_select_pages(const PagedSelectArgs& a, cudaStream_t st) {
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) return d64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return d64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}

}  // namespace qwen
