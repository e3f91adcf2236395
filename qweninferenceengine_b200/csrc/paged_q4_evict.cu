// paged_q4_evict.cu -- cuts the sequences of a 4-bit paged cache to a budget: of each
// (sequence, kv head) the n_keep slots stay that come first by (guarded, weight, slot).
#include "paged_q4.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kThreads = 1024;

// A weight as a number that grows with it: NaN greatest, -0 like 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}

// What the first kernel leaves for the second, per (sequence, kv head): pairs of slots,
// (where to, where from), and their number; per sequence its new length or -1.
struct Moves {
  int* count;
  int2* pairs;    // [units][n_keep]
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

// The sum of x over the threads before this one; *total: over all (two barriers).
__device__ __forceinline__ int scan_block(int x, int* warp_sums, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    const int v = warp_sums[w];
    before += w < warp ? v : 0;
    all += v;
  }
  __syncthreads();
  *total = all;
  return before + inc - x;
}

__global__ void __launch_bounds__(kThreads) k_evict_select(const __grid_constant__ Q4EvictArgs a) {
  __shared__ int sums[kThreads / 32], histogram[256], s_newest, s_digit, s_rank;
  const int K = a.kv.n_kv_heads, unit = blockIdx.x, s = unit / K, tid = threadIdx.x;
  const Moves out = moves_of(a);
  const uint32_t len = a.seq_len[s];
  const bool fits = len <= q4_capacity(a.kv);
  if (tid == 0) {
    if (!fits) raise_error(a.err, kDevBadArgument);
    if (unit % K == 0) out.length[s] = fits ? min((int)len, a.n_keep) : -1;
  }
  if (!fits || (int)len <= a.n_keep) {
    if (tid == 0) out.count[unit] = 0;
    return;
  }
  const int L = (int)len;
  const float* weights = a.kv.weights + (long long)unit * q4_capacity(a.kv);
  const int32_t* positions = a.kv.positions + (long long)unit * q4_capacity(a.kv);
  if (tid == 0) s_newest = INT_MIN;
  __syncthreads();
  int newest = INT_MIN;
  for (int i = tid; i < L; i += kThreads) newest = max(newest, positions[i]);
  atomicMax(&s_newest, newest);
  __syncthreads();
  const long long recent = (long long)s_newest - a.n_recent;
  auto guarded = [&](int i) { return positions[i] < a.n_first || (long long)positions[i] > recent; };
  int n = 0, n_guarded;
  for (int i = tid; i < L; i += kThreads) n += guarded(i);
  scan_block(n, sums, &n_guarded);
  // Of the class that is cut (the guarded, if there are more than n_keep, else the others)
  // the rank-th greatest key: digit by digit, then the lowest slots of those equal to it.
  const bool cut = n_guarded > a.n_keep;
  int rank = cut ? a.n_keep : a.n_keep - n_guarded;
  uint32_t key = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) histogram[tid] = 0;
    __syncthreads();
    for (int i = tid; i < L; i += kThreads) {
      const uint32_t k = weight_key(weights[i]);
      if (guarded(i) == cut && (k & mask) == key) atomicAdd(&histogram[k >> shift & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, left = rank;
      while (d > 0 && histogram[d] < left) left -= histogram[d--];
      s_digit = d;
      s_rank = left;
    }
    __syncthreads();
    key |= (uint32_t)s_digit << shift;
    mask |= 255u << shift;
    rank = s_rank;   // of the slots with this key, the first `rank` stay
    __syncthreads();
  }
  // In slot order: which stay, the holes below n_keep and what comes into them.
  int equal = 0, holes = 0, comes = 0;
  int2* pairs = out.pairs + (long long)unit * a.n_keep;
  for (int base = 0; base < L; base += kThreads) {
    const int i = base + tid;
    bool mine = false, same = false;
    if (i < L) {
      const bool g = guarded(i);
      const uint32_t k = weight_key(weights[i]);
      mine = g && !cut;
      if (g == cut) {
        mine = k > key;
        same = k == key;
      }
    }
    int total;
    const int before = scan_block(same, sums, &total);
    if (same) mine = equal + before < rank;
    equal += total;
    const bool hole = i < a.n_keep && !mine, come = i >= a.n_keep && i < L && mine;
    const int at_hole = scan_block(hole, sums, &total) + holes;
    holes += total;
    const int at_come = scan_block(come, sums, &total) + comes;
    comes += total;
    if (hole) pairs[at_hole].x = i;
    if (come) pairs[at_come].y = i;
  }
  if (tid == 0) out.count[unit] = holes;
}

// A warp per pair: 1.25 D bytes of codes, steps and lows, weight and position.
template <int D>
__global__ void __launch_bounds__(256) k_evict_move(const __grid_constant__ Q4EvictArgs a) {
  constexpr int G = D / 32;
  const int K = a.kv.n_kv_heads, unit = blockIdx.x, s = unit / K, h = unit - s * K, lane = threadIdx.x & 31;
  const Moves in = moves_of(a);
  if (blockIdx.y == 0 && threadIdx.x == 0 && h == 0 && in.length[s] >= 0) a.new_len[s] = (uint32_t)in.length[s];
  const int n = in.count[unit], P = a.kv.page_size;
  const long long row = (long long)unit * q4_capacity(a.kv);
  for (int i = blockIdx.y * 8 + (threadIdx.x >> 5); i < n; i += gridDim.y * 8) {
    const int2 p = in.pairs[(long long)unit * a.n_keep + i];
    if (lane == 0) {
      a.kv.weights[row + p.x] = a.kv.weights[row + p.y];
      a.kv.positions[row + p.x] = a.kv.positions[row + p.y];
    }
    const int to = q4_page(a.kv, a.err, s, p.x >> a.page_shift), from = q4_page(a.kv, a.err, s, p.y >> a.page_shift);
    if (to < 0 || from < 0) continue;
    uint8_t* dst = q4_block<D>(a.kv, to, h, p.x & (P - 1));
    const uint8_t* src = q4_block<D>(a.kv, from, h, p.y & (P - 1));
    const int rd = p.x & 15, rs = p.y & 15;
    if (lane < 2 * G) {   // codes of a group
      *reinterpret_cast<uint4*>(dst + lane * 256 + rd * 16) = *reinterpret_cast<const uint4*>(src + lane * 256 + rs * 16);
    } else if (lane < 4 * G) {   // step and low of a group
      const int g = lane - 2 * G;
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
  const unsigned units = a.kv.n_seq * a.kv.n_kv_heads;
  k_evict_select<<<units, kThreads, 0, st>>>(a);
  const dim3 grid(units, std::min(32, (a.n_keep + 7) / 8));
  if (a.kv.head_dim == 64) k_evict_move<64><<<grid, 256, 0, st>>>(a);
  else k_evict_move<128><<<grid, 256, 0, st>>>(a);
  return 0;
}

}  // namespace qwen
