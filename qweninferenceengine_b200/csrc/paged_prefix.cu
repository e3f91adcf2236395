// paged_prefix.cu -- decode attention of a batch over a prefix that all its
// sequences share, held once in the pool, and the join with their own positions.
//
// For one kv head the batch's queries are a matrix of n_seq x group rows against
// the same keys, so the prefix is read once and its products fill the tensor
// cores: 4 rows D L flops against 4 D L bytes -- from ~250 rows on it is bound by
// tcgen05 (and by the exponentials: 128 x 128 of them take the SFUs as long as the
// two MMAs of a tile take), below that by HBM.  64 sequences behind 131072 positions, 32
// query and 8 kv heads of 128: 143 us, 960 TFLOP/s.  What it has there is the chain of a
// stream's step, S -> weights -> O and the next S, with its four hand-overs: ~3650
// clocks a step of both streams where the MMAs take 2048; without any exponential the
// kernel is 1% faster.
//
// Three launches, each a programmatic dependent of the one before:
//   k_prefix        below, on part of the SMs
//   k_paged_decode (paged_decode.cu)  every sequence's own positions, beside it: on the
//       other SMs, or, where those would take longer, on all of them in the end; it
//       leaves (max, sum, unnormalised row) per query head instead of outputs
//   k_prefix_join   per query head: own part and the prefix's partials, in a fixed
//       order, into out and lse
// One is arithmetic, the other a stream, and each spends 5 to 8 us on its beginning and
// end.  One after the other / side by side: 64 sequences behind 8704 positions with 75
// to 300 own ones, 32 query and 8 kv heads 43.4 / 34.0 us; 256 behind 32768 with 65 to
// 257, 12 and 2 heads 73.1 / 62.9 us (55 us of it k_prefix, 5 us the join).
//
// k_prefix: a unit is a kv head and 256 rows (two tiles of M = 128; an odd last
// tile stands alone), its steps the prefix's 128-position tiles.  With fewer units
// than SMs each gets a whole number of CTAs, by its MMAs, which share its steps:
// a CTA that went on from one unit to the next would load queries and store
// partials twice (~5 us; a call with 8 units of 68 steps took 57 us so, 44 us with
// one unit a CTA).  With more, all steps stand in one row, weighted by their MMAs,
// and one CTA per SM takes an equal run of it (256 sequences behind 1000 positions, 64
// and 8 heads: 62 us; 1024 behind 32768, 32 and 8 heads: 571 us, 960 TFLOP/s).  Warps of a
// CTA:
//   0-7, 8-15  softmax of stream 0 and 1: a thread has half a row (64 scores) of S
//       from tensor memory, and puts the weights back over it as fp16 / bf16 (P);
//       the two halves of a row agree on its maximum through shared memory
//   16 producer: page table, TMA loads of tiles, three of K and two of V held, K's a
//       step ahead (in one ring of five, K of the second next step would wait for V of
//       this one)
//   17 MMA issue: S = Q K^T (smem x smem), O += P V (tensor memory x smem, V read
//       N-major as it lies in the pool)
// The two streams are the unit's two row tiles over the same K / V slots; a lone
// row tile runs alternate position tiles in each stream instead.  While one
// stream's softmax runs, the tensor core works for the other.  O stays in tensor
// memory; it is rescaled by its row's thread only when a score passes the row's
// reference by 2^15 (weights are 2^(s - r) with r = max - 7 when last moved, see
// paged_decode.cu).  A weight is rounded once to the cache's type (relative 2^-11 or 2^-8,
// averaged over positions).  With a second product of what that leaves, half as many MMAs
// again and twice the writes to tensor memory in a step whose chain is the bound, 64 x 8704
// take 42.5 us against 34.1, 256 x 32768 89.4 against 62.1, and V would have to be cleared of
// infinities.  Sums and outputs are fp32.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "paged_common.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kKSlots = 3, kVSlots = 2;    // tiles of K and of V held
constexpr uint32_t kSmemBytes = 227 * 1024;
constexpr int kPrefixThreads = 576;
constexpr int kProducer = 16, kIssuer = 17;
constexpr int kColS = 0, kColO = 256;      // tensor-memory columns: S0 S1 (P over S), O0 O1

struct PrefixArgs : PrefixSplit {
  PagedAttnArgs a;
  float scale_log2;                // above 0: a negative scale's sign is put on the queries
  uint32_t negate;                 // 0x80008000 then, else 0
  float* part_o;                   // [units + runs][2][128][D]
  float2* part_ml;                 // [units + runs][2][128]
  const float* own_o;              // [n_seq][n_heads][D]
  const float2* own_ml;
};

template <int D>
struct PrefixSmem {   // on a 1024-byte boundary
  uint8_t q[2][kRows * D * 2];             // [half][row][128 B], swizzled
  uint8_t k[kKSlots][kPos * D * 2], v[kVSlots][kPos * D * 2];
  uint64_t kfull[kKSlots], kempty[kKSlots], vfull[kVSlots], vempty[kVSlots], qfull[2], sfull[2], pfull[2], ofull[2], done;
  uint32_t groups[8];                      // of a step: 16-position groups that are there (read after K's slot is free)
  float top[2][2][kRows];                  // [stream][half][row]
  uint32_t tmem;
  int abort;
};

// ------------------------------------------------------------ tcgen05 PTX --
__device__ __forceinline__ void t5_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void t5_free(uint32_t t) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(t) : "memory");
}
__device__ __forceinline__ void t5_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void t5_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void t5_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void t5_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void t5_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
#define T5_R32(v) \
  "=r"((v)[0]), "=r"((v)[1]), "=r"((v)[2]), "=r"((v)[3]), "=r"((v)[4]), "=r"((v)[5]), "=r"((v)[6]), "=r"((v)[7]), \
  "=r"((v)[8]), "=r"((v)[9]), "=r"((v)[10]), "=r"((v)[11]), "=r"((v)[12]), "=r"((v)[13]), "=r"((v)[14]), \
  "=r"((v)[15]), "=r"((v)[16]), "=r"((v)[17]), "=r"((v)[18]), "=r"((v)[19]), "=r"((v)[20]), "=r"((v)[21]), \
  "=r"((v)[22]), "=r"((v)[23]), "=r"((v)[24]), "=r"((v)[25]), "=r"((v)[26]), "=r"((v)[27]), "=r"((v)[28]), \
  "=r"((v)[29]), "=r"((v)[30]), "=r"((v)[31])
#define T5_RW32(v) \
  "+r"((v)[0]), "+r"((v)[1]), "+r"((v)[2]), "+r"((v)[3]), "+r"((v)[4]), "+r"((v)[5]), "+r"((v)[6]), "+r"((v)[7]), \
  "+r"((v)[8]), "+r"((v)[9]), "+r"((v)[10]), "+r"((v)[11]), "+r"((v)[12]), "+r"((v)[13]), "+r"((v)[14]), \
  "+r"((v)[15]), "+r"((v)[16]), "+r"((v)[17]), "+r"((v)[18]), "+r"((v)[19]), "+r"((v)[20]), "+r"((v)[21]), \
  "+r"((v)[22]), "+r"((v)[23]), "+r"((v)[24]), "+r"((v)[25]), "+r"((v)[26]), "+r"((v)[27]), "+r"((v)[28]), \
  "+r"((v)[29]), "+r"((v)[30]), "+r"((v)[31])
#define T5_IN32(v) \
  "r"((v)[0]), "r"((v)[1]), "r"((v)[2]), "r"((v)[3]), "r"((v)[4]), "r"((v)[5]), "r"((v)[6]), "r"((v)[7]), \
  "r"((v)[8]), "r"((v)[9]), "r"((v)[10]), "r"((v)[11]), "r"((v)[12]), "r"((v)[13]), "r"((v)[14]), "r"((v)[15]), \
  "r"((v)[16]), "r"((v)[17]), "r"((v)[18]), "r"((v)[19]), "r"((v)[20]), "r"((v)[21]), "r"((v)[22]), "r"((v)[23]), \
  "r"((v)[24]), "r"((v)[25]), "r"((v)[26]), "r"((v)[27]), "r"((v)[28]), "r"((v)[29]), "r"((v)[30]), "r"((v)[31])
// 32 columns of this thread's lane; the values are there after t5_landed on them.
__device__ __forceinline__ void t5_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : T5_R32(v)
      : "r"(addr));
}
__device__ __forceinline__ void t5_ld16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
  for (int x = 16; x < 32; ++x) v[x] = 0;
}
__device__ __forceinline__ void t5_landed(uint32_t* v) {   // names the registers: no use of them moves before it
  asm volatile("tcgen05.wait::ld.sync.aligned;" : T5_RW32(v)::"memory");
}
__device__ __forceinline__ void t5_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::T5_IN32(v),
      "r"(addr)
      : "memory");
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// Eight columns times f, in place (few registers: the caller holds 64 scores).
__device__ __forceinline__ void t5_scale8(uint32_t addr, float f) {
  uint32_t v[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])::"memory");
#pragma unroll
  for (int x = 0; x < 8; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * f);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(addr)
               : "memory");
}
// Sixteen columns, those from `valid` on overwritten with `none`.
__device__ __forceinline__ void t5_mask16(uint32_t addr, int valid, uint32_t none) {
#pragma unroll 1
  for (int x = max(valid, 0); x < 16; ++x)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr + x), "r"(none) : "memory");
}
__device__ __forceinline__ void t5_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of the warp; the branch on it is warp-uniform to the compiler, which
// keeps descriptors in uniform registers.
__device__ __forceinline__ bool t5_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Shared-memory matrix descriptors, 128-byte swizzle, version 1.  K-major: 8-row
// groups 1024 B apart.  N-major (V as [position][64 elements]): 8-position groups
// 1024 B apart (SBO), the next 64 elements kPos * 128 B on (LBO).
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_n(uint32_t addr) {
  return desc_k(addr) | ((uint64_t)((kPos * 128) >> 4) << 16);
}
// kind::f16: fp32 accumulator; A and B both fp16 or both bf16; B N-major if nmajor.
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_of(int n, bool nmajor) {
  const uint32_t bf = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (bf << 7) | (bf << 10) | ((nmajor ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kRows >> 4) << 24);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPrefixThreads, 1)
    k_prefix(const __grid_constant__ PrefixArgs p, int box_rows, const __grid_constant__ CUtensorMap tmk,
             const __grid_constant__ CUtensorMap tmv) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;   // 0: nothing lies before it
  const PagedAttnArgs& a = p.a;
  if (pad + sizeof(PrefixSmem<D>) > kSmemBytes) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadArgument);
    return;
  }
  PrefixSmem<D>& s = *reinterpret_cast<PrefixSmem<D>*>(smem_raw + pad);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x, G = gridDim.x;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kKSlots; ++i) {
      mbar_init(&s.kfull[i], 1);
      mbar_init(&s.kempty[i], 1);
    }
    for (int i = 0; i < kVSlots; ++i) {
      mbar_init(&s.vfull[i], 1);
      mbar_init(&s.vempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.qfull[i], 8);
      mbar_init(&s.sfull[i], 1);
      mbar_init(&s.pfull[i], 8);
      mbar_init(&s.ofull[i], 1);
    }
    mbar_init(&s.done, 1);
    s.abort = 0;
    fence_mbar_init();
  }
  if (warp == kIssuer) t5_alloc(&s.tmem);
  t5_before();
  __syncthreads();
  t5_after();
  const uint32_t tmem = s.tmem;
  Pieces piece(p, c, G);
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();

  if (warp == kProducer) {
    // ------------------------------------------------------------ producer --
    const int P = a.kv.page_size, boxes = kPos / box_rows, halves = D / 64;
    uint32_t nk = 0, nv = 0;   // tiles loaded so far
    bool alive = true;
    // lane: box lane / halves of a tile, half lane % halves
    const int box = lane / halves, half = lane % halves;
    const bool loads = box < boxes;
    const int at = half * kPos * 128 + box * box_rows * 128;   // in a slot
    while (alive && piece.next()) {
      const int h = piece.h, i0 = piece.i0, i1 = piece.i1;
      int page = 0, next_page = 0;
      // K of a step goes before V of the one before: a K slot is free as soon as its
      // products are formed, and the stream that waits for it is not to wait for the
      // weights that free a V slot.
      for (int step = i0; step <= i1 && alive; ++step) {
        if (step < i1) {
          const int pos = step * kPos + box * box_rows;
          next_page = (int)a.kv.n_pages;   // outside the pool: the box is filled with zeros
          bool there = false;
          if (loads && pos < (int)a.prefix_len) {
            const int x = a.prefix_pages[pos >> a.page_shift];
            there = x >= 0 && (uint32_t)x < a.kv.n_pages;
            if (there) next_page = x;
            else raise_error(a.err, kDevBadArgument);
          }
          const uint32_t have = __ballot_sync(0xffffffffu, there && half == 0);
          const int slot = nk % kKSlots;
          if (nk >= kKSlots &&
              !__all_sync(0xffffffffu, paged_wait(&s.kempty[slot], (nk / kKSlots - 1) & 1, &s.abort, a.err))) {
            alive = false;
            break;
          }
          if (lane == 0) {
            uint32_t groups = 0;
            for (int b = 0; b < boxes; ++b)
              if (have >> (b * halves) & 1) groups |= ((1u << (box_rows / 16)) - 1) << (b * box_rows / 16);
            s.groups[nk % 8] = groups;
            mbar_arrive_expect_tx(&s.kfull[slot], kPos * D * 2);
          }
          __syncwarp();
          if (loads) tma_load_half(s.k[slot] + at, &tmk, pos & (P - 1), half, h, next_page, &s.kfull[slot]);
          ++nk;
        }
        if (step > i0) {
          const int slot = nv % kVSlots;
          if (nv >= kVSlots &&
              !__all_sync(0xffffffffu, paged_wait(&s.vempty[slot], (nv / kVSlots - 1) & 1, &s.abort, a.err))) {
            alive = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&s.vfull[slot], kPos * D * 2);
          __syncwarp();
          const int pos = (step - 1) * kPos + box * box_rows;
          if (loads) tma_load_half(s.v[slot] + at, &tmv, pos & (P - 1), half, h, page, &s.vfull[slot]);
          ++nv;
        }
        page = next_page;
      }
    }
    __syncwarp();
    // Every issued copy lands before the CTA may exit.
    for (uint32_t j = nk > kKSlots ? nk - kKSlots : 0; j < nk; ++j)
      paged_wait(&s.kfull[j % kKSlots], (j / kKSlots) & 1, &s.abort, a.err, false);
    for (uint32_t j = nv > kVSlots ? nv - kVSlots : 0; j < nv; ++j)
      paged_wait(&s.vfull[j % kVSlots], (j / kVSlots) & 1, &s.abort, a.err, false);
  } else if (warp == kIssuer) {
    // ----------------------------------------------------------------- MMA --
    constexpr uint32_t id_s = idesc_of<T>(kPos, false), id_o = idesc_of<T>(D, true);
    uint32_t base = 0, qcount[2] = {0, 0}, pcount[2] = {0, 0};
    bool alive = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, paged_wait(bar, parity, &s.abort, a.err));
    };
    while (alive && piece.next()) {
      const int i0 = piece.i0, n = piece.i1 - i0, w = piece.w;
      // stream i's k-th step: k, or (a lone row tile) 2 k + i
      const int cnt[2] = {w == 2 ? n : (n + 1) / 2, w == 2 ? n : n / 2};
      auto step_of = [&](int i, int k) { return w == 2 ? k : 2 * k + i; };
      auto qk = [&](int i, int k) {   // the K tile has landed
        const uint32_t slot = (base + step_of(i, k)) % kKSlots;
        if (t5_elect()) {
          // +32 B of d an MMA inside the 128-byte rows, then the other half
          const uint64_t qd = desc_k(smem_u32(s.q[i])), kd = desc_k(smem_u32(s.k[slot]));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            t5_mma_ss(tmem + kColS + 128 * i, qd + (kk >> 2) * (kRows * 128 >> 4) + (kk & 3) * 2,
                      kd + (kk >> 2) * (kPos * 128 >> 4) + (kk & 3) * 2, id_s, kk > 0);
          t5_commit(&s.sfull[i]);
          if (w == 1 || i == 1) t5_commit(&s.kempty[slot]);
        }
        __syncwarp();
      };
      auto pv = [&](int i, int k) -> bool {
        const uint32_t slot = (base + step_of(i, k)) % kVSlots;
        // One wait for P, its V tile and the stream's next K tile: a wait on a completed
        // barrier takes ~150 cycles while MMAs run, so a softmax warp makes the other two.
        if (!wait(&s.pfull[i], pcount[i]++ & 1)) return false;
        t5_after();
        const int valid = (int)a.prefix_len - (i0 + step_of(i, k)) * kPos;   // positions of the tile
        if (valid < kPos && (w == 1 || i == 0)) {
          // past the prefix's end a page holds anything, and 0 weight times NaN is NaN
          for (int x = valid * 8 + lane; x < kPos * 8; x += 32)
#pragma unroll
            for (int half = 0; half < D / 64; ++half)
              *reinterpret_cast<uint4*>(s.v[slot] + half * kPos * 128 + x * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
          __syncwarp();
        }
        if (t5_elect()) {
          const uint64_t vd = desc_n(smem_u32(s.v[slot]));   // +16 positions of 128 B an MMA
#pragma unroll
          for (int kk = 0; kk < kPos / 16; ++kk)
            t5_mma_ts(tmem + kColO + 128 * i, tmem + kColS + 128 * i + 8 * kk, vd + kk * (2048 >> 4), id_o,
                      k > 0 || kk > 0);
          t5_commit(&s.ofull[i]);
          if (w == 1 || i == 1) t5_commit(&s.vempty[slot]);
        }
        __syncwarp();
        return true;
      };
      for (int i = 0; i < 2 && alive; ++i)
        if (cnt[i] > 0) alive = wait(&s.qfull[i], qcount[i]++ & 1);
      t5_after();
      for (int i = 0; i < 2 && alive; ++i)
        if (cnt[i] > 0) {
          const uint32_t ld = base + step_of(i, 0);
          alive = wait(&s.kfull[ld % kKSlots], (ld / kKSlots) & 1);
          t5_after();
          if (alive) qk(i, 0);
        }
      for (int k = 0; k < cnt[0] && alive; ++k)
        for (int i = 0; i < 2 && alive; ++i) {
          if (k < cnt[i]) alive = pv(i, k);
          if (alive && k + 1 < cnt[i]) qk(i, k + 1);
        }
      base += n;
    }
    // All MMAs have completed before tensor memory is freed.
    if (lane == 0) t5_commit(&s.done);
    __syncwarp();
    paged_wait(&s.done, 0, &s.abort, a.err, false);
  } else {
    // ------------------------------------------------------------- softmax --
    // On a wait that ran out the loop goes on (every later wait gives up at once), so
    // that the two warps of a row block keep meeting at their barrier.
    const int i = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + kColS + 128 * i + 64 * half, tp = tmem + lanes + kColS + 128 * i + 32 * half;
    const uint32_t to = tmem + lanes + kColO + 128 * i + D / 2 * half;
    const int pair_bar = 1 + i * 4 + (warp & 3);
    uint32_t base = 0, scount = 0, ocount = 0;
    auto wait = [&](uint64_t* bar, uint32_t parity) { paged_wait(bar, parity, &s.abort, a.err); __syncwarp(); };
    while (piece.next()) {
      const int i0 = piece.i0, n = piece.i1 - i0, w = piece.w, pair = piece.pair, h = piece.h;
      const int cnt = w == 2 ? n : i == 0 ? (n + 1) / 2 : n / 2;
      // this thread's half row of Q into shared memory
      const int r = (2 * pair + (w == 2 ? i : 0)) * kRows + row;   // of the kv head's rows
      // (a warp takes 16 whole rows of the stream's 128, lanes side by side)
      if (cnt > 0) {
        constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kLoads = 16 / kAtOnce;   // lanes of a row, rows of a load
        const int row0 = (warp & 7) * kWarpRows, x = lane % kLanes;
        // lane l < 16 finds row l's place
        const int r_of = r - row + row0 + (lane & 15);
        const long long at = r_of < p.rows ? (long long)(r_of / p.group) * a.q_stride + (long long)(h * p.group + r_of % p.group) * D : -1;
        uint4 v[kLoads];
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
          const long long src = __shfl_sync(0xffffffffu, at, q * kAtOnce + lane / kLanes);
          v[q] = src >= 0 ? *reinterpret_cast<const uint4*>(a.q + src + 8 * x) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
          const int rr = row0 + q * kAtOnce + lane / kLanes;
          const uint32_t m = p.negate;
          *reinterpret_cast<uint4*>(s.q[i] + query_byte(rr, x)) =
              make_uint4(v[q].x ^ m, v[q].y ^ m, v[q].z ^ m, v[q].w ^ m);
        }
        fence_proxy_async();
        t5_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.qfull[i]);
      }
      float ref = -INFINITY, sum = 0.f;
      for (int k = 0; k < cnt; ++k) {
        const int step = w == 2 ? k : 2 * k + i;
        if ((warp & 7) == 0) {   // for the issuer: this step's V tile, the stream's next K tile
          const uint32_t ld = base + step, next = base + (w == 2 ? k + 1 : 2 * k + 2 + i);
          wait(&s.vfull[ld % kVSlots], (ld / kVSlots) & 1);
          if (k + 1 < cnt) wait(&s.kfull[next % kKSlots], (next / kKSlots) & 1);
        }
        wait(&s.sfull[i], scount++ & 1);
        t5_after();
        const uint32_t groups = s.groups[(base + step) % 8] >> (4 * half);
        const int valid = (int)a.prefix_len - (i0 + step) * kPos - 64 * half;
        const bool whole = (groups & 15u) == 15u && valid >= 64;
        if (!whole) {   // scores of what is not there never win: written back over S
          const uint32_t none = __float_as_uint(-INFINITY);
#pragma unroll 1
          for (int x = 0; x < 64; x += 16) t5_mask16(ts + x, groups >> (x / 16) & 1 ? valid - x : 0, none);
          t5_stored();
        }
        uint32_t w2[32];
        float add;
        // Weights against reference `off`, their sum, and the greatest score.
        auto weigh = [&](float off) -> float {
          uint32_t v[64];
          t5_ld32(ts, v);
          t5_ld32(ts + 32, v + 32);
          float mx[4];
          float2 part[2] = {};
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = -INFINITY;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            t5_landed(v + 32 * b);
#pragma unroll
            for (int x = 32 * b; x < 32 * b + 32; x += 2) {
              const float2 s = make_float2(__uint_as_float(v[x]), __uint_as_float(v[x + 1]));
              mx[x / 2 & 3] = fmaxf(mx[x / 2 & 3], fmaxf(s.x, s.y));
              float2 e = fma2(s, make_float2(p.scale_log2, p.scale_log2), make_float2(-off, -off));
              e.x = exp2_fast(e.x);
              e.y = exp2_fast(e.y);
              part[x / 2 & 1] = add2(part[x / 2 & 1], e);
              w2[x / 2] = pack2(T{}, e.x, e.y);
            }
          }
          add = (part[0].x + part[0].y) + (part[1].x + part[1].y);
          return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
        };
        // The reference holds for nearly every tile, so the weights are formed with it
        // while the maximum is still being found, and again where it had to move.
        const float mine = weigh(ref == -INFINITY ? 0.f : ref);
        // The row's other half; also: both halves have read S before either writes P.
        // (They have read the last step's maxima: the next S takes both their P.)
        float* tops = &s.top[i][0][row];
        tops[kRows * half] = mine;
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        const float top = fmaxf(tops[0], tops[kRows]);
        const bool grown = top > ref + 15.f;
        if (__any_sync(0xffffffffu, grown)) {   // the same in both halves
          const float now = grown ? top - 7.f : ref;
          const float f = ref == now ? 1.f : exp2_fast(ref - now);
          ref = now;
          sum *= f;
          if (k > 0) {
            wait(&s.ofull[i], (ocount - 1) & 1);   // the last O += P V has completed
            t5_after();
#pragma unroll 1
            for (int q = 0; q < D / 2; q += 8) t5_scale8(to + q, f);
          }
          weigh(ref == -INFINITY ? 0.f : ref);
          asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");   // S is read again before P
        }
        t5_st32(tp, w2);
        sum += add;
        t5_stored();
        t5_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.pfull[i]);
        ++ocount;
      }
      // the stream's partial: the first half adds up the sums
      const long long slot = ((long long)piece.id * 2 + i) * kRows + row;
      if (cnt > 0) {
        wait(&s.ofull[i], (ocount - 1) & 1);
        t5_after();
      }
      if (cnt > 0) {
        float* sums = &s.top[i][0][row];
        if (half == 1) sums[0] = sum;
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        if (half == 0) sum += sums[0];
      }
      if (half == 0 && r < p.rows) p.part_ml[slot] = make_float2(ref, sum);
      // O through this warp's bytes of the query tile (stage_byte), whose MMAs are done,
      // so that rows go out in whole 128-byte lines.
      if (cnt > 0) {
        constexpr int kCols = D / 4;   // fp32 columns a round: 4 KB (2 KB) of 32 rows
        static_assert(32 * kCols * 4 == kRows * D * 2 / 8, "a warp's share of the query tile");
#pragma unroll 1
        for (int q = 0; q < 2; ++q) {
          uint32_t o[32];
          if constexpr (kCols == 32) t5_ld32(to + kCols * q, o);
          else t5_ld16(to + kCols * q, o);
          t5_landed(o);
          constexpr int kChunks = kCols / 4;
#pragma unroll
          for (int x = 0; x < kChunks; ++x)
            *reinterpret_cast<uint4*>(s.q[i] + stage_byte(D, warp & 7, lane, x)) =
                make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          __syncwarp();
          const int rows_here = p.rows - (r - lane);   // of this warp's 32
#pragma unroll
          for (int x = 0; x < kChunks; ++x) {
            const int rr = x * (32 / kChunks) + lane / kChunks, ch = lane % kChunks;
            const uint4 v = *reinterpret_cast<const uint4*>(s.q[i] + stage_byte(D, warp & 7, rr, ch));
            if (rr < rows_here)
              *reinterpret_cast<uint4*>(p.part_o + (slot - lane + rr) * D + D / 2 * half + kCols * q + 4 * ch) = v;
          }
          __syncwarp();
        }
      }
      t5_before();
      base += n;
    }
  }
  t5_before();
  __syncthreads();
  if (warp == kIssuer) t5_free(tmem);
}

// One warp per query row: its own part and the prefix's partials, in order.  What it
// reads it asks for at once, eight partials at a time: the kernel is one round
// trip or two to L2.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_prefix_join(const __grid_constant__ PrefixArgs p, int G) {
  constexpr int V = D / 32, kAtOnce = 8;
  const PagedAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const bool mine = id < (long long)a.kv.n_seq * a.n_heads;
  const int seq = mine ? (int)(id / a.n_heads) : 0, head = mine ? (int)(id - (long long)seq * a.n_heads) : 0;
  const int h = head / p.group, r = seq * p.group + head - h * p.group;
  const Partials part(p, h, r / kRows, G);
  const int n = part.n;
  auto slot_of = [&](int k) { return part.slot(k) * kRows + r % kRows; };
  pdl_wait();
  if (!mine) return;
  const uint32_t L = a.seq_len[seq];
  const float2 own = p.own_ml[id];
  float M = own.x, sum = own.y, v[V];
  load_vec(v, p.own_o + id * D + V * lane);
  for (int b = 0; b < n; b += 32) {
    const int m = min(32, n - b);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < m) {
      ml = __ldcg(p.part_ml + slot_of(b + lane));
      if (!part.there(p, b + lane, G)) ml = make_float2(-INFINITY, 0.f);
    }
    float f = 0.f;
    for (int k0 = 0; k0 < m; k0 += kAtOnce) {
      float x[kAtOnce][V];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q)
        load_vec(x[q], p.part_o + (long long)slot_of(b + min(k0 + q, m - 1)) * D + V * lane);
      if (k0 == 0) {
        const bool some = ml.y != 0.f;   // NaN counts as some
        const float m1 = fmaxf(sum == 0.f ? -INFINITY : M, warp_max(some ? ml.x : -INFINITY));
        const float f0 = sum == 0.f ? 0.f : exp2_fast(M - m1);
        f = some ? exp2_fast(ml.x - m1) : 0.f;
        M = m1;
        sum = sum * f0 + warp_sum(ml.y * f);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = f0 == 0.f ? 0.f : v[k] * f0;
      }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const float fq = __shfl_sync(0xffffffffu, f, (k0 + q) & 31);
        if (k0 + q < m && fq != 0.f) {   // what no piece has written is not read into the sum
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] += x[q][k] * fq;
        }
      }
    }
  }
  if (L > a.kv.max_pages * a.kv.page_size) return;   // reported by the own-positions kernel
  write_row<T, D>(a, seq, head, as_float4(v), M, sum, lane);
}

template <typename T, int D>
int launch(const PrefixArgs& p, const PagedOwn& own, int G, const CUtensorMap& tmk, const CUtensorMap& tmv, int box_rows,
           cudaStream_t st) {
  auto kern = k_prefix<T, D>;
  const int smem = (int)kSmemBytes;
  static_assert(sizeof(PrefixSmem<D>) <= kSmemBytes - 768, "shared memory");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(G);
  cfg.blockDim = dim3(kPrefixThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static OncePerDevice once;
  if (once.launch(reinterpret_cast<const void*>(kern), smem, [&] {
        return cudaLaunchKernelEx(&cfg, kern, p, box_rows, tmk, tmv);
      }) != cudaSuccess)
    return -1;
  if (launch_paged_decode(p.a, st, own) != 0) return -1;
  const long long rows = (long long)p.a.kv.n_seq * p.a.n_heads;
  cfg.gridDim = dim3((unsigned)((rows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, k_prefix_join<T, D>, p, G) == cudaSuccess ? 0 : -1;
}

// How many tiles of own positions `few` CTAs finish by the time that the prefix is done
// and all CTAs would be: a CTA takes 0.75 us a tile and 0.85 us a unit.  (Own positions
// divided among all CTAs whatever their number: 256 behind 32768 75 us against 64,
// since those that find room at first have only their equal shares.)
uint32_t own_tiles(const PrefixSplit& p, const qwen_paged_kv& kv, int few, double us) {
  const double units = (double)kv.n_seq * kv.n_kv_heads * ((p.group + 15) / 16);
  return (uint32_t)std::max(0.0, std::min(2e9, (few * (us + 8) - 0.85 * units) / 0.75));
}

struct Layout {
  size_t own_o, own_ml, part_o, part_ml, bytes;   // offsets after the decode kernel's part
};
Layout layout(const PrefixSplit& p, const qwen_paged_kv& kv, int n_heads, int G) {
  const size_t heads = (size_t)kv.n_seq * n_heads, D = kv.head_dim;
  const size_t slots = ((size_t)kv.n_kv_heads * p.pairs + G) * 2 * kRows;
  Layout l;
  l.own_o = (paged_decode_workspace(kv, n_heads) + 255) / 256 * 256;
  l.own_ml = l.own_o + heads * D * 4;
  l.part_o = (l.own_ml + heads * 8 + 255) / 256 * 256;
  l.part_ml = l.part_o + slots * D * 4;
  l.bytes = l.part_ml + slots * 8;
  return l;
}

}  // namespace

size_t paged_prefix_workspace(const qwen_paged_kv& kv, int n_heads, uint32_t prefix_len) {
  if (prefix_len == 0) return paged_decode_workspace(kv, n_heads);
  PrefixSplit p{};
  const int G = plan_prefix(p, (int)kv.n_kv_heads, (int)kv.n_seq, n_heads, prefix_len, paged_sm_count());
  return layout(p, kv, n_heads, G).bytes;
}

int launch_paged_prefix(const PagedAttnArgs& a, cudaStream_t st) {
  PrefixArgs p{};
  p.a = a;
  const int G = plan_prefix(p, (int)a.kv.n_kv_heads, (int)a.kv.n_seq, a.n_heads, a.prefix_len, paged_sm_count());
  const Layout l = layout(p, a.kv, a.n_heads, G);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  PagedOwn own;
  p.own_o = own.o = reinterpret_cast<float*>(ws + l.own_o);
  p.own_ml = own.ml = reinterpret_cast<float2*>(ws + l.own_ml);
  own.few = std::max(1, 2 * (paged_sm_count() - G));   // two of its CTAs share an SM
  own.few_tiles = G < paged_sm_count() ? own_tiles(p, a.kv, own.few, prefix_us(p) / G) : 0;
  p.part_o = reinterpret_cast<float*>(ws + l.part_o);
  p.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  // (above 0, so that a masked score, -inf, stays one: products scaled so weigh alike)
  p.scale_log2 = std::max(std::fabs(a.scale) * kLog2e, 1e-37f);
  p.negate = a.scale < 0.f ? 0x80008000u : 0u;
  const int box_rows = a.kv.page_size < (uint32_t)kPos ? (int)a.kv.page_size : kPos;
  CUtensorMap tmk, tmv;
  if (encode_pages_map(&tmk, a.kv, a.kv.k, box_rows, 1) || encode_pages_map(&tmv, a.kv, a.kv.v, box_rows, 1)) return -1;
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16)
    return d64 ? launch<__half, 64>(p, own, G, tmk, tmv, box_rows, st) : launch<__half, 128>(p, own, G, tmk, tmv, box_rows, st);
  return d64 ? launch<__nv_bfloat16, 64>(p, own, G, tmk, tmv, box_rows, st)
             : launch<__nv_bfloat16, 128>(p, own, G, tmk, tmv, box_rows, st);
}

}  // namespace qwen
