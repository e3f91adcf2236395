// paged_q4_decode.cu -- decode attention over a 4-bit paged cache, one query token per
// sequence, and the weights that each cached slot was given:
//   out = sum_t softmax(scale q . K_t) V_t,  K_t, V_t = low + code step
//
// Work, runs of tiles, partials and their join: as in paged_decode.cu (paged_runs.cuh).  A
// tile is 128 slots, a unit (sequence, kv head, up to 8 query heads).  A CTA has a producer
// warp, which looks pages up and copies a tile's 8 blocks of 16 slots (codes and parameters of
// K and V lie side by side, so a copy takes all of a page's blocks in the tile), and 4 consumer
// warps, one a scheduler, each with two blocks of a tile, whose instructions fill one another's
// gaps.  Three such CTAs an SM leave a thread 128 registers.  (16 x 8704 of 8 kv heads, fp16,
// now 34 us, when it took 36: with runs of blocks 46; with 6 such warps in two CTAs, which the
// schedulers do not divide evenly, 51; with 12 in one, which all wait at a piece's end, 58.)
//
// What bounds it is not the bytes alone, 2.5 KB a block of 128-element heads, but the
// instructions that turn them into products; so nothing is dequantised.  Per block a warp
// computes, with m16n8k16 MMAs,
//   A_g[16 slots x 8 heads] = codes_g q_g^T for each group g of 32 elements,
//   S = sum_g step_g A_g + sum_g low_g (sum q_g),
// and with P = exp(S - reference)
//   o^T[d x 8] += codes^T (step_g P)^T,  o_g += sum_t P low_g  (added at the end).
// Codes are exact as MMA operands: four bits at the bottom of an fp16 are c 2^-24, so a
// word's eight keys take four ANDs and a shift (those from bits 4..7 are 16 c 2^-24; their
// query elements are divided by 16).  Queries are brought to 2^14 .. 2^15 a head by a power
// of two and are exact in fp16 but for what is 2^-33 of the head's largest.  For the values
// the codes are bf16.  Weights are at most 2^8, so that the sums over L slots are finite while
// L times the greatest value is below 10^35 (weights of at most 1, by a reference that is moved 8
// above the greatest score, would give 10^38, but not the very value where there is one slot).
// The sums of P with lows are one MMA over the slots, q's group sums with lows another (three
// terms of 8 or 11 bits).  Weights P and step P are two bf16 values (off by at most 2^-17 of one,
// a 64th of what fp16 outputs are rounded by).  Sums, maxima and outputs are fp32.  An MMA cuts
// its sum off, always toward zero, which over a run would add up, so that each tile's start from
// 0 and are added to the others' by additions that round (4% of a long call).
//
// Measured: 32 sequences of 16384 slots, 32 and 8 heads of 128, bf16: 161 us (4.2 TB/s), fp16
// 167; their 671 MB take 102.  A block takes a warp some 395 instructions (bf16, starts and
// joins included); with lengths of a quarter to all of that, 104 us, the schedulers issue 58% of
// the time, the integer pipe is busy for 46%, the tensor pipe for 31%.  8, 12 or 16 warps an SM,
// with 2 or 4 blocks at once, are within 6%.  A call of 512 slots takes 8.5, 64 sequences of
// 512 .. 2048 slots and 2 kv heads 16.4 (their bytes 3.8): launch, lengths, page numbers, first
// tile, join.  Warps that load their own blocks, sixteen an SM without producers, took 172 in
// place of 150 at that time.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_q4.cuh"
#include "paged_runs.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kWarps = 4;                     // consumer warps
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kBlocks = 2 * kWarps;           // of a tile: a warp takes two
static_assert(16 * kBlocks == 1 << 7, "tile");
constexpr int kTileShift = 7;
constexpr int kCtasPerSm = 3;
constexpr int kSlotHeads = 8;                 // query heads of a unit
constexpr int kQuerySlots = 4;

// A run's part of a unit.
struct Piece {
  int heads;           // query heads, or 0: the run has no more pieces
  int seq, head;       // sequence, first query head
  int dest;            // partial slot, or -1: the whole unit, or -2: nothing is written
  float2* scores;      // of the unit's slot 0, or null
};
struct StageMeta {
  int valid[kBlocks];  // slots of each block that count
  int first;           // the tile's first slot
  int last;            // of the piece
};

template <int D>
struct __align__(128) Q4DecodeSmem {
  static constexpr int kStages = D == 128 ? 3 : 6;
  uint8_t kv[kStages][kBlocks][Q4Block<D>::kBytes];
  uint16_t q[kQuerySlots][kSlotHeads * D];
  float2 ml[2][kWarps][kSlotHeads];   // by piece parity: maximum and sum of each warp
  Piece piece[kQuerySlots];
  StageMeta meta[kStages];
  uint64_t full[kStages], empty[kStages], qfull[kQuerySlots], qempty[kQuerySlots], joined, early;
  CutUnit cut[2];
  int n_cut, n_early;   // cut pieces; of those counted in before the end
  int runs;
  int last[2];
  int abort;
};

struct Q4DecodeArgs : DecodeArgs {
  qwen_paged_kv_q4 kv;
  float* scores;     // where weights are kept: [unit][capacity][2 score_pairs], log2 domain
  int score_pairs;   // query heads of a unit in pairs
};

__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }   // -126 <= e <= 127

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
// (step, low) of a word: its low and high half.
__device__ __forceinline__ float step_of(__half, uint32_t w) { return __low2float(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float step_of(__nv_bfloat16, uint32_t w) { return __uint_as_float(w << 16); }
// Weights times steps: the product rounded, and what that left of it and of the weight's rest.
__device__ __forceinline__ void step_weights(uint32_t hi, uint32_t rest, uint32_t step, uint32_t* w, uint32_t* left) {
  const __nv_bfloat162 h = *reinterpret_cast<__nv_bfloat162*>(&hi), e = *reinterpret_cast<__nv_bfloat162*>(&rest),
                       s = *reinterpret_cast<__nv_bfloat162*>(&step);
  const __nv_bfloat162 x = __hmul2(h, s), y = __hfma2(e, s, __hfma2(h, s, __hneg2(x)));
  *w = *reinterpret_cast<const uint32_t*>(&x);
  *left = *reinterpret_cast<const uint32_t*>(&y);
}
// Two fp32 values as two pairs of the type: rounded, and what that left.
template <typename T>
__device__ __forceinline__ void split2(float x, float y, uint32_t* hi, uint32_t* lo) {
  *hi = pack2(T{}, x, y);
  const float2 r = unpack2(T{}, *hi);
  *lo = pack2(T{}, x - r.x, y - r.y);
}

// D = A B + D, and from zeros (which need no registers).  Not volatile: what they depend on
// orders them.
#define QWEN_MMA(name, type)                                                                                   \
  __device__ __forceinline__ void mma_add(name, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." type "." type ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "  \
        "{%0,%1,%2,%3};"                                                                                       \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                       \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                       \
  }                                                                                                            \
  __device__ __forceinline__ void mma_zero(name, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." type "." type ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "  \
        "{%10,%10,%10,%10};"                                                                                   \
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                       \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));                             \
  }
QWEN_MMA(__half, "f16")
QWEN_MMA(__nv_bfloat16, "bf16")
#undef QWEN_MMA

// What a warp keeps of a unit's queries.
template <int D>
struct Queries {
  uint32_t f[D / 32][4];   // B operands: elements 8t + {0, 4}, {2, 6}, then {1, 5} / 16, {3, 7} / 16 of head g
  uint32_t sums[2];        // of groups (0, 1), (2, 3): term t of three
  float c1[2], c2[2];      // of heads 2t, 2t + 1: what a score in MMA units is multiplied with
};
// From rows of q in shared memory (lane 4 g + t: elements 8 t .. of each group of head g).
template <typename T, int D>
__device__ __forceinline__ void load_queries(Queries<D>& u, const T* q, int heads, float scale_log2, int lane) {
  constexpr int G = D / 32;
  const int g = lane >> 2, t = lane & 3;
  float x[G][8], top = 0.f;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (g < heads) w = *reinterpret_cast<const uint4*>(q + g * D + 32 * i + 8 * t);
    const float2 a = unpack2(T{}, w.x), b = unpack2(T{}, w.y), c = unpack2(T{}, w.z), d = unpack2(T{}, w.w);
    x[i][0] = a.x, x[i][1] = a.y, x[i][2] = b.x, x[i][3] = b.y, x[i][4] = c.x, x[i][5] = c.y, x[i][6] = d.x, x[i][7] = d.y;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int k = top > 0.f && top < INFINITY ? 14 - ilogbf(top) : 0;   // -113 .. 163
  const float f1 = pow2(k / 2), f2 = pow2(k - k / 2);
  float sum[4] = {};
#pragma unroll
  for (int i = 0; i < G; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[i][e] = x[i][e] * f1 * f2;
      sum[i] += x[i][e];
    }
    u.f[i][0] = pack2(__half{}, x[i][0], x[i][4]);
    u.f[i][1] = pack2(__half{}, x[i][2], x[i][6]);
    u.f[i][2] = pack2(__half{}, x[i][1] * 0.0625f, x[i][5] * 0.0625f);
    u.f[i][3] = pack2(__half{}, x[i][3] * 0.0625f, x[i][7] * 0.0625f);
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    sum[i] *= 0.015625f;   // at most 2^14: within fp16
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float a = sum[2 * i], b = sum[2 * i + 1];
    uint32_t r = 0;
#pragma unroll
    for (int term = 0; term < 3; ++term) {
      const uint32_t w = pack2(T{}, a, b);
      const float2 y = unpack2(T{}, w);
      a -= y.x;
      b -= y.y;
      if (term == t) r = w;
    }
    u.sums[i] = r;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int kk = 6 - __shfl_sync(0xffffffffu, k, 8 * t + 4 * e);
    u.c1[e] = pow2(kk / 2);
    u.c2[e] = pow2(kk - kk / 2) * scale_log2;
  }
}

// Codes of a word in fp16 units of 2^-24: elements (0, 4), (2, 6), then 16 times (1, 5), (3, 7).
__device__ __forceinline__ void small_codes(uint32_t w, uint32_t (&c)[4]) {
  const uint32_t v = w >> 8;
  c[0] = w & 0x000f000fu;
  c[1] = v & 0x000f000fu;
  c[2] = w & 0x00f000f0u;
  c[3] = v & 0x00f000f0u;
}
// Codes in bf16 of bits 4 j .. 4 j + 3 of both halves of a word, as they are and not with a bias
// that is taken off the sums: there it stood against weights that had been rounded otherwise
// (elements whose codes and lows are all 0 came out as 3e-6 in place of 0, bf16, 1000 slots; and
// 128 or 16 times a weight's error against a code of 7.5).
// fp16 caches: a code at the bottom of a bf16 is c 2^-133, for odd j 16 times that (bit 7, the
// exponent's first, counts on), and weights are brought to 2^kRaise: an AND for two codes.  The
// steps of bf16 caches leave no room for that: there 128 + code less 128, which is exact
// (32 x 16384: bf16 156 -> 161 us with it, fp16 171 -> 179 and without it 167).
constexpr int kRaise = 72;   // 2^(72 + 8 + 13 + 24) at most: weight, step, slots
template <typename T>
__device__ __forceinline__ uint32_t value_code(uint32_t w, int j) {
  if constexpr (std::is_same<T, __half>::value) return (j & 2 ? w >> 8 : w) & (j & 1 ? 0x00f000f0u : 0x000f000fu);
  const uint32_t v = lop3_and_or(w >> (4 * j), 0x000f000fu, 0x43004300u);
  const __nv_bfloat162 c = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(128.f));
  return *reinterpret_cast<const uint32_t*>(&c);
}

// Scores of a block, log2 domain: s = (slot g: heads 2t, 2t+1), (slot g + 8: the same).
// codes[half][group]: word t of slot 8 half + g; params the same slots' (step, low).
template <typename T, int D>
__device__ __forceinline__ void block_scores(const Queries<D>& u, const uint32_t (&codes)[2][D / 32],
                                             const uint32_t (&params)[2][D / 32], float (&s)[4]) {
  constexpr int G = D / 32;
  float low[4], sum[4];
  uint32_t a[4];
  a[0] = prmt(params[0][0], params[0][1], 0x7632);
  a[1] = prmt(params[1][0], params[1][1], 0x7632);
  a[2] = a[3] = 0;
  if constexpr (G == 4) {
    a[2] = prmt(params[0][2], params[0][3], 0x7632);
    a[3] = prmt(params[1][2], params[1][3], 0x7632);
  }
  mma_zero(T{}, low, a, u.sums[0], u.sums[1]);
#pragma unroll
  for (int i = 0; i < G; ++i) {
    uint32_t x[4], y[4];
    small_codes(codes[0][i], x);
    small_codes(codes[1][i], y);
    const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
    float d[4];
    mma_zero(__half{}, d, a0, u.f[i][0], u.f[i][1]);
    mma_add(__half{}, d, a1, u.f[i][2], u.f[i][3]);
    const float s0 = step_of(T{}, params[0][i]), s1 = step_of(T{}, params[1][i]);
    sum[0] = i ? fmaf(d[0], s0, sum[0]) : d[0] * s0;
    sum[1] = i ? fmaf(d[1], s0, sum[1]) : d[1] * s0;
    sum[2] = i ? fmaf(d[2], s1, sum[2]) : d[2] * s1;
    sum[3] = i ? fmaf(d[3], s1, sum[3]) : d[3] * s1;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = fmaf(sum[e], 262144.f, low[e]) * u.c1[e & 1] * u.c2[e & 1];
}

// What a warp keeps of a unit.
template <int D>
struct Stream {
  Queries<D> u;
  float o[D / 32][2][4];      // element 32 i + 4 g + 2 j of heads 2t, 2t + 1, then the next one
  float extra[4];             // sums of weights with lows (row g: of group g; fp16: and g - 4)
  float m[2], ref[2], l[2];   // of heads 2t, 2t + 1; ref: m, or 0 where there is none
};

// Takes kN blocks in.  valid: their slots that count (of blocks[0] there may be none);
// scores: where blocks[0]'s go, blocks[1]'s 16 kWarps slots behind, or null.
template <typename T, int D, int kN>
__device__ __forceinline__ void take_blocks(Stream<D>& w, uint8_t* const (&blocks)[2], const int (&valid)[2], int lane,
                                            float2* scores, int score_pairs) {
  using Block = Q4Block<D>;
  constexpr int G = D / 32;
  constexpr bool kF16 = std::is_same<T, __half>::value;
  const int g = lane >> 2, t4 = lane & 3;
  const bool whole = kN == 2 ? valid[0] + valid[1] == 32 : valid[0] == 16;
  if (!whole) {
    // what lies behind the end may be anything, and 0 weight times NaN would be NaN
#pragma unroll
    for (int n = 0; n < kN; ++n)
      for (int i = lane; i < 16 * G; i += 32)
        if ((i & 15) >= valid[n]) reinterpret_cast<uint32_t*>(blocks[n] + Block::kValueSteps)[i] = 0;
    __syncwarp();
  }
  // ---- scores: lane 4 g + t has word t of slots g and g + 8
  float sv[kN][4];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const uint32_t at = smem_u32(blocks[n]);
    uint32_t codes[2][G], params[2][G], r[4];
    if constexpr (G == 4) {
      const uint32_t row = at + (lane >> 3) * 256 + (lane & 7) * 16;
      ldmatrix_x4(r, row);
#pragma unroll
      for (int i = 0; i < 4; ++i) codes[0][i] = r[i];
      ldmatrix_x4(r, row + 128);
#pragma unroll
      for (int i = 0; i < 4; ++i) codes[1][i] = r[i];
    } else {
      ldmatrix_x4(r, at + lane * 16);   // group 0: slots 0 .. 7, 8 .. 15, group 1
      codes[0][0] = r[0], codes[1][0] = r[1], codes[0][1] = r[2], codes[1][1] = r[3];
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
      params[0][i] = lds32(at + Block::kKeySteps + i * 64 + g * 4);
      params[1][i] = lds32(at + Block::kKeySteps + i * 64 + 32 + g * 4);
    }
    block_scores<T, D>(w.u, codes, params, sv[n]);
  }
  if (!whole) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (g >= valid[n]) sv[n][0] = sv[n][1] = -INFINITY;
      if (g + 8 >= valid[n]) sv[n][2] = sv[n][3] = -INFINITY;
    }
  }
  if (scores && t4 < score_pairs) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
      if (valid[n] > 0) {
        float2* to = scores + (16 * kWarps * n + g) * score_pairs + t4;
        to[0] = make_float2(sv[n][0], sv[n][1]);
        to[8 * score_pairs] = make_float2(sv[n][2], sv[n][3]);
      }
  }
  // ---- the running reference moves when a score passes it by 8
  float mx[2] = {fmaxf(sv[0][0], sv[0][2]), fmaxf(sv[0][1], sv[0][3])};
  if constexpr (kN == 2) {
    mx[0] = fmaxf(mx[0], fmaxf(sv[1][0], sv[1][2]));
    mx[1] = fmaxf(mx[1], fmaxf(sv[1][1], sv[1][3]));
  }
  if (__any_sync(0xffffffffu, mx[0] > w.m[0] + 8.f || mx[1] > w.m[1] + 8.f)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = mx[e];
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
      const float r = fmaxf(w.m[e], x);
      const float f = r == -INFINITY ? 1.f : exp2_fast(w.m[e] - r);
      w.m[e] = r;
      w.ref[e] = r == -INFINITY ? 0.f : r;
      w.l[e] *= f;
      w.extra[e] *= f;
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          w.o[i][j][e] *= f;
          w.o[i][j][2 + e] *= f;
        }
    }
  }
  // ---- weights, turned: lane 4 g + t has head g, slots 2t, 2t+1 and 8 + those
  uint32_t h0[kN], h1[kN], e0[kN], e1[kN];   // in bf16, and what rounding left
  float pw[kN][4];                           // fp16: the weights themselves, raised
  uint32_t vs[kN];
  float extra[4];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    vs[n] = smem_u32(blocks[n]) + Block::kValueSteps + t4 * 8;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      sv[n][e] = exp2_fast(sv[n][e] - w.ref[e]);
      sv[n][2 + e] = exp2_fast(sv[n][2 + e] - w.ref[e]);
      w.l[e] += sv[n][e] + sv[n][2 + e];
    }
    if constexpr (kF16) {
      const uint32_t x0 = movmatrix(prmt(__float_as_uint(sv[n][0]), __float_as_uint(sv[n][1]), 0x7632));
      const uint32_t y0 = movmatrix(prmt(__float_as_uint(sv[n][0]), __float_as_uint(sv[n][1]), 0x5410));
      const uint32_t x1 = movmatrix(prmt(__float_as_uint(sv[n][2]), __float_as_uint(sv[n][3]), 0x7632));
      const uint32_t y1 = movmatrix(prmt(__float_as_uint(sv[n][2]), __float_as_uint(sv[n][3]), 0x5410));
      pw[n][0] = __uint_as_float(prmt(y0, x0, 0x5410)) * pow2(kRaise);
      pw[n][1] = __uint_as_float(prmt(y0, x0, 0x7632)) * pow2(kRaise);
      pw[n][2] = __uint_as_float(prmt(y1, x1, 0x5410)) * pow2(kRaise);
      pw[n][3] = __uint_as_float(prmt(y1, x1, 0x7632)) * pow2(kRaise);
      split2<__nv_bfloat16>(pw[n][0], pw[n][1], &h0[n], &e0[n]);
      split2<__nv_bfloat16>(pw[n][2], pw[n][3], &h1[n], &e1[n]);
    } else {
      split2<T>(sv[n][0], sv[n][1], &h0[n], &e0[n]);
      split2<T>(sv[n][2], sv[n][3], &h1[n], &e1[n]);
      h0[n] = movmatrix(h0[n]);
      h1[n] = movmatrix(h1[n]);
      e0[n] = movmatrix(e0[n]);
      e1[n] = movmatrix(e1[n]);
    }
    // Sums of weights with lows: row g is the low of group g.  Weights as bf16, whatever the
    // cache's type: fp16 ends at 2^-24, and sums over thousands of slots far below the heaviest
    // lose what lies under it.  Lows of fp16 are two bf16 each, the second in rows 4 ..
    uint32_t x[4] = {};
    const int i = kF16 ? g & 3 : g;
    if (i < G) {
      const uint2 v0 = lds64(vs[n] + i * 64), v1 = lds64(vs[n] + i * 64 + 32);
      x[0] = prmt(v0.x, v0.y, 0x7632);
      x[2] = prmt(v1.x, v1.y, 0x7632);
      if constexpr (kF16) {   // the 8 bits that cutting it to bf16 leaves, or the others
        const uint32_t cut = g < 4 ? 0 : 0xffff0000u;
        auto part = [&](float y) { return __float_as_uint(y - __uint_as_float(__float_as_uint(y) & cut)); };
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const float2 low = unpack2(T{}, x[k]);
          x[k] = prmt(part(low.x), part(low.y), 0x7632);
        }
      }
    }
    if (n == 0) mma_zero(__nv_bfloat16{}, extra, x, h0[n], h1[n]);
    else mma_add(__nv_bfloat16{}, extra, x, h0[n], h1[n]);
    mma_add(__nv_bfloat16{}, extra, x, e0[n], e1[n]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) w.extra[e] += extra[e];
  // ---- o^T += codes^T (step weights)^T
#pragma unroll
  for (int pair = 0; pair < G / 2; ++pair) {
    uint32_t vc[kN][4];   // [group][half]: unit g (elements 4 g ..) of slots 2t, 2t+1 of that half
#pragma unroll
    for (int n = 0; n < kN; ++n) ldmatrix_x4_trans(vc[n], smem_u32(blocks[n]) + Block::kValues + pair * 512 + lane * 16);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = 2 * pair + k;
      float o[2][4];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const uint2 v0 = lds64(vs[n] + i * 64), v1 = lds64(vs[n] + i * 64 + 32);
        uint32_t b0, b1, c0, c1;
        if constexpr (kF16) {
          split2<__nv_bfloat16>(pw[n][0] * step_of(T{}, v0.x), pw[n][1] * step_of(T{}, v0.y), &b0, &c0);
          split2<__nv_bfloat16>(pw[n][2] * step_of(T{}, v1.x), pw[n][3] * step_of(T{}, v1.y), &b1, &c1);
        } else {
          step_weights(h0[n], e0[n], prmt(v0.x, v0.y, 0x5410), &b0, &c0);
          step_weights(h1[n], e1[n], prmt(v1.x, v1.y, 0x5410), &b1, &c1);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t x[4] = {value_code<T>(vc[n][2 * k], 2 * j), value_code<T>(vc[n][2 * k], 2 * j + 1),
                                 value_code<T>(vc[n][2 * k + 1], 2 * j), value_code<T>(vc[n][2 * k + 1], 2 * j + 1)};
          if (n == 0) mma_zero(__nv_bfloat16{}, o[j], x, b0, b1);
          else mma_add(__nv_bfloat16{}, o[j], x, b0, b1);
          mma_add(__nv_bfloat16{}, o[j], x, c0, c1);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) w.o[i][j][e] += o[j][e];
    }
  }
  if (!whole) fence_proxy_async();   // the zeros before the next copy
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) k_q4_decode(const __grid_constant__ Q4DecodeArgs p) {
  using Block = Q4Block<D>;
  using Smem = Q4DecodeSmem<D>;
  constexpr int ST = Smem::kStages, G = D / 32, QS = kQuerySlots;
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u));
  const PagedAttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&s.full[i], 1);
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
  }
  __syncthreads();
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int c = blockIdx.x;

  if (warp >= kWarps) {
    // ------------------------------------------------------------ producer --
    const int P = a.kv.page_size;
    const uint32_t capacity = a.kv.max_pages * a.kv.page_size;
    uint32_t it = 0, pieces = 0;
    int seq, n_cut = 0;
    uint32_t before, L, runs = gridDim.x;
    const uint32_t total = find_run(p, c, runs, lane, &seq, &before, &L);
    const uint32_t t1 = c < (int)runs ? run_start(total, c + 1, runs) : 0;
    uint32_t t = run_start(total, c, runs), ts = seq_tiles(p, L);   // (c >= runs: no run)
    // lane i: pages of the table row's entries base + i and base + 32 + i, -1: none
    int cached_seq = -1, base = 0, page_lo = -1, page_hi = -1;
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
      const int head = h * p.group + chunk * kSlotHeads, heads = min(kSlotHeads, p.group - chunk * kSlotHeads);
      const bool fits = L <= capacity;
      if (!fits && lane == 0) raise_error(a.err, kDevBadArgument);
      const int dest = !fits ? -2 : tile0 == 0 && tile1 == ts ? -1 : 2 * c + (tile0 == 0 ? 1 : 0);
      // ---- the piece and its queries
      const int qs = pieces % QS;
      if (pieces >= QS &&
          !__all_sync(0xffffffffu, paged_wait(&s.qempty[qs], (pieces / QS - 1) & 1, &s.abort, a.err))) {
        alive = false;
        break;
      }
      if (lane == 0) {
        Piece& x = s.piece[qs];
        x.heads = heads;
        x.seq = seq;
        x.head = head;
        x.dest = dest;
        x.scores = p.scores ? reinterpret_cast<float2*>(p.scores) +
                                  ((long long)seq * p.units_per_seq + unit) * capacity * p.score_pairs
                            : nullptr;
        mbar_arrive_expect_tx(&s.qfull[qs], (uint32_t)heads * D * 2);
        bulk_g2s(s.q[qs], a.q + (long long)seq * a.q_stride + (long long)head * D, (uint32_t)heads * D * 2, &s.qfull[qs]);
      }
      ++pieces;
      const int32_t* table = a.kv.page_table + (long long)seq * a.kv.table_stride;
      const int n_entries = fits ? (int)((L + P - 1) >> a.page_shift) : 0;
      const uint8_t* pool = p.kv.pool + (long long)h * p.kv.head_stride;
      auto look_up = [&](int entry) {
        int page = -1;
        if (entry < n_entries) {
          page = table[entry];
          if (page < 0 || (uint32_t)page >= a.kv.n_pages) {
            raise_error(a.err, kDevBadArgument);
            page = -1;
          }
        }
        return page;
      };
#pragma unroll 1
      for (uint32_t tile = tile0; tile < tile1; ++tile) {
        // lane l < 8: block l of the tile; the first of each page's copies them all
        const int first = (int)tile << kTileShift, slot = first + 16 * lane, first_entry = first >> a.page_shift;
        if (cached_seq != seq || first_entry < base || first_entry >= base + 32) {
          if (cached_seq == seq && first_entry >= base + 32 && first_entry < base + 64) {
            base += 32;
            page_lo = page_hi;
          } else {
            base = first_entry;
            page_lo = look_up(base + lane);
          }
          cached_seq = seq;
          page_hi = look_up(base + 32 + lane);   // asked for long before its turn
        }
        const int from = (slot >> a.page_shift) - base, off = slot & (P - 1);
        const int lo = __shfl_sync(0xffffffffu, page_lo, from & 31), hi = __shfl_sync(0xffffffffu, page_hi, from & 31);
        const int page = from < 32 ? lo : hi;
        const int valid = lane < kBlocks && page >= 0 ? max(0, min(16, (int)L - slot)) : 0;
        const uint32_t there = __ballot_sync(0xffffffffu, valid > 0);
        const bool last = tile + 1 == tile1;
        if (there == 0 && !last) continue;
        const int st = it % ST;
        if (it >= ST &&
            !__all_sync(0xffffffffu, paged_wait(&s.empty[st], ((it / ST) - 1) & 1, &s.abort, a.err))) {
          alive = false;
          break;
        }
        StageMeta& meta = s.meta[st];
        if (lane < kBlocks) meta.valid[lane] = valid;
        if (lane == 0) {
          meta.first = first;
          meta.last = last;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&s.full[st], __popc(there) * Block::kBytes);
        __syncwarp();
        if (valid > 0 && (lane == 0 || off == 0)) {   // (its page's blocks of the tile all count, but what is behind the end)
          const int of_page = min((P - off) >> 4, kBlocks - lane);
          const uint32_t mine = there >> lane & ((1u << of_page) - 1);
          bulk_g2s(s.kv[st][lane], pool + (long long)page * p.kv.page_stride + (off >> 4) * Block::kBytes,
                   __popc(mine) * Block::kBytes, &s.full[st]);
        }
        ++it;
      }
      if (dest >= 0) {
        CutUnit u;
        static_cast<CutPiece&>(u) = cut_piece(total, begin, ts, tile0, c, runs);
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
    // While the last tiles are on their way: the counts of the units it shares, and
    // the arrival of a piece that is not the run's last.
    if (lane < n_cut) {
      const CutUnit& u = s.cut[lane];
      open_count(p.arrived + 2 * runs + u.unit, p.tag);
      if (u.pieces > kJoin) open_count(p.arrived + piece_slot(u, u.piece / kJoin * kJoin, runs), p.tag);
    }
    const int n_early = alive && n_cut > 0 && pieces > 1 && cut_first ? 1 : 0;
    if (n_early) {
      alive = __all_sync(0xffffffffu, paged_wait(&s.early, 0, &s.abort, a.err));
      if (alive && lane == 0) s.last[0] = arrive_first(p, s.cut[0], runs);
    }
    if (lane == 0) {
      s.n_cut = n_cut;
      s.runs = (int)runs;
      s.n_early = n_early;
    }
    __syncwarp();
    uint32_t q_drained = pieces > (uint32_t)QS ? pieces - QS : 0;
    if (alive) {   // the end of the run, in a slot whose last piece was consumed
      const int qs = pieces % QS;
      alive = pieces < QS || __all_sync(0xffffffffu, paged_wait(&s.qempty[qs], (pieces / QS - 1) & 1, &s.abort, a.err));
      if (alive) {
        if (pieces >= QS) ++q_drained;
        if (lane == 0) {
          s.piece[qs].heads = 0;
          mbar_arrive(&s.qfull[qs]);
        }
      }
    }
    __syncwarp();
    // Every issued copy lands before the CTA may exit.
#pragma unroll 1
    for (uint32_t j = it > (uint32_t)ST ? it - ST : 0; j < it; ++j)
      paged_wait(&s.full[j % ST], (j / ST) & 1, &s.abort, a.err, false);
#pragma unroll 1
    for (uint32_t j = q_drained; j < pieces; ++j)
      paged_wait(&s.qfull[j % QS], (j / QS) & 1, &s.abort, a.err, false);
    return;
  }

  // -------------------------------------------------------------- consumers --
  const int g = lane >> 2, t4 = lane & 3;
  Stream<D> w;
  uint32_t joins = 0, it = 0;
  auto join = [&]() {   // the consumer warps' barrier
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.joined);
    return __all_sync(0xffffffffu, paged_wait(&s.joined, joins++ & 1, &s.abort, a.err));
  };
#pragma unroll 1
  for (uint32_t pieces = 0;; ++pieces) {
    const int qs = pieces % QS;
    if (!__all_sync(0xffffffffu, paged_wait(&s.qfull[qs], (pieces / QS) & 1, &s.abort, a.err))) return;
    const Piece& piece = s.piece[qs];
    const int heads = piece.heads;
    if (heads == 0) break;
    load_queries<T, D>(w.u, reinterpret_cast<const T*>(s.q[qs]), heads, p.scale_log2, lane);
    w.m[0] = w.m[1] = -INFINITY;
    w.ref[0] = w.ref[1] = w.l[0] = w.l[1] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w.extra[e] = 0.f;
#pragma unroll
      for (int i = 0; i < G; ++i) w.o[i][0][e] = w.o[i][1][e] = 0.f;
    }
    int st;
#pragma unroll 1
    for (;; ++it) {
      st = it % ST;
      if (!__all_sync(0xffffffffu, paged_wait(&s.full[st], (it / ST) & 1, &s.abort, a.err))) return;
      const StageMeta& meta = s.meta[st];
      const int valid[2] = {meta.valid[warp], meta.valid[warp + kWarps]};
      const bool last = meta.last;
      uint8_t* const blocks[2] = {s.kv[st][warp], s.kv[st][warp + kWarps]};
      float2* scores = p.scores ? piece.scores + (long long)(meta.first + 16 * warp) * p.score_pairs : nullptr;
      if (valid[1] > 0) take_blocks<T, D, 2>(w, blocks, valid, lane, scores, p.score_pairs);
      else if (valid[0] > 0) take_blocks<T, D, 1>(w, blocks, valid, lane, scores, p.score_pairs);
      if (last) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[st]);
    }
    // ---- the end of a piece.  Join the warps: the last stage, which every warp is done with
    // after the first join, holds their rows, [warp][head][chunk of 4 ^ (head & 6)].
    ++it;
    float2(*ml)[kSlotHeads] = s.ml[pieces & 1];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = w.l[e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) ml[warp][2 * t4 + e] = make_float2(w.m[e], x);
    }
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float add = __shfl_sync(0xffffffffu, w.extra[e], 4 * i + t4);
        if constexpr (std::is_same<T, __half>::value) {
          add = (add + __shfl_sync(0xffffffffu, w.extra[e], 4 * (4 + i) + t4)) * pow2(-kRaise);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            w.o[i][j][e] *= pow2(133 - kRaise);
            w.o[i][j][2 + e] *= pow2(133 - kRaise - 4);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          w.o[i][j][e] += add;
          w.o[i][j][2 + e] += add;
        }
      }
    if (!join()) return;
    auto rows = reinterpret_cast<float4(*)[kSlotHeads][D / 4]>(s.kv[st][0]);
    static_assert(sizeof(float4) * kWarps * kSlotHeads * (D / 4) <= kBlocks * Block::kBytes, "the warps' rows exceed a stage");
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) M = fmaxf(M, ml[k][2 * t4 + e].x);
      const float f = w.m[e] == -INFINITY ? 0.f : exp2_fast(w.m[e] - M);
#pragma unroll
      for (int i = 0; i < G; ++i)
        rows[warp][2 * t4 + e][(8 * i + g) ^ (2 * t4)] =
            make_float4(w.o[i][0][e] * f, w.o[i][0][2 + e] * f, w.o[i][1][e] * f, w.o[i][1][2 + e] * f);
    }
    if (!join()) return;
#pragma unroll 1
    for (int head = warp; head < heads && piece.dest != -2; head += kWarps) {
      constexpr int V = D / 32;   // elements of this lane
      float M = -INFINITY, sum = 0.f, v[V];
#pragma unroll
      for (int k = 0; k < kWarps; ++k) M = fmaxf(M, ml[k][head].x);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        // (a warp without a maximum has the sum 0, or NaN, which stays)
        sum += ml[k][head].y * (ml[k][head].x == -INFINITY ? 0.f : exp2_fast(ml[k][head].x - M));
        const float* row = reinterpret_cast<const float*>(rows[k][head]) + ((V * lane) ^ (4 * (head & 6)));
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += row[i];
      }
      if (piece.dest == -1) finish_row<T, D, false>(p, piece.seq, piece.head + head, as_float4(v), M, sum, lane);
      else store_partial<D>(p, piece.dest * kSlotHeads + head, as_float4(v), M, sum, lane);
    }
    fence_proxy_async();   // the rows before the next copy
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&s.empty[st]);
      mbar_arrive(&s.qempty[qs]);
      if (pieces == 0) mbar_arrive(&s.early);   // the run's first piece is written
    }
  }

  // ---- the last pieces to arrive join the others'
  const int n_cut = s.n_cut, n_early = s.n_early, runs = s.runs;
  if (n_cut == 0) return;
  if (!join()) return;   // every warp's partials are written
  if (threadIdx.x == 0 && n_early < n_cut) s.last[n_early] = arrive_first(p, s.cut[n_early], runs);
  if (!join()) return;
#pragma unroll 1
  for (int k = 0; k < n_cut; ++k) {
    if (!s.last[k]) continue;
    const CutUnit& cu = s.cut[k];
    const int groups = (cu.pieces + kJoin - 1) / kJoin, first = cu.piece / kJoin * kJoin;
    int from = first, step = 1, n = min(kJoin, cu.pieces - first);
    bool final = groups == 1;
#pragma unroll 1
    for (;;) {   // its sixteen, then the unit's sixteens
      join_pieces<T, D, false, kSlotHeads, kWarps>(p, cu, runs, from, step, n, final, warp, lane);
      if (final) break;
      if (!join()) return;
      if (threadIdx.x == 0) s.last[k] = arrive_last(p.arrived + 2 * runs + cu.unit, p.tag, groups);
      if (!join()) return;
      if (!s.last[k]) break;
      from = 0;
      step = kJoin;
      n = groups;
      final = true;
    }
  }
}

// weights[s][h][slot] += sum over the query heads of kv head h of exp(scale q k - lse), from
// the scores that k_q4_decode left.  Each warp has a run of tiles of 32 slots, a lane a slot,
// as the decode kernel's CTAs have runs of theirs; the next tile is on its way while one is
// summed.  (A pass over the keys that forms the scores again, 80 B a slot and kv head of 128
// instead of 8 a query head, took 32 us behind 16 x 8704 of 8 kv heads where this takes
// 8: it has all the instructions of a score once more.  Groups of more than 8 query heads read
// their further lse's slot by slot: 32 x 16384 of 2 kv heads with 16 each 58 us, and 76 with weights.)
constexpr int kWeighWarps = 8, kWeighTileShift = 5, kWeighCtasPerSm = 4;

template <int kPairs>   // query heads of a unit in pairs
__global__ void __launch_bounds__(kWeighWarps * 32, kWeighCtasPerSm) k_q4_weigh(const __grid_constant__ Q4DecodeArgs p, int chunks) {
  const PagedAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  // (Lengths and tables were there before the attention, which this need not wait for.)
  const uint32_t c = blockIdx.x * kWeighWarps + (threadIdx.x >> 5);
  uint32_t runs = gridDim.x * kWeighWarps, before, L;
  int seq;
  const uint32_t total = find_run(p, c, runs, lane, &seq, &before, &L);
  const uint32_t t1 = run_start(total, c + 1, runs), capacity = a.kv.max_pages * a.kv.page_size;
  uint32_t t = run_start(total, c, runs), ts = seq_tiles(p, L);
  struct Slot {
    float2 s[kPairs];
    float old;
    const float2* more;   // the next chunk's scores
    float* to;            // null: nothing to add to
    int seq, head;
  } next;
  auto load = [&](Slot& x) {
    while (t >= before + ts * p.units_per_seq) {
      before += ts * p.units_per_seq;
      L = a.seq_len[++seq];
      ts = seq_tiles(p, L);
    }
    const int h = (int)((t - before) / ts);
    const uint32_t slot = ((t - before - h * ts) << kWeighTileShift) + lane, len = L <= capacity ? L : 0;
    ++t;
    x.seq = seq;
    x.head = h;
    x.to = nullptr;
    if (slot >= len) return;
    const int page = a.kv.page_table[(long long)seq * a.kv.table_stride + (slot >> a.page_shift)];
    if (page < 0 || (uint32_t)page >= a.kv.n_pages) return;   // (reported by the attention)
    const long long unit = (long long)seq * a.kv.n_kv_heads + h;
    x.to = p.kv.weights + unit * capacity + slot;
    x.more = reinterpret_cast<const float2*>(p.scores) + (unit * chunks * capacity + slot) * kPairs;
    x.old = *x.to;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) x.s[i] = __ldcs(x.more + i);
    x.more += (long long)capacity * kPairs;
  };
  pdl_wait();
  if (t >= t1) return;
  load(next);
  int l_seq = -1, l_head = -1;
  float lse[2 * kPairs];
  while (true) {
    Slot x = next;
    const bool more = t < t1;
    if (more) load(next);
    if (l_seq != x.seq || l_head != x.head || chunks > 1) {
#pragma unroll
      for (int i = 0; i < 2 * kPairs; ++i)   // a head that is not there: no weight
        lse[i] = i < p.group ? a.lse[(long long)x.seq * a.n_heads + x.head * p.group + i] * kLog2e : INFINITY;
      l_seq = x.seq;
      l_head = x.head;
    }
    if (x.to) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) sum += exp2_fast(x.s[i].x - lse[2 * i]) + exp2_fast(x.s[i].y - lse[2 * i + 1]);
      for (int chunk = 1; chunk < chunks; ++chunk, x.more += (long long)capacity * kPairs)
#pragma unroll
        for (int i = 0; i < 2 * kPairs; ++i) {
          const int head = chunk * kSlotHeads + i;
          if (head < p.group)
            sum += exp2_fast(reinterpret_cast<const float*>(x.more)[i] -
                             a.lse[(long long)x.seq * a.n_heads + x.head * p.group + head] * kLog2e);
        }
      *x.to = x.old + sum;
    }
    if (!more) return;
  }
}

template <typename T, int D>
int launch(const Q4AttnArgs& args, const Q4DecodeArgs& p, int runs, cudaStream_t st) {
  auto kern = k_q4_decode<T, D>;
  const int smem = (int)sizeof(Q4DecodeSmem<D>) + 128;
  static_assert((sizeof(Q4DecodeSmem<D>) + 128 + 1024) * kCtasPerSm <= 228 * 1024, "CTAs per SM");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(runs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static OncePerDevice once;
  if (once.launch(reinterpret_cast<const void*>(kern), smem, [&] { return cudaLaunchKernelEx(&cfg, kern, p); }) != cudaSuccess)
    return -1;
  if (!args.kv.weights) return 0;
  Q4DecodeArgs w = p;   // its units are whole kv heads
  w.units_per_seq = (int)args.kv.n_kv_heads;
  w.tile_shift = kWeighTileShift;
  cfg.gridDim = dim3(kWeighCtasPerSm * paged_sm_count());
  cfg.blockDim = dim3(kWeighWarps * 32);
  cfg.dynamicSmemBytes = 0;
  auto weigh = p.score_pairs == 1 ? k_q4_weigh<1> : p.score_pairs == 2 ? k_q4_weigh<2> : p.score_pairs == 3 ? k_q4_weigh<3> : k_q4_weigh<4>;
  return cudaLaunchKernelEx(&cfg, weigh, w, p.chunks) == cudaSuccess ? 0 : -1;
}

int units_per_head(const qwen_paged_kv_q4& kv, int n_heads) {
  return (n_heads / (int)kv.n_kv_heads + kSlotHeads - 1) / kSlotHeads;
}
int score_pairs(const qwen_paged_kv_q4& kv, int n_heads) {
  return (std::min(kSlotHeads, n_heads / (int)kv.n_kv_heads) + 1) / 2;
}
size_t units_of(const qwen_paged_kv_q4& kv, int n_heads) {
  return (size_t)kv.n_seq * kv.n_kv_heads * units_per_head(kv, n_heads);
}

}  // namespace

bool attention_q4_fits(const qwen_paged_kv_q4& kv, int n_heads) {
  const double slots = (double)kv.max_pages * kv.page_size;
  return (double)units_of(kv, n_heads) * std::ceil(slots / (1 << kTileShift)) < 2147483648.0 &&
         (!kv.weights || (double)kv.n_seq * kv.n_kv_heads * std::ceil(slots / (1 << kWeighTileShift)) < 2147483648.0);
}

// Partials and arrivals, as DecodeArgs has them, and where weights are kept the scores of
// every unit at its capacity and the lse.
size_t attention_q4_workspace(const qwen_paged_kv_q4& kv, int n_heads) {
  const size_t runs = kCtasPerSm * paged_sm_count(), units = units_of(kv, n_heads);
  size_t bytes = 2 * runs * kSlotHeads * (kv.head_dim + 2) * sizeof(float) + (2 * runs + units) * sizeof(unsigned long long);
  if (kv.weights)
    bytes += units * kv.max_pages * kv.page_size * score_pairs(kv, n_heads) * sizeof(float2) +
             (size_t)kv.n_seq * n_heads * sizeof(float);
  return bytes;
}

int launch_attention_q4(const Q4AttnArgs& a, cudaStream_t st) {
  Q4DecodeArgs p{};
  p.kv = a.kv;
  p.a.kv.page_table = a.kv.page_table;
  p.a.kv.n_pages = a.kv.n_pages;
  p.a.kv.page_size = a.kv.page_size;
  p.a.kv.n_kv_heads = a.kv.n_kv_heads;
  p.a.kv.head_dim = a.kv.head_dim;
  p.a.kv.n_seq = a.kv.n_seq;
  p.a.kv.max_pages = a.kv.max_pages;
  p.a.kv.table_stride = a.kv.table_stride;
  p.a.page_shift = a.page_shift;
  p.a.q = a.q;
  p.a.q_stride = a.q_stride;
  p.a.out = a.out;
  p.a.out_stride = a.out_stride;
  p.a.n_heads = a.n_heads;
  p.a.seq_len = a.seq_len;
  p.a.err = a.err;
  p.chunks = units_per_head(a.kv, a.n_heads);
  p.group = a.n_heads / (int)a.kv.n_kv_heads;
  p.units_per_seq = (int)a.kv.n_kv_heads * p.chunks;
  p.tile_shift = kTileShift;
  p.scale_log2 = a.scale * kLog2e;
  const int runs = kCtasPerSm * paged_sm_count();
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = p.part_o + (size_t)2 * runs * kSlotHeads * a.kv.head_dim;
  p.arrived = reinterpret_cast<unsigned long long*>(p.part_ml + (size_t)2 * runs * kSlotHeads * 2);
  p.a.lse = a.lse;
  if (a.kv.weights) {
    p.score_pairs = score_pairs(a.kv, a.n_heads);
    p.scores = reinterpret_cast<float*>(p.arrived + 2 * runs + units_of(a.kv, a.n_heads));
    if (!a.lse)
      p.a.lse = p.scores + units_of(a.kv, a.n_heads) * a.kv.max_pages * a.kv.page_size * 2 * p.score_pairs;
  }
  p.tag = paged_call_tag();
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) return d64 ? launch<__half, 64>(a, p, runs, st) : launch<__half, 128>(a, p, runs, st);
  return d64 ? launch<__nv_bfloat16, 64>(a, p, runs, st) : launch<__nv_bfloat16, 128>(a, p, runs, st);
}

}  // namespace qwen
