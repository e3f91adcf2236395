// paged_split.h -- how the paged kernels divide their work, and where the warps of k_prefix
// put their rows in shared memory: arithmetic that the host can run too, so that the tests
// check what the kernels use (paged_hooks.cu).  What takes kernel parameters by reference
// is inlined: through a reference each is a load from memory, ~0.4 us after another.
#pragma once
#include <stdint.h>

#include <algorithm>

#ifdef __CUDACC__
#define QWEN_HD __host__ __device__ __forceinline__
#define QWEN_HD_CALL __host__ __device__ __noinline__
#else
#define QWEN_HD inline
#define QWEN_HD_CALL
#endif

namespace qwen {

// x / d.  Out of line, with its operands in registers.
inline QWEN_HD_CALL unsigned long long divide(unsigned long long x, unsigned long long d) {
  return (x | d) >> 32 ? x / d : (uint32_t)x / (uint32_t)d;
}

// -------------------------------------------------------- k_paged_decode --
// Run c of G: tiles run_start(c) .. run_start(c + 1) - 1 of total < 2^31 (the entry points
// refuse more).
QWEN_HD uint32_t run_start(uint32_t total, uint32_t c, uint32_t G) {
  const uint32_t q = total / G;
  return q * c + (total - q * G) * c / G;   // = total c / G, in 32 bits
}
// The run that holds tile x: the largest c with run_start(c) <= x.
QWEN_HD int run_of(uint32_t total, uint32_t x, uint32_t G) {
  return (int)divide((unsigned long long)(x + 1) * G - 1, total);
}
// A unit that several runs share, and the piece of it that one of them has.
struct CutPiece {
  int pieces, piece, run0;   // of the unit, this one, run of the first
  uint32_t total, begin;     // fewer tiles than runs: their number, the unit's first
};
// The unit has tiles begin .. begin + tiles - 1, run c those from its tile0 on.
QWEN_HD CutPiece cut_piece(uint32_t total, uint32_t begin, uint32_t tiles, uint32_t tile0, int c, uint32_t G) {
  CutPiece u;
  u.run0 = run_of(total, begin, G);
  u.pieces = total < G ? (int)tiles : run_of(total, begin + tiles - 1, G) - u.run0 + 1;
  u.piece = total < G ? (int)tile0 : c - u.run0;
  u.total = total < G ? total : G;
  u.begin = begin;
  return u;
}
// The partial slot of piece i: runs follow one another, or (fewer tiles than runs)
// each has one tile or none.
QWEN_HD int piece_slot(const CutPiece& u, int i, int G) {
  const int r = u.total < (unsigned)G ? run_of(u.total, u.begin + i, G) : u.run0 + i;
  return 2 * r + (i == 0 ? 1 : 0);
}

// --------------------------------------------------------------- k_prefix --
constexpr int kRows = 128;                 // rows of a stream (M)
constexpr int kPos = 128;                  // positions of a tile
constexpr int kWarpRows = 16;              // of a stream's rows, those whose queries a softmax warp loads

struct PrefixSplit {
  int kv_heads, group, rows;       // query heads and rows per kv head
  int tiles, pairs;                // row tiles, units
  int steps;                       // position tiles
  unsigned long long total;        // weighted steps of all units
  int share2, share1;              // CTAs of a unit of two tiles, of one; 0: runs over all units
};

// Units of a kv head come pair by pair, an odd tile's last; a step weighs its MMAs.
QWEN_HD int unit_weight(const PrefixSplit& p, int pair) { return 2 * pair + 1 < p.tiles ? 2 : 1; }
QWEN_HD unsigned long long unit_begin(const PrefixSplit& p, int unit) {
  const int h = unit / p.pairs, pair = unit % p.pairs;
  return (unsigned long long)p.steps * ((unsigned long long)h * p.tiles + 2 * pair);
}
QWEN_HD unsigned long long prefix_run_start(const PrefixSplit& p, int c, int G) {
  return divide(p.total * (unsigned)c, (unsigned)G);
}
// Steps i of a unit that run c takes: those that begin (at begin + w i) in it.
QWEN_HD void steps_of(const PrefixSplit& p, unsigned long long begin, int w, int c, int G, int* i0, int* i1) {
  const unsigned long long x0 = prefix_run_start(p, c, G), x1 = prefix_run_start(p, c + 1, G), n = p.steps;
  const unsigned long long y0 = (x0 - begin + w - 1) >> (w - 1), y1 = (x1 - begin + w - 1) >> (w - 1);
  *i0 = x0 <= begin ? 0 : (int)(y0 < n ? y0 : n);
  *i1 = x1 <= begin ? 0 : (int)(y1 < n ? y1 : n);
}
// CTAs of a kv head whose units have CTAs of their own.
QWEN_HD int ctas_per_head(const PrefixSplit& p) { return p.tiles / 2 * p.share2 + (p.tiles & 1) * p.share1; }

// The pieces of CTA c, one after another: steps [i0, i1) of a unit, partials in
// slots 2 id, 2 id + 1.
struct Pieces {
  const PrefixSplit& p;
  int c, G, unit, w, h, pair, i0, i1, id;
  QWEN_HD Pieces(const PrefixSplit& p, int c, int G) : p(p), c(c), G(G), unit(-1) {}
  QWEN_HD bool next() {
    if (p.share2) {
      if (unit >= 0) return false;
      const int per_head = ctas_per_head(p);
      h = c / per_head;
      const int rest = c - h * per_head;
      if (h >= p.kv_heads) return false;
      pair = rest / p.share2 < p.pairs - 1 ? rest / p.share2 : p.pairs - 1;
      w = unit_weight(p, pair);
      const int part = rest - pair * p.share2, parts = w == 2 ? p.share2 : p.share1;
      unit = h * p.pairs + pair;
      i0 = (int)((uint32_t)p.steps * (uint32_t)part / (uint32_t)parts);   // 2^17 steps, 2^8 parts at most
      i1 = (int)((uint32_t)p.steps * (uint32_t)(part + 1) / (uint32_t)parts);
      id = c;
      return i1 > i0;
    }
    const int units = p.kv_heads * p.pairs;
    const unsigned long long x0 = prefix_run_start(p, c, G), x1 = prefix_run_start(p, c + 1, G);
    if (unit < 0) {
      if (x0 >= x1) return false;
      const unsigned long long per_head = (unsigned long long)p.steps * p.tiles;
      const int hh = (int)divide(x0, per_head);
      unit = hh * p.pairs + (int)divide(x0 - hh * per_head, 2ull * p.steps) - 1;
    }
    for (;;) {
      if (++unit >= units) return false;
      const unsigned long long begin = unit_begin(p, unit);
      if (begin >= x1) return false;
      h = unit / p.pairs;
      pair = unit - h * p.pairs;
      w = unit_weight(p, pair);
      id = unit + c;
      steps_of(p, begin, w, c, G, &i0, &i1);
      if (i1 > i0) return true;
    }
  }
};

// What the join reads for the rows of one row tile: partials 0 .. n - 1 in slot(k).  A
// lone tile's pieces leave two, one a stream.
struct Partials {
  unsigned long long begin;
  int n, w, c0, first, odd;
  QWEN_HD Partials(const PrefixSplit& p, int h, int tile, int G) {
    const int pair = tile / 2, unit = h * p.pairs + pair;
    w = unit_weight(p, pair);
    odd = tile & 1;
    begin = unit_begin(p, unit);
    if (p.share2) {
      c0 = first = h * ctas_per_head(p) + pair * p.share2;
      n = w == 2 ? p.share2 : 2 * p.share1;
    } else {
      c0 = (int)divide((begin + 1) * G - 1, p.total);
      first = c0 + unit;
      n = ((int)divide((begin + (unsigned long long)w * (p.steps - 1) + 1) * G - 1, p.total) - c0 + 1) * (w == 2 ? 1 : 2);
    }
  }
  QWEN_HD int slot(int k) const { return (first + (w == 2 ? k : k / 2)) * 2 + (w == 2 ? odd : k & 1); }
  QWEN_HD bool there(const PrefixSplit& p, int k, int G) const {   // a run may have none of the unit's steps
    if (p.share2) return true;
    int i0, i1;
    steps_of(p, begin, w, c0 + (w == 2 ? k : k / 2), G, &i0, &i1);
    return i1 > i0;
  }
};

// What the steps take one SM: 1.92 us for two row tiles, their chain; 1.5 us for a lone
// one, its loads.  With head_dim 64 MMAs and loads halve and the chain does not: with half
// of these figures 256 sequences behind 32768 positions, 14 and 2 heads, take 68 us
// against 58, 64 behind 8704 and 256 behind 8704 what they take now.
inline double prefix_us(const PrefixSplit& p) {
  return (double)p.kv_heads * p.steps * (p.tiles / 2 * 1.92 + (p.tiles & 1) * 1.5);
}
// Fills in the division of the prefix; returns the number of CTAs.  Up to two fifths of
// the SMs, as many as cost the prefix 8 us, are left to the own positions, whose lengths
// the host does not know.  (A half at most: 16 sequences behind 20000 positions 43 us
// against 39; a third: 64 behind 8704 37.6 against 34.2; 5 us instead of 8: 256 behind
// 32768 73 against 64, though 64 behind 32768 with 16 and 8 heads of 64 39 against 46.)
inline int plan_prefix(PrefixSplit& p, int kv_heads, int n_seq, int n_heads, uint32_t prefix_len, int sms) {
  p.kv_heads = kv_heads;
  p.group = n_heads / kv_heads;
  p.rows = n_seq * p.group;
  p.tiles = (p.rows + kRows - 1) / kRows;
  p.pairs = (p.tiles + 1) / 2;
  p.steps = (int)((prefix_len + kPos - 1) / kPos);
  p.total = (unsigned long long)kv_heads * p.tiles * p.steps;
  const int G = sms - (int)std::min(0.4 * sms, 8.0 * sms * sms / prefix_us(p));
  const int weight = kv_heads * p.tiles;   // one row tile: 1
  if (weight > G) {
    p.share1 = p.share2 = 0;
    return G;
  }
  // whole CTAs for each unit, the number that comes nearest to G
  const int share = std::min(2 * sms / weight, (4 * G + weight) / (2 * weight));
  p.share2 = std::min(p.steps, share);
  p.share1 = std::min(p.steps, std::max(1, share / 2));
  return kv_heads * ctas_per_head(p);
}

// Byte of 16-byte chunk x of row r in a stream's query tile: [half][row][128 B], swizzled.
QWEN_HD int query_byte(int r, int x) { return (x >> 3) * kRows * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4); }
// Byte of 16-byte chunk x of row r < 32 (D / 16 chunks of fp32 a row) that the stream's
// softmax warp j stages in the same tile: the bytes that its own 16 rows of queries take,
// 2 KB of each half, since a warp goes on from one piece's output to the next piece's
// queries without waiting for the others.
QWEN_HD int stage_byte(int D, int j, int r, int x) {
  const int at = r * D;   // of the warp's 32 D bytes
  return (at >> 11) * kRows * 128 + j * kWarpRows * 128 + (at & 2047) + ((x ^ (r & (D / 16 - 1))) << 4);
}

}  // namespace qwen
