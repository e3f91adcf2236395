// paged_hooks.cu -- test hooks: the paged kernels' host arithmetic (paged_split.h), for
// tests without a GPU.
#include "paged_split.h"

using namespace qwen;

extern "C" {

// k_paged_decode: the first tile of run c, and the run that holds tile x.
unsigned qwen_paged_run_start(unsigned total, unsigned c, unsigned G) { return run_start(total, c, G); }
int qwen_paged_run_of(unsigned total, unsigned x, unsigned G) { return run_of(total, x, G); }
// The piece that run c has of a unit of `tiles` tiles from `begin` on, from its tile0 on:
// its number, and the slots of all the unit's pieces (room for `cap`); returns their number.
int qwen_paged_cut_piece(unsigned total, unsigned begin, unsigned tiles, unsigned tile0, int c, unsigned G, int* piece,
                         int* slots, int cap) {
  const CutPiece u = cut_piece(total, begin, tiles, tile0, c, G);
  *piece = u.piece;
  for (int i = 0; i < u.pieces && i < cap; ++i) slots[i] = piece_slot(u, i, (int)G);
  return u.pieces;
}

// k_prefix on `sms` SMs.  plan: row tiles, units of a kv head, steps, share2, share1;
// pieces: (CTA, kv head, unit of the head, its weight, first and last + 1 step, id) of every
// CTA's pieces, room for cap; returns the number of CTAs, the number of pieces in *n.
int qwen_paged_prefix_pieces(int kv_heads, int n_seq, int n_heads, unsigned prefix_len, int sms, int* plan, int* pieces,
                             int cap, int* n) {
  PrefixSplit p{};
  const int G = plan_prefix(p, kv_heads, n_seq, n_heads, prefix_len, sms);
  const int fields[5] = {p.tiles, p.pairs, p.steps, p.share2, p.share1};
  for (int i = 0; i < 5; ++i) plan[i] = fields[i];
  *n = 0;
  for (int c = 0; c < G; ++c) {
    Pieces piece(p, c, G);
    while (piece.next()) {
      const int row[7] = {c, piece.h, piece.pair, piece.w, piece.i0, piece.i1, piece.id};
      for (int i = 0; i < 7 && *n < cap; ++i) pieces[7 * *n + i] = row[i];
      ++*n;
    }
  }
  return G;
}
// The slots that the join reads for row tile `tile` of kv head h (room for cap); returns
// their number.
int qwen_paged_prefix_partials(int kv_heads, int n_seq, int n_heads, unsigned prefix_len, int sms, int h, int tile,
                               int* slots, int cap) {
  PrefixSplit p{};
  const int G = plan_prefix(p, kv_heads, n_seq, n_heads, prefix_len, sms);
  const Partials part(p, h, tile, G);
  int n = 0;
  for (int k = 0; k < part.n; ++k)
    if (part.there(p, k, G)) {
      if (n < cap) slots[n] = part.slot(k);
      ++n;
    }
  return n;
}

// Bytes of the query tile that softmax warp j of a stream of k_prefix writes queries to
// (query: [8][16 rows][dim / 8]) and stages output rows in (stage: [8][32 rows][dim / 16]).
void qwen_paged_prefix_tile(int dim, int* query, int* stage) {
  for (int j = 0; j < 8; ++j) {
    for (int r = 0; r < kWarpRows; ++r)
      for (int x = 0; x < dim / 8; ++x) *query++ = query_byte(j * kWarpRows + r, x);
    for (int r = 0; r < 32; ++r)
      for (int x = 0; x < dim / 16; ++x) *stage++ = stage_byte(dim, j, r, x);
  }
}

}  // extern "C"
