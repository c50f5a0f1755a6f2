// Turns of two query tiles with the exponentials, where they share a ring of key and value tiles (attn_prefill.cu, attn_q8_prefill.cu):
// tile 0, tile 1, tile 0, ...  They take turns at the key tiles that both attend to, or, where the second query tile begins later, the
// first one at a key tile and the second at the next: it begins a turn earlier so (bf16 pages, windows of 128 and of 700 over 4 x 2000
// tokens: 70 and 146 us, 81 and 158 with turns at the same key tile).  A turn waits for one at the same key tile or an
// earlier one, which the ring has let through already, so no turn can wait for a tile that the ring keeps back.  (Counted from each one's own
// first tile, a mask that begins much later for the second query tile makes the first wait for tiles that are further ahead than the
// ring reaches.)
#pragma once

#ifdef __CUDACC__
#define NKB_TURNS static inline __host__ __device__
#else
#define NKB_TURNS static inline
#endif

struct NkbTurns {
  int first, count;                      // of this query tile: at key tiles [first, first + count)
};
// Query tile t's, where the two attend to key tiles [lo0, hi0) and [lo1, hi1).
NKB_TURNS NkbTurns nkb_turns(int t, int lo0, int hi0, int lo1, int hi1) {
  const int late = lo1 > lo0 ? 1 : 0, first = lo1 - late > lo0 ? lo1 - late : lo0, end = hi1 - late < hi0 ? hi1 - late : hi0;
  NkbTurns o;
  o.first = t == 0 ? first : first + late;
  o.count = end > first ? end - first : 0;
  return o;
}
// the turn at a key tile, < 0: none
NKB_TURNS int nkb_turn_at(const NkbTurns& turns, int tile) {
  return unsigned(tile - turns.first) < unsigned(turns.count) ? tile - turns.first : -1;
}
// How many there are, for a kernel whose turns are counted from each one's first key tile; none where that is not where they begin.  (In the loop
// over 8-bit pages the general form costs more than such works gain: 16 prompts of 1024 tokens 217.6 us, 220.7 with it.)
NKB_TURNS int nkb_turns_from_first(int lo0, int hi0, int lo1, int hi1) {
  const NkbTurns a = nkb_turns(0, lo0, hi0, lo1, hi1), b = nkb_turns(1, lo0, hi0, lo1, hi1);
  return a.first == lo0 && b.first == lo1 ? a.count : 0;
}
#undef NKB_TURNS
