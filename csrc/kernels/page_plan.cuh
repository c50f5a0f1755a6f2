// How decode attention (attn_decode.cu, attn_q8_decode.cu) divides the pages of a batch among its CTAs.  P has the kernel's arguments: batch, units, q_len,
// window, chunk, qkv_partials (not null: the newest token is not read from its page), context(b), and mods with MODS.
#pragma once
#include "common.cuh"
#include "attn_maps.h"
#include "api.h"

namespace nkb {

constexpr int kPage = 32;

// Pages a sequence of ctx tokens has to be read (fused: all tokens but the new one), `kept` of them first tokens' ahead of the window's.
template <bool MODS, class P>
__device__ __forceinline__ int pages_of(const P& p, int ctx, int& page_lo, int& kept) {
  const int first_tok = nkb_first_visible(max(ctx - p.q_len, 0), p.window, p.chunk);
  page_lo = first_tok / kPage;
  const int page_hi = ((p.qkv_partials ? ctx - 1 : ctx) + kPage - 1) / kPage;
  kept = 0;
  if constexpr (MODS) kept = min((p.mods.keep_first + kPage - 1) / kPage, page_lo);
  return kept + max(page_hi - page_lo, 0);
}

// Divides the pages of all sequences among `units` CTAs: every CTA of a kv head takes up to `per` pages of one sequence, per the
// same for all, so that long sequences get more CTAs and all of them end together.  (Divided into equal numbers of CTAs per sequence, a
// batch waits for its longest one: 7 sequences of 3500 to 7000 tokens 38.5 us, 33.7 here; one of 32000 36 and 30.)  At least `least`
// pages each, because partial results cost a merge: one sequence of 203 tokens in single pages 15.5 us, as a whole 6.2.
// units >= 2 * batch; returns false for a CTA without work.  One warp's lanes agree on everything.
struct PagePlan {
  int b, split, splits, per;
};
template <bool MODS, class P>
__device__ __forceinline__ bool plan_pages(const P& p, int unit, int least, int lane, PagePlan& o) {
  constexpr uint32_t kAll = 0xffffffffu;
  int lo, kept, total = 0, mine = 0;
  for (int i = lane; i < p.batch; i += 32) {
    const int n = pages_of<MODS>(p, p.context(i), lo, kept);
    total += n;
    if (i < 32) mine = n;
  }
  total = __reduce_add_sync(kAll, total);
  // lane i tries first + first * i / 31 pages; the last one, twice the mean, always does: sum ceil(n / per) <= total / per + batch
  const int first = max((total + p.units - 1) / p.units, least), per_i = first + (first * lane + 30) / 31;
  const float inv = 1.f / float(per_i);
  float count = 0.f;
  for (int i0 = 0; i0 < p.batch; i0 += 32) {
    if (i0 > 0) mine = i0 + lane < p.batch ? pages_of<MODS>(p, p.context(i0 + lane), lo, kept) : 0;
    const int m = min(p.batch - i0, 32);
    for (int i = 0; i < m; ++i)          // (n - 1/2) / per lies half a part off any whole number, far beyond the rounding
      count += fmaxf(ceilf((float(__shfl_sync(kAll, mine, i)) - 0.5f) * inv), 1.f);
  }
  const uint32_t fits = __ballot_sync(kAll, count <= float(p.units)) | 0x80000000u;
  o.per = __shfl_sync(kAll, per_i, __ffs(fits) - 1);
  int base = 0;                          // units of the sequences before i0
  for (int i0 = 0; i0 < p.batch; i0 += 32) {
    const bool in = i0 + lane < p.batch;
    const int n = in ? pages_of<MODS>(p, p.context(i0 + lane), lo, kept) : 0;
    const int want = in ? max((n + o.per - 1) / o.per, 1) : 0;
    int end = want;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(kAll, end, d);
      if (lane >= d) end += x;
    }
    const uint32_t past = __ballot_sync(kAll, in && unit < base + end);
    if (past) {
      const int at = __ffs(past) - 1;
      o.b = i0 + at;
      o.splits = __shfl_sync(kAll, want, at);
      o.split = unit - base - (__shfl_sync(kAll, end, at) - o.splits);
      return true;
    }
    base += __shfl_sync(kAll, end, 31);
  }
  return false;
}

// Units of the page plan: num_splits per sequence, rounded up to one wave of one CTA per SM, or of two (the scratch, which is sized for nq
// heads, has room for num_splits * group per sequence).
inline int plan_units(int batch, int nkv, int group, int num_splits) {
  if (num_splits <= 1) return 0;
  const int asked = batch * num_splits, one = num_sms() / nkv, two = 2 * num_sms() / nkv;
  const int wave = asked <= one ? one : (asked <= two ? two : asked);
  return wave < asked * group ? wave : asked * group;
}

}  // namespace nkb
