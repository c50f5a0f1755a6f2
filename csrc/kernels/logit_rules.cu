// Rules on logits: penalties for repeated tokens, biases and masks; the logits that are left, or the most likely token.
//
// Mathematics, per row, for the tokens that the rules name, in 64 bits and rounded once, to the logits' type, or to 32 bits where they are compared:
//   seen (in the prompt or the answer):  l = l > 0 ? l / repetition : l * repetition
//   n times among the answer's tokens:   l -= frequency * n;  l -= presence where n > 0
//   biases:                              l += the sum of the token's entries, in their order
//   mask bit zero:                       l = -inf
// Most tokens are named by none: they pass as they are, and in place they are not even read.
//
// A slice of the vocabulary per CTA.  Its counts lie in shared memory, half a word per token (highest bit: seen in the prompt, next: has a bias, below:
// times in the answer; a whole word where a list may be longer than 14 bits), filled from the row's whole list of tokens, so there is no state to
// keep beside that list, no hashing, and no limit on its length; whole numbers, so the order of the counting changes nothing.  Then one pass over the
// slice's logits, whose first loads are on their way while the counting goes on.  The counting also puts every token that it meets on a list, which the
// whole CTA works off: named tokens lie close together (a text has its frequent ones), and 64-bit divisions in the pass itself would be one thread's, one
// after another.  A token with biases is worked out by the thread of its first entry, which looks through the others for its sum, all lanes at the same
// ones at a time (26 rows of 151936, 300 biases: 46 us; each named token looking for its own 82).  The most likely token of a row's slices is found by the CTAs of a cluster through distributed shared
// memory: no workspace that calls could share, and ties go to the lowest index.
#include "api.h"
#include "common.cuh"
#include "rules_args.h"
#include <type_traits>

namespace nkb {

constexpr int kRuleThreads = 512;
constexpr int kCountBytes = 96 * 1024;  // counts of the tokens that a CTA holds at a time: two CTAs per SM
constexpr int kListMost = 2048;         // named tokens on the list
constexpr int kBiasMost = 512;          // entries of a row that lie in shared memory; the ones behind are read where they are
constexpr int kPer = 8;                 // tokens of a piece

template <bool WIDE>
struct Counts {
  static constexpr uint32_t kSeen = WIDE ? 0x80000000u : 0x8000u, kBiased = kSeen >> 1, kTimes = kBiased - 1;
  static constexpr int kTokens = kCountBytes / (WIDE ? 4 : 2);
  uint32_t* w;
  // (both say whether the token had not been named before: one of all threads is told so)
  __device__ __forceinline__ bool add(int t, uint32_t v) const {
    if (WIDE) return atomicAdd(w + t, v) == 0u;
    return ((atomicAdd(w + (t >> 1), v << (16 * (t & 1))) >> (16 * (t & 1))) & 0xffffu) == 0u;
  }
  __device__ __forceinline__ bool mark(int t, uint32_t v) const {
    if (WIDE) return atomicOr(w + t, v) == 0u;
    return ((atomicOr(w + (t >> 1), v << (16 * (t & 1))) >> (16 * (t & 1))) & 0xffffu) == 0u;
  }
  __device__ __forceinline__ uint32_t get(int t) const { return WIDE ? w[t] : (w[t >> 1] >> (16 * (t & 1))) & 0xffffu; }
  // which tokens of a piece are named
  __device__ __forceinline__ uint32_t named(int piece) const {
    uint32_t b = 0;
    if constexpr (WIDE) {
      const uint4 x = reinterpret_cast<const uint4*>(w)[2 * piece], y = reinterpret_cast<const uint4*>(w)[2 * piece + 1];
      const uint32_t c[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) b |= (c[j] ? 1u : 0u) << j;
    } else {
      const uint4 x = reinterpret_cast<const uint4*>(w)[piece];
      if ((x.x | x.y | x.z | x.w) == 0u) return 0u;
      const uint32_t c[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) b |= ((c[j] & 0xffffu) ? 1u << (2 * j) : 0u) | ((c[j] >> 16) ? 2u << (2 * j) : 0u);
    }
    return b;
  }
};

struct RuleRow {
  float rep, freq, pres;
  const int4* near_ids;         // the first entries in shared memory, filled up with -1
  const float* near_values;
  const int* bias_ids;
  const float* bias_values;
  int biases;
};

template <bool WIDE>
__device__ __noinline__ double ruled(const RuleRow& r, float l0, uint32_t c, double bias) {
  using C = Counts<WIDE>;
  double l = l0;
  const uint32_t n = c & C::kTimes;
  if (n || (c & C::kSeen)) {
    if (r.rep != 1.f) l = l > 0.0 ? l / double(r.rep) : l * double(r.rep);
    l -= double(r.freq) * double(n);
    if (n) l -= double(r.pres);
  }
  return l + bias;
}
// 64 bits on their way to bf16, rounded to odd: the rounding that follows is then the only one (to the nearest here, a value beside the middle of two bf16
// numbers would become the middle, and 1 + 2^-8 + 2^-31 the lower one).
__device__ __forceinline__ float to_odd(double l) {
  const float f = __double2float_rz(l);
  return double(f) == l ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// The sum of a token's biases, and through `first` whether entry `at` is the first of them.
__device__ __noinline__ double bias_sum(const RuleRow& r, int at, int token, bool& first) {
  double sum = 0.0;
  int least = at;
  const int near = min(r.biases, kBiasMost);
#pragma unroll 4
  for (int i = 0; i < near; i += 4) {         // (the same entries in every lane)
    const int4 id = r.near_ids[i >> 2];
    const bool e[4] = {id.x == token, id.y == token, id.z == token, id.w == token};
    if (e[0] || e[1] || e[2] || e[3]) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e[j]) {
          least = min(least, i + j);
          sum += double(r.near_values[i + j]);
        }
    }
  }
#pragma unroll 8
  for (int i = near; i < r.biases; ++i)
    if (r.bias_ids[i] == token) {
      least = min(least, i);
      sum += double(r.bias_values[i]);
    }
  first = least == at;
  return sum;
}

template <bool F32>
__device__ __forceinline__ float rule_logit(const void* p, long long i) {
  return F32 ? reinterpret_cast<const float*>(p)[i] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
template <bool F32>
__device__ __forceinline__ void rule_store(void* p, long long i, float v) {
  if constexpr (F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
}

// Logits of a whole piece as they lie in memory, on sixteen bytes.
template <bool F32>
struct Piece {
  static constexpr int kWords = F32 ? 2 : 1;
  uint4 r[kWords];
  __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) r[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ float value(int j) const {
    const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[F32].x, r[F32].y, r[F32].z, r[F32].w};
    return F32 ? __uint_as_float(w[j]) : __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
  }
  // minus infinity where `left` has no bit
  __device__ __forceinline__ Piece masked(uint32_t left) const {
    Piece o = *this;
    uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[F32].x, r[F32].y, r[F32].z, r[F32].w};
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) w[j] = (left >> j) & 1u ? w[j] : 0xff800000u;
      o.r[F32] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t keep = ((((left >> (2 * e)) & 3u) * 0x8001u) & 0x10001u) * 0xffffu;       // two bits, sixteen times each
        w[e] = (w[e] & keep) | (0xff80ff80u & ~keep);
      }
    }
    o.r[0] = make_uint4(w[0], w[1], w[2], w[3]);
    return o;
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = r[i];
  }
  // The largest number; a NaN loses against every number.
  __device__ __forceinline__ float largest() const {
    if constexpr (F32) {
      return fmaxf(fmaxf(fmaxf(value(0), value(1)), fmaxf(value(2), value(3))), fmaxf(fmaxf(value(4), value(5)), fmaxf(value(6), value(7))));
    } else {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r[0]);
      const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
      return fmaxf(f.x, f.y);
    }
  }
};

// Grid: x = slices of a row (a cluster where ids are wanted), y: rows.  Either out or out_ids.
template <bool F32, bool VEC, bool WIDE>
__global__ void __launch_bounds__(kRuleThreads, 2) logit_rules_kernel(const NkbLogitRules a, int slice) {
  using C = Counts<WIDE>;
  extern __shared__ __align__(16) uint32_t words[];
  __shared__ int s_list[kListMost];
  __shared__ __align__(16) int s_bias_ids[kBiasMost];
  __shared__ float s_bias_values[kBiasMost];
  __shared__ int s_n;
  __shared__ float s_best[kRuleThreads / 32];
  __shared__ int s_at[kRuleThreads / 32];
  __shared__ int2 s_slices[8];          // in the cluster's first CTA: best of every slice, bits of the value and token
  constexpr int kBytes = F32 ? 4 : 2, kAhead = F32 ? 4 : 8;       // pieces of a thread on their way: 128 bytes
  const C counts{words};
  const int row = blockIdx.y, tid = threadIdx.x;
  const int first = blockIdx.x * slice, last = min(a.vocab, first + slice);
  const uint8_t* in = reinterpret_cast<const uint8_t*>(a.logits) + (long long)row * a.ld * kBytes;
  uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + (a.out ? (long long)row * a.out_ld * kBytes : 0);
  const bool ids = a.out_ids != nullptr, in_place = !ids && out == in;
  const bool joined = ids && gridDim.x > 1;
  if (joined) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");       // (waited for before the first access to another CTA)
  griddep_wait();
  griddep_launch();

  // VEC: whole pieces of sixteen-byte words; what is left of a slice, and everything where rows do not start on sixteen bytes, token by token
  constexpr int kPiece = kPer * kBytes;
  Piece<F32> x[VEC ? kAhead : 1];
  auto load = [&](int lo, int pieces, int p0) {
    if (!VEC || in_place) return;
    const uint8_t* p = in + (long long)lo * kBytes + (p0 + tid) * kPiece;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (p0 + tid + i * kRuleThreads < pieces) x[VEC ? i : 0].load(p + i * (kRuleThreads * kPiece));
  };
  load(first, (min(last, first + C::kTokens) - first) / kPer, 0);

  int* tokens = a.tokens ? a.tokens + row * a.tokens_ld : nullptr;
  // the first tokens of the list, too, whose length is not known yet
  const bool token16 = (reinterpret_cast<uintptr_t>(tokens) & 15) == 0;
  const bool early = tokens && token16 && 4 * tid + 4 <= a.width;
  int4 ahead = make_int4(-1, -1, -1, -1);
  if (early) ahead = *reinterpret_cast<const int4*>(tokens + 4 * tid);
  const int len = a.tokens ? min(a.lens[row], a.width) : 0;
  const bool fresh = a.ids && len > 0;
  const int newest = fresh ? a.ids[row] : 0;
  if (fresh && blockIdx.x == 0 && tid == 0) tokens[len - 1] = newest;      // (the others take it from ids)
  RuleRow r;
  r.rep = a.repetition ? a.repetition[row] : 1.f;
  r.freq = a.frequency ? a.frequency[row] : 0.f;
  r.pres = a.presence ? a.presence[row] : 0.f;
  r.bias_ids = a.bias_ids + row * a.bias_ld;
  r.bias_values = a.bias_values + row * a.bias_ld;
  r.biases = a.biases;
  r.near_ids = reinterpret_cast<const int4*>(s_bias_ids);
  r.near_values = s_bias_values;
  for (int i = tid; i < min(kBiasMost, (a.biases + 3) & ~3); i += kRuleThreads) {        // (a barrier before they are read comes with the counts)
    s_bias_ids[i] = i < a.biases ? r.bias_ids[i] : -1;
    s_bias_values[i] = i < a.biases ? r.bias_values[i] : 0.f;
  }
  const bool counted = len > 0 && (r.rep != 1.f || r.freq != 0.f || r.pres != 0.f);
  const int prompt = a.prompts && counted ? a.prompts[row] : 0;
  const int mrow = a.mask_rows ? a.mask_rows[row] : row;
  const int* mask = a.mask && mrow >= 0 && mrow < a.mask_count ? a.mask + mrow * a.mask_ld : nullptr;
  const bool named = counted || a.biases > 0;
  float best = -INFINITY;
  int at = 0x7fffffff;
  auto better = [&](float v, int i) {
    if (v > best || (v == best && i < at)) {
      best = v;
      at = i;
    }
  };

  // The tokens on the list; one that ran over is left alone, and every token looked at.
  auto named_tokens = [&](int lo, int hi) {
    const bool listed = s_n <= kListMost;
    const int n = listed ? s_n : hi - lo;
    for (int e = tid; e < n; e += kRuleThreads) {
      const int t = listed ? s_list[e] : lo + e;
      const uint32_t c = counts.get(t - lo);
      if (!c || (c & C::kBiased) || (mask && !((uint32_t(mask[t >> 5]) >> (t & 31)) & 1u))) continue;
      const double l = ruled<WIDE>(r, rule_logit<F32>(in, t), c, 0.0);
      if (ids) better(float(l), t);
      else rule_store<F32>(out, t, F32 ? float(l) : to_odd(l));
    }
    // tokens with biases: the first entry of each
    for (int e = tid; e < a.biases; e += kRuleThreads) {
      const int t = e < kBiasMost ? s_bias_ids[e] : r.bias_ids[e];
      if (t < lo || t >= hi || (mask && !((uint32_t(mask[t >> 5]) >> (t & 31)) & 1u))) continue;
      bool first;
      const double bias = bias_sum(r, e, t, first);
      if (!first) continue;
      const double l = ruled<WIDE>(r, rule_logit<F32>(in, t), counts.get(t - lo), bias);
      if (ids) better(float(l), t);
      else rule_store<F32>(out, t, F32 ? float(l) : to_odd(l));
    }
  };

  for (int lo = first; lo < last; lo += C::kTokens) {
    const int hi = min(last, lo + C::kTokens), pieces = VEC ? (hi - lo) / kPer : 0;
    if (lo > first) load(lo, pieces, 0);
    if (named) {
      for (int i = tid; i < (WIDE ? 2 : 1) * ((hi - lo + kPer - 1) / kPer); i += kRuleThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0u, 0u, 0u, 0u);
      if (tid == 0) s_n = 0;
      __syncthreads();
      // who names a token first puts it on the list; places for a whole warp at once: one counter that many lanes add to takes them one after another
      auto list = [&](bool first_time, int t) {
        const uint32_t lanes = __ballot_sync(0xffffffffu, first_time);
        if (lanes == 0u) return;
        int base = 0;
        if ((tid & 31) == 0) base = atomicAdd(&s_n, __popc(lanes));
        const int e = __shfl_sync(0xffffffffu, base, 0) + __popc(lanes & ((1u << (tid & 31)) - 1u));
        if (first_time && e < kListMost) s_list[e] = t;
      };
      auto count = [&](int t, int i) {
        if (fresh && i == len - 1) t = newest;
        bool first_time = false;
        if (i < len && t >= lo && t < hi) first_time = i >= prompt ? counts.add(t - lo, 1u) : counts.mark(t - lo, C::kSeen);
        list(first_time, t);
      };
      if (counted) {
        const int most = (len + 127) & ~127;           // whole warps
        for (int i = 4 * tid; i < most; i += 4 * kRuleThreads) {
          int4 t = make_int4(-1, -1, -1, -1);
          if (early && i == 4 * tid) {
            t = ahead;
          } else if (token16 && i + 4 <= a.width) {
            t = *reinterpret_cast<const int4*>(tokens + i);
          } else {
            if (i < len) t.x = tokens[i];
            if (i + 1 < len) t.y = tokens[i + 1];
            if (i + 2 < len) t.z = tokens[i + 2];
            if (i + 3 < len) t.w = tokens[i + 3];
          }
          count(t.x, i);
          count(t.y, i + 1);
          count(t.z, i + 2);
          count(t.w, i + 3);
        }
      }
      for (int i = tid; i < a.biases; i += kRuleThreads) {
        const int t = r.bias_ids[i];
        if (t >= lo && t < hi) counts.mark(t - lo, C::kBiased);
      }
      __syncthreads();
      if (ids) named_tokens(lo, hi);
    }
    const uint8_t* mask8 = reinterpret_cast<const uint8_t*>(mask) + (lo >> 3);           // (slices begin at whole words)
    float top = -INFINITY;                  // of this thread's pieces, which come in ascending order
    int top_piece = -1;
    for (int p0 = 0; p0 < pieces; p0 += kAhead * kRuleThreads) {
      uint32_t left[VEC ? kAhead : 1];
#pragma unroll
      for (int i = 0; i < (VEC ? kAhead : 0); ++i) {
        const int p = p0 + i * kRuleThreads + tid;
        left[i] = mask && p < pieces ? mask8[p] : 255u;
      }
      uint8_t* to = out + (long long)lo * kBytes + (p0 + tid) * kPiece;
#pragma unroll
      for (int i = 0; i < (VEC ? kAhead : 0); ++i) {
        const int p = p0 + i * kRuleThreads + tid;
        if (p >= pieces) continue;
        if (ids) {
          const uint32_t plain = named ? left[i] & ~counts.named(p) : left[i];
          const float m = plain == 255u ? x[i].largest() : x[i].masked(plain).largest();
          if (m > top) {
            top = m;
            top_piece = p;
          }
        } else if (!in_place) {
          if (left[i] == 255u) x[i].store(to + i * (kRuleThreads * kPiece));
          else x[i].masked(left[i]).store(to + i * (kRuleThreads * kPiece));
        } else if (left[i] != 255u) {
          Piece<F32> y;
          y.load(to + i * (kRuleThreads * kPiece));
          y.masked(left[i]).store(to + i * (kRuleThreads * kPiece));
        }
      }
      if (p0 + kAhead * kRuleThreads < pieces) load(lo, pieces, p0 + kAhead * kRuleThreads);
    }
    if (top_piece >= 0) {
      // which of the piece's tokens it was
      Piece<F32> y;
      y.load(in + ((long long)lo + top_piece * kPer) * kBytes);
      uint32_t plain = mask ? mask8[top_piece] : 255u;
      if (named) plain &= ~counts.named(top_piece);
      int j = kPer;
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i)
        if (((plain >> i) & 1u) && y.value(i) == top) j = i;
      better(top, lo + top_piece * kPer + j);
    }
    constexpr int kSingles = VEC ? 1 : 8;       // tokens of a thread whose loads come together
    for (int t0 = lo + pieces * kPer + tid; t0 < hi; t0 += kSingles * kRuleThreads) {
      float l[kSingles];
      uint32_t word[kSingles];
#pragma unroll
      for (int i = 0; i < kSingles; ++i) {
        const int t = t0 + i * kRuleThreads;
        l[i] = t < hi && !in_place ? rule_logit<F32>(in, t) : 0.f;
        word[i] = t < hi && mask ? uint32_t(mask[t >> 5]) : ~0u;
      }
#pragma unroll
      for (int i = 0; i < kSingles; ++i) {
        const int t = t0 + i * kRuleThreads;
        if (t >= hi) break;
        const bool allowed = (word[i] >> (t & 31)) & 1u;
        if (ids) {
          if (allowed && !(named && counts.get(t - lo))) better(l[i], t);
        } else if (!allowed) {
          rule_store<F32>(out, t, -INFINITY);
        } else if (!in_place) {
          rule_store<F32>(out, t, l[i]);
        }
      }
    }
    if (named) {
      __syncthreads();
      if (!ids) named_tokens(lo, hi);        // over what the pass has written
      __syncthreads();
    }
  }
  if (!ids) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    better(v, i);
  }
  if ((tid & 31) == 0) {
    s_best[tid >> 5] = best;
    s_at[tid >> 5] = at;
  }
  __syncthreads();
  if (joined) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (tid == 0) {
    for (int w = 1; w < kRuleThreads / 32; ++w) better(s_best[w], s_at[w]);
    if (joined)
      asm volatile("st.shared::cluster.v2.s32 [%0], {%1, %2};" ::"r"(map_to_cta(&s_slices[blockIdx.x], 0)), "r"(__float_as_int(best)), "r"(at)
                   : "memory");
  }
  if (joined) {
    // the first CTA's shared memory has every slice's best once all have arrived; the others have nothing that anyone reads, and may leave
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (blockIdx.x != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0)
      for (unsigned c = 1; c < gridDim.x; ++c) better(__int_as_float(s_slices[c].x), s_slices[c].y);
  }
  if (blockIdx.x == 0 && tid == 0) a.out_ids[row] = best == -INFINITY ? -1 : at;
}

template <bool F32, bool VEC, bool WIDE>
static int launch_rules(const NkbLogitRules& a) {
  // Slices of a row: as few rounds of two CTAs per SM as may be, a round's time being some 3 us for every turn of counting and its logits at
  // an SM's share of the memory's rate; at most eight where a cluster joins them.
  const int slots = 2 * num_sms(), most = a.out_ids ? 8 : slots;
  constexpr int kStep = 512;
  int slices = 1;
  double best = 0.0;
  for (int s = 1; s <= most && (s == 1 || a.vocab > (s - 1) * kStep); ++s) {
    const double each = (double(a.vocab) + s - 1) / s;
    const double turns = double(int(each / Counts<WIDE>::kTokens) + 1), rounds = double(((long long)a.rows * s + slots - 1) / slots);
    const double us = rounds * (3.0 * turns + each * (F32 ? 4 : 2) * (a.out ? 2 : 1) / 22e3);
    if (s == 1 || us < best) {
      best = us;
      slices = s;
    }
  }
  const int slice = ((a.vocab + slices - 1) / slices + kStep - 1) / kStep * kStep;
  slices = (a.vocab + slice - 1) / slice;
  const int bytes = slice * (WIDE ? 4 : 2), smem = bytes < kCountBytes ? bytes : kCountBytes;
  constexpr int kMaxDev = 64;
  static bool ready[kMaxDev] = {false};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return -1;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(logit_rules_kernel<F32, VEC, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCountBytes);
    if (e != cudaSuccess) return int(e);
    ready[dev] = true;
  }
  return launch_pdl_cluster(logit_rules_kernel<F32, VEC, WIDE>, dim3(unsigned(slices), unsigned(a.rows)), dim3(kRuleThreads), size_t(smem),
                            reinterpret_cast<cudaStream_t>(a.stream), a.out_ids ? slices : 1, a, slice);
}

}  // namespace nkb

using namespace nkb;

extern "C" int nkb_logit_rules(const void* packed) {
  const NkbLogitRules& a = *reinterpret_cast<const NkbLogitRules*>(packed);
  if (!status_word() && nkb_init() != 0) return -1;
  if (a.rows <= 0) return 0;
  if (a.vocab <= 0 || a.rows > 65535 || (!a.out && !a.out_ids) || a.biases < 0 || a.width < 0) return -2;
  if (a.tokens && !a.lens) return -2;
  if (a.out && a.out_ids) return -2;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out);
  const bool vec = (at & 15) == 0 && ((a.ld | (a.out ? a.out_ld : 0)) & (a.fp32 ? 3 : 7)) == 0;
  const bool wide = a.width > int(Counts<false>::kTimes);
  auto go = [&](auto f32, auto v) {
    constexpr bool F = decltype(f32)::value, V = decltype(v)::value;
    return wide ? launch_rules<F, V, true>(a) : launch_rules<F, V, false>(a);
  };
  using T = std::true_type;
  using N = std::false_type;
  if (a.fp32) return vec ? go(T{}, T{}) : go(T{}, N{});
  return vec ? go(N{}, T{}) : go(N{}, N{});
}
