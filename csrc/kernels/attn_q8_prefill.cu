// Attention of packed prompts over 8-bit pages (kv_quant.cuh) on tcgen05.
//
//   o_i = sum_j 2^{s_ij + v_j} v8_j / sum_j 2^{s_ij},    s_ij = (scale / ln 2) 2^{k_j} (q_i . k8_j)
//
// The structure is that of prefill attention over bf16 pages (attn_prefill.cu: two 128-row query tiles in ping-pong, one MMA issuer each,
// S and O in tensor memory, one softmax thread per row, turns with the exponentials), with what 8 bits change:
//
//   warps 0-3    convert: a warp makes its page of every 128-token tile f16 in the swizzled layout that the MMA reads, and brings the
//                tokens to the tile's largest scale, 2^K for keys and 2^V for values, on the way
//   warps 4-11   softmax
//   warps 12, 13 issue tcgen05.mma
//   warp 14      reads the scales of the tiles to come and finds K and V
//   warp 15      fetches the pages, by bulk copies
//
// An e4m3 value is a multiple of 2^-9 and f16's steps end at 2^-24: with the tile's largest scale brought to 2^6, f16 holds the values of
// tokens down to 2^-21 of that scale exactly, and is off by 2^-25 at most (2^-38 of the largest value) below.  A tile's exponents are two
// numbers that enter where one number did before: 2^K in the multiplier of the scores, V in the exponent of the weights, 2^-V where the
// weights are summed.  Nothing is added per score.  There is no MMA of 16-bit queries with e4m3 keys, and keys in two parts on the 8-bit MMA
// would double the products.
//
// Rows of a query tile are (token, head of the group): short prompts fill tiles, and a tile's rows end close to one another.  Queries become
// f16 as they are loaded, each row scaled below 2^15 by a power of two.
//
// 128 exponentials per row want 2048 cycles per 256 x 128 scores, as many as its MMAs at 128 columns, so conversion has warps of its own, with
// the registers that the softmax leaves: 56 and 200 a thread (64 and 192: 2 sequences of 8000 753 us, 741 here).  What the loop takes is some
// 4000 cycles.  Two softmax warps and a converting one share a scheduler's issue slots: exponentials on the multiply-add units, which spare
// the special-function unit and take more instructions, made it slower (an eighth of them 793 us).  Shared memory, which MMAs, weights,
// conversion and copies share, is busy for 3500 cycles.  Weights in tensor memory would spare a fifth of those bytes; at 128 columns there is
// room for them only where the scores are, whose next product then waits for theirs (856 us, where it was 801), or with one place for the scores
// of both query tiles, which then wait for each other (781 for 741).
//
// Measured, beside the MMAs at 1658 TFLOP/s and bf16 pages: 32 heads of 128 on 8, 16 prompts of 1024 160 us (52, 195), 2 of 8000 737 (494, 785),
// one of 77 11.2 (0.2, 6.7; a fixed part of some 8 us); 64 heads of 64 on 8, 3 portions of up to 500 behind 4000 to 8000 tokens 241 (81, 258).
#include "api.h"
#include "kv_quant.cuh"
#include "attn_maps.h"
#include "query_turns.h"
#include <cuda_fp16.h>
#include <float.h>
#include <limits.h>
#include <math.h>

namespace nkb {

constexpr int kP8Tile = 128;             // query rows of an MMA tile, tokens of a K or V tile
constexpr int kP8Threads = 512;
constexpr int kP8Regs = 128;             // a thread's registers at launch; 2 * 128 * (56 + 200) is all of them
constexpr int kP8Slots = 8;              // tiles whose scales are kept
constexpr int kP8Lead = 4;               // tiles that warp 14 is ahead of the conversion of V at most
constexpr float kP8Grow = 8.f;           // log2 of the growth of a row's maximum that makes O follow
constexpr float kP8Lift = 6.f;           // log2 of a weight at the maximum, and of a value at the tile's largest scale
// log2 of what a tile's scales may lie above all that a row sees.  A key's elements are then off by 2^-20 of the row's largest at most (2^-25 of
// what is 2^6 at scale K; the largest is 224 or more at its own), and weights, whose exponent V is part of, by 2^-18 of the largest contribution
// (2^-25 of 2^6, by 2^12, and half of that).
constexpr int kP8MoreK = 18, kP8MoreV = 12;
constexpr int kP8Apart = 92;             // log2 of V of one tile over that of another: what is below 2^-126 is 2^-34 of the denominator then

struct PrefillQ8Params {
  const __nv_bfloat16* q;
  const uint8_t *k_values, *k_scales, *v_values, *v_scales;
  const int *block_table, *q_start, *q_lens, *context_lens;
  __nv_bfloat16* out;
  const float* sinks;
  int* status;
  int batch, total_q, nq, nkv, group, num_blocks, table_width, causal, window, chunk;
  int q_blocks;                          // 256-row blocks of the longest sequence
  long long table_stride;
  float scale_log2;
  unsigned int* sched;                   // [0] works taken, [1] CTAs done; zero between calls
  int parts;                             // of a block's tiles at most, each a work of its own
  int* counts;                           // [block] how many there are
  float* partials;                       // their results: [block][part][256 rows of D columns, then maxima, then sums]
  int* again;                            // [block][part] the work that this CTA looks at again behind this one (see p8_again)
};

// Piece of work of a CTA: 256 rows of a sequence's kv head
struct P8Range {                         // tiles [lo, hi) that a query tile attends to, and its rows
  int lo, hi, rows;
};
struct P8Work {
  int b, kvh, q_len, ctx, row0, q_start; // b < 0: none
  int block, part;                       // part: its number, and << 8 how many there are
  int u_lo, n_union;                     // tiles that either query tile attends to
  P8Range tr0, tr1;
  // tiles, from each one's first, whose exponentials the two take turns with
  __device__ __forceinline__ int paired() const { return tr1.rows > 0 ? nkb_turns_from_first(tr0.lo, tr0.hi, tr1.lo, tr1.hi) : 0; }
};
constexpr int kP8Least = 4;              // tiles that are divided, one or more to a part
constexpr int kP8Works = 3;              // works ahead of their use
constexpr int kP8Counts = 1024;          // blocks that may be divided: fewer than SMs
constexpr int kP8Readers = 15;           // warps 0 to 14 read them

struct PrefillQ8Ctrl {
  uint64_t q_full[2];
  uint64_t raw_full[4], raw_empty[4], kv_full[4], kv_empty[4];
  uint64_t e_full[kP8Slots], e_empty[kP8Slots];
  uint64_t s_full[2], s_empty[2], p_full[2], o_full[2], o_empty[2];
  uint64_t turn[2][4];
  uint64_t w_full[kP8Works], w_empty[kP8Works];
  P8Work works[kP8Works];
  int e_k[kP8Slots], e_v[kP8Slots];
  int pages[kP8Slots];                   // bits 0 to 3: the page is there; 4: all tokens of the tile are seen and are numbers
  uint8_t bytes[kP8Slots][2][kP8Tile];   // scales of K and of V
  uint32_t tmem_base;
  int abort;
  // (behind the others, whose places matter: with these two among them 16 prompts of 1024 tokens took 228 us for 224)
  int again;                             // the first work to look at again, < 0: none
  uint64_t done;                         // softmax warps and warp 14 have done all works
};

// Bounded barrier wait of a few instructions: the kernel has two dozen of them beside its unrolled loops, and a call would not allow the
// register split.  A try waits for some time by itself; so many tries are seconds.
constexpr uint32_t kP8Tries = 1u << 22;
__device__ __forceinline__ bool p8_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  uint32_t left = kP8Tries;
  while (!mbar_try_wait(bar, parity)) {
    if ((--left & 255u) == 0 && (left == 0 || *abort_flag)) {
      *abort_flag = 1;
      atomicCAS(status, 0, code | (blockIdx.x << 8));
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ P8Range p8_range(const PrefillQ8Params& p, int row0, int all_rows, int q_len, int ctx) {
  P8Range r{0, 0, 0};
  if (row0 >= all_rows) return r;
  r.rows = min(kP8Tile, all_rows - row0);
  const int first = ctx - q_len + row0 / p.group, last = ctx - q_len + (row0 + r.rows - 1) / p.group;
  r.hi = (max(ctx, 0) + kP8Tile - 1) / kP8Tile;
  if (p.causal) r.hi = min(r.hi, (max(last, -1) + kP8Tile) / kP8Tile);
  r.lo = nkb_first_visible(first, p.window, p.chunk) / kP8Tile;
  if (r.hi < r.lo) r.hi = r.lo;
  return r;
}
// Rows row0 .. of sequence b and kv head kvh; false: there are none
__device__ __forceinline__ bool p8_work(const PrefillQ8Params& p, int b, int kvh, int row0, int part, P8Work& o) {
  o.b = b;
  o.kvh = kvh;
  o.row0 = row0;
  o.block = (row0 / (2 * kP8Tile) * p.batch + b) * p.nkv + kvh;
  o.q_len = p.q_lens[b];
  o.q_start = p.q_start[b];
  o.ctx = min(p.context_lens[b], p.table_width * kQ8Page);
  if (row0 >= (long long)o.q_len * p.group) return false;
  const int all_rows = o.q_len * p.group;
  o.tr0 = p8_range(p, row0, all_rows, o.q_len, o.ctx);
  o.tr1 = p8_range(p, row0 + kP8Tile, all_rows, o.q_len, o.ctx);
  o.u_lo = o.tr0.lo;
  o.n_union = (o.tr1.rows > 0 ? max(o.tr0.hi, o.tr1.hi) : o.tr0.hi) - o.u_lo;
  // A block that sees little, of a table that may hold much, is one work: 77 tokens with a table of 8192 20.7 us in nine parts,
  // 13.7 here.
  const int parts = o.n_union < kP8Least ? 1 : min(p.parts, o.n_union);
  if (part >= parts) return false;
  o.part = part | parts << 8;
  if (parts > 1) {
    const int lo = o.u_lo + o.n_union * part / parts, hi = o.u_lo + o.n_union * (part + 1) / parts;
    for (P8Range* r : {&o.tr0, &o.tr1}) {
      r->lo = max(r->lo, lo);
      r->hi = max(min(r->hi, hi), r->lo);
    }
    o.u_lo = lo;
    o.n_union = hi - lo;
  }
  return true;
}
// The next work for a warp or (one = true) a single thread; n counts them.  False: there are no more, or the wait has run out.
__device__ __forceinline__ bool p8_next(PrefillQ8Ctrl* ctrl, uint32_t& n, P8Work& k, bool one, int* status) {
  const uint32_t slot = n % kP8Works;
  bool ok = p8_wait(&ctrl->w_full[slot], n / kP8Works & 1u, &ctrl->abort, status, ERR_WAIT_SMEM_FULL);
  if (!one) ok = __all_sync(0xffffffffu, ok);
  if (!ok) return false;
  k = ctrl->works[slot];
  ++n;
  if (!one) __syncwarp();
  if (one || (threadIdx.x & 31) == 0) mbar_arrive(&ctrl->w_empty[slot]);
  return k.b >= 0;
}
// Tokens [lo, hi) that some row of the work sees
__device__ __forceinline__ void p8_seen(const PrefillQ8Params& p, const P8Work& k, int& lo, int& hi) {
  lo = nkb_first_visible(k.ctx - k.q_len + k.row0 / p.group, p.window, p.chunk);
  hi = p.causal ? min(k.ctx, k.ctx - k.q_len + (min(k.row0 + 2 * kP8Tile, k.q_len * p.group) - 1) / p.group + 1) : k.ctx;
}
// Block of a page of walk position x; -1: none
__device__ __forceinline__ int p8_block(const PrefillQ8Params& p, const P8Work& k, int x, int page_of_tile) {
  const int page = (k.u_lo + x) * 4 + page_of_tile;
  const int blk = x < k.n_union && page * kQ8Page < k.ctx ? p.block_table[k.b * p.table_stride + page] : -1;
  return blk >= 0 && blk < p.num_blocks ? blk : -1;
}
// Ring items of a work in the order the issuers take them: K(0), then K(u + 1), V(u)
__device__ __forceinline__ bool p8_is_v(int i, int items) { return i > 0 && ((i & 1) == 0 || i == items - 1); }
__device__ __forceinline__ int p8_tile(int i, int items) { return i == 0 ? 0 : ((i & 1) == 0 ? i / 2 - 1 : min((i + 1) / 2, items / 2 - 1)); }

// What a row's sum of weighted values is multiplied by, from the exponent m of its weights and their sum (values are larger by 2^lift)
__device__ __forceinline__ float p8_inverse(const PrefillQ8Params& p, int head, float m, float l) {
  float scale = exp2f(-kP8Lift);
  if (p.sinks) {
    const float sk = p.sinks[head] * 1.4426950408889634f, m2 = fmaxf(m, sk), keep = m == -INFINITY ? 0.f : exp2f(m - m2);
    scale *= keep;
    l = l * keep + (sk == -INFINITY ? 0.f : exp2f(sk - m2 + kP8Lift));      // (no sink, and nothing seen: the sum stays zero)
  }
  return l == 0.f ? 0.f : scale / l;
}

template <int D>
struct PrefillQ8Smem {
  static constexpr int NH = D / 64;                       // 128-byte halves of a row
  static constexpr int kHalf = kP8Tile * 128;             // [128 rows][64 f16], swizzled
  static constexpr int kTile = NH * kHalf;                // Q, K or V tile
  static constexpr int kP = 2 * kHalf;                    // weights [128][128]
  static constexpr int kStages = D == 64 ? 4 : 2;         // of the f16 ring, and of every warp's ring of pages
  static constexpr int kPageBytes = kQ8Page * D;
  static constexpr int kBytes = 2 * kTile + kStages * (kTile + 4 * kPageBytes) + 2 * kP + int(sizeof(PrefillQ8Ctrl));
  static_assert(kBytes <= 232448, "shared memory of a CTA");
};

// 2^d as a pair of f16, 0 below what f16 has
__device__ __forceinline__ uint32_t f16x2_pow2(int d) {
  const uint32_t h = d >= -14 ? uint32_t(d + 15) << 10 : (d >= -24 ? 1u << (d + 24) : 0u);
  return h | (h << 16);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t p8_pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void st_shared_16(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Instruction descriptor for kind::f16 with f16 inputs and fp32 accumulation
__host__ __device__ constexpr uint32_t p8_idesc(int m, int n, int b_mn_major) {
  return (1u << 4) | (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// A warp's 32 rows in a swizzled tile, as it reads q and writes out: D / 8 lanes have a row's sixteen-byte pieces, kRows rows at a time.  (With
// a thread to a row every access would touch 32 lines: 16 sequences of 1024 tokens took 192 us for 166.)
template <int D>
struct P8Rows {
  static constexpr int kRows = 256 / D;
  int lane, piece, row;
  uint8_t* tile;
  __device__ __forceinline__ P8Rows(uint8_t* tile, int lane) : lane(lane), piece(lane % (D / 8)), row(lane / (D / 8)), tile(tile) {}
  // the piece of row `first` + row
  __device__ __forceinline__ uint4* wide(int first) const {
    return reinterpret_cast<uint4*>(tile + (piece >> 3) * kP8Tile * 128 + (first + row) * 128 + (((piece ^ (first + row)) & 7) << 4));
  }
  // piece i of row `lane`
  __device__ __forceinline__ uint4* own(int i) const {
    return reinterpret_cast<uint4*>(tile + (i >> 3) * kP8Tile * 128 + lane * 128 + (((i ^ lane) & 7) << 4));
  }
};

// ---- rows whose tiles hold scales far above all that they see
// A tile's scales K and V are the largest of its tokens, which some row sees and another does not.  To a row that sees only far smaller
// ones f16 has little of them left, and weights below a maximum that V is part of.  So warp 14 marks works where that may be: where a
// tile that not all rows see has scales far above its smallest and above those of the tiles that all rows see, or where V of the tiles lies so far
// apart that the denominator may lose a tile.  When a CTA has no more works, the four converting warps look at the rows of those once more
// and compute those that it concerns by 32-bit products, token by token (some 2 us of a warp per row and page, most of it latency), in the
// place of the first result.  Nothing of this is in the loop over tiles; what warp 14 notes costs a percent (16 prompts of 1024 157.3 -> 159.5
// us, 4 x 2000 of 64 columns with a window of 128 68.4 -> 70.1; noted by the converting warps half as much again).  16 prompts of 1024 with
// a first value of 2^-10 164 us, with a first key and value of zero 191.

__device__ __forceinline__ int p8_page_block(const PrefillQ8Params& p, int b, int page) {
  const int blk = p.block_table[b * p.table_stride + page];
  return blk >= 0 && blk < p.num_blocks ? blk : -1;
}

// Largest scales (bytes) of a tile: of what the work sees, and of what this lane's row sees of it, [lo, hi].  Lanes have four tokens each.
struct P8Largest {
  int k_tile, v_tile, k_row, v_row;
};
__device__ __forceinline__ int p8_top_byte(uint32_t pairs) { return int(max(pairs & 0xffffu, pairs >> 16)); }
__device__ __forceinline__ void p8_largest(const PrefillQ8Params& p, const P8Work& k, int tile, int vis_lo, int vis_hi, int lo, int hi, int lane,
                                           bool mine, P8Largest& o) {
  constexpr uint32_t kAll = 0xffffffffu, kEven = 0x00ff00ffu;
  const int page = tile * 4 + (lane >> 3), tok0 = tile * kP8Tile + lane * 4;
  const int blk = page * kQ8Page < k.ctx ? p8_page_block(p, k.b, page) : -1;
  uint32_t kb = 0u, vb = 0u;
  if (blk >= 0) {
    const long long at = ((long long)blk * p.nkv + k.kvh) * kQ8Page + (lane & 7) * 4;
    kb = *reinterpret_cast<const uint32_t*>(p.k_scales + at);
    vb = *reinterpret_cast<const uint32_t*>(p.v_scales + at);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (tok0 + j < vis_lo || tok0 + j >= vis_hi || ((kb >> (8 * j)) & 255) == 255 || ((vb >> (8 * j)) & 255) == 255) {
      kb &= ~(255u << (8 * j));
      vb &= ~(255u << (8 * j));
    }
  }
  const int k_top = __reduce_max_sync(kAll, p8_top_byte(__vmaxu2(kb & kEven, (kb >> 8) & kEven)));
  const int v_top = __reduce_max_sync(kAll, p8_top_byte(__vmaxu2(vb & kEven, (vb >> 8) & kEven)));
  uint32_t k_row = 0u, v_row = 0u;
#pragma unroll 4
  for (int i = 0; i < 32; ++i) {
    const int from = min(max(lo - (tile * kP8Tile + 4 * i), 0), 4), end = min(max(hi + 1 - (tile * kP8Tile + 4 * i), 0), 4);
    const uint32_t seen = end > from ? (0xffffffffu >> (8 * (4 - end + from))) << (8 * from) : 0u;
    const uint32_t kw = __shfl_sync(kAll, kb, i) & seen, vw = __shfl_sync(kAll, vb, i) & seen;
    k_row = __vmaxu2(__vmaxu2(k_row, kw & kEven), (kw >> 8) & kEven);
    v_row = __vmaxu2(__vmaxu2(v_row, vw & kEven), (vw >> 8) & kEven);
  }
  if (mine) {
    o.k_tile = max(o.k_tile, k_top);
    o.v_tile = max(o.v_tile, v_top);
    o.k_row = max(o.k_row, p8_top_byte(k_row));
    o.v_row = max(o.v_row, p8_top_byte(v_row));
  }
}

// One row (`at`, of heads) by a warp, over positions [lo, hi].  A whole result goes to its place; that of a part to `part`, with its maximum
// and sum at `tail`.
template <int D>
__device__ __forceinline__ void p8_row(const PrefillQ8Params& p, const P8Work& k, long long at, int head, int lo, int hi, float* part, float* tail,
                                       int lane) {
  constexpr int N = D / 32;
  constexpr uint32_t kAll = 0xffffffffu;
  const __nv_bfloat16* q = p.q + at * D;
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) mx = fmaxf(mx, fabsf(__bfloat162float(q[lane * N + i])));
  mx = warp_max(mx);
  const int e = max((__float_as_int(mx) >> 23) - 127, -100);
  const float up = exp2_int(14 - e), rs = p.scale_log2 * exp2_int(e - 14);
  float m = -INFINITY, l = 0.f, o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  const int last = hi >> 5;
  int blk_n = p8_page_block(p, k.b, lo >> 5);
  const auto scale_of = [&](const uint8_t* scales, int blk) {
    return blk >= 0 ? scales[((long long)blk * p.nkv + k.kvh) * kQ8Page + lane] : 127;
  };
  int kb_n = scale_of(p.k_scales, blk_n), vb_n = scale_of(p.v_scales, blk_n);
#pragma unroll 1
  for (int page = lo >> 5; page <= last; ++page) {
    const int blk = blk_n, kb = kb_n, vb = vb_n, tok = page * kQ8Page + lane;
    const long long first = ((long long)max(blk, 0) * p.nkv + k.kvh) * kQ8Page;
    blk_n = page < last ? p8_page_block(p, k.b, page + 1) : -1;
    float dot = 0.f;
    if (blk >= 0) {
      const uint4* key = reinterpret_cast<const uint4*>(p.k_values + (first + lane) * D);
      constexpr int kAhead = 4;
#pragma unroll 1
      for (int c = 0; c < D / 16; c += kAhead) {
        uint4 x4[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x4[i] = key[c + i];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const uint32_t x[4] = {x4[i].x, x4[i].y, x4[i].z, x4[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint2 q4 = *reinterpret_cast<const uint2*>(q + (c + i) * 16 + j * 4);
            const float2 q0 = unpack_bf16x2(q4.x), q1 = unpack_bf16x2(q4.y);
            const uint32_t h0 = e4m3x2_to_f16x2(uint16_t(x[j])), h1 = e4m3x2_to_f16x2(uint16_t(x[j] >> 16));
            const float2 k0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), k1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
            dot = fmaf(q0.x * up, k0.x, fmaf(q0.y * up, k0.y, fmaf(q1.x * up, k1.x, fmaf(q1.y * up, k1.y, dot))));
          }
        }
      }
    }
    kb_n = scale_of(p.k_scales, blk_n);
    vb_n = scale_of(p.v_scales, blk_n);
    float s = dot * rs * q8_factor_of(kb);
    if (vb == 255) s = __int_as_float(0x7fc00000);
    const bool seen = tok >= lo && tok <= hi;
    if (!seen) s = -INFINITY;
    const float top = fmaxf(m, warp_max(s));
    const float keep = m == top ? 1.f : exp2f(m - top), w = exp2f(s - (top == -INFINITY ? 0.f : top) + kP8Lift);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= keep;
    // (NaN goes on; what is not seen may be anything)
    const float to_o = seen ? w * exp2_int(q8_log2_of(vb) + int(kP8Lift)) : 0.f;
    if (blk < 0) continue;
    const uint8_t* value = p.v_values + first * D + lane * N;
    constexpr int kRows = 16;
#pragma unroll 1
    for (int j0 = 0; j0 < kQ8Page; j0 += kRows) {
      uint32_t x[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if constexpr (N == 4) x[j] = *reinterpret_cast<const uint32_t*>(value + (j0 + j) * D);
        else x[j] = *reinterpret_cast<const uint16_t*>(value + (j0 + j) * D);
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const float wj = __shfl_sync(kAll, to_o, j0 + j);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const uint32_t h = e4m3x2_to_f16x2(uint16_t(x[j] >> (8 * i)));
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
          o[i] = wj == 0.f ? o[i] : fmaf(wj, v.x, o[i]);
          o[i + 1] = wj == 0.f ? o[i + 1] : fmaf(wj, v.y, o[i + 1]);
        }
      }
    }
  }
  l = warp_sum(l);
  if (part) {
#pragma unroll
    for (int i = 0; i < N; ++i) part[lane * N + i] = o[i];
    if (lane == 0) {
      tail[0] = m;
      tail[2 * kP8Tile] = l;
    }
  } else {
    const float inv = p8_inverse(p, head, m, l);
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + at * D) + lane * (N / 2);
#pragma unroll
    for (int i = 0; i < N; i += 2) dst[i / 2] = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
  }
}

// The works from `head` on; a warp has every fourth of a work's rows.
template <int D>
__device__ __forceinline__ void p8_again(const PrefillQ8Params& p, int head, int warp, int lane) {
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr long long kPart = 2 * kP8Tile * (D + 2);
#pragma unroll 1
  while (head >= 0) {
    const int id = head >> 1, block = id / p.parts;
    const bool apart = head & 1;
    head = *(volatile const int*)(p.again + id);
    P8Work k;
    if (!p8_work(p, block / p.nkv % p.batch, block % p.nkv, block / (p.nkv * p.batch) * 2 * kP8Tile, id % p.parts, k)) return;
    int vis_lo, vis_hi;
    p8_seen(p, k, vis_lo, vis_hi);
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const P8Range tr = t == 0 ? k.tr0 : k.tr1;
      const int r = lane * 4 + warp, row = k.row0 + t * kP8Tile + r, token = row / p.group, q_pos = k.ctx - k.q_len + token;
      const long long q_row = (long long)k.q_start + token;
      const int hi = min(p.causal ? min(k.ctx - 1, q_pos) : k.ctx - 1, tr.hi * kP8Tile - 1);
      const int lo = max(nkb_first_visible(q_pos, p.window, p.chunk), tr.lo * kP8Tile);
      const bool there = r < tr.rows && q_row >= 0 && q_row < p.total_q && lo <= hi;
      bool concerned = there && apart;
      if (!apart) {
        // the tiles at the ends of what the row sees, and the whole one before its last
        P8Largest most{0, 0, 0, 0};
        const int first = __reduce_min_sync(kAll, there ? lo >> 7 : INT_MAX), last = __reduce_max_sync(kAll, there ? hi >> 7 : -1);
        for (int tile = first; tile <= last; ++tile) {
          const bool mine = there && (tile == lo >> 7 || tile == hi >> 7 || (tile == (hi >> 7) - 1 && tile >= lo >> 7));
          if (!__any_sync(kAll, mine)) continue;
          p8_largest(p, k, tile, vis_lo, vis_hi, lo, hi, lane, mine, most);
        }
        concerned = there && (q8_log2_of(most.k_tile) - q8_log2_of(most.k_row) > kP8MoreK || q8_log2_of(most.v_tile) - q8_log2_of(most.v_row) > kP8MoreV);
      }
      uint32_t todo = __ballot_sync(kAll, concerned);
#pragma unroll 1
      while (todo) {
        const int j = __ffs(todo) - 1;
        todo &= todo - 1;
        const int one = __shfl_sync(kAll, row, j), one_token = one / p.group, one_head = k.kvh * p.group + one % p.group;
        const long long at = ((long long)k.q_start + one_token) * p.nq + one_head;
        float *part = nullptr, *tail = nullptr;
        if (k.part >> 8 > 1) {
          float* mine = p.partials + ((long long)k.block * p.parts + (k.part & 255)) * kPart;
          const int in_pair = t * kP8Tile + j * 4 + warp;
          part = mine + in_pair * D;
          tail = mine + 2 * kP8Tile * D + in_pair;
        }
        p8_row<D>(p, k, at, one_head, __shfl_sync(kAll, lo, j), __shfl_sync(kAll, hi, j), part, tail, lane);
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kP8Threads, 1) attn_q8_prefill_kernel(const PrefillQ8Params p) {
  using L = PrefillQ8Smem<D>;
  constexpr int NH = L::NH, kHalf = L::kHalf, kStages = L::kStages;
  constexpr uint32_t kAll = 0xffffffffu, kTmemCols = 512, kSCol = 0, kOCol = 256;
  extern __shared__ __align__(1024) uint8_t p8_smem[];    // the swizzle wants it on 1024 bytes, and there is no static memory ahead of it
  uint8_t* q_s = p8_smem;
  uint8_t* kv_s = q_s + 2 * L::kTile;
  uint8_t* raw_s = kv_s + kStages * L::kTile;
  uint8_t* p_s = raw_s + kStages * 4 * L::kPageBytes;
  PrefillQ8Ctrl* ctrl = reinterpret_cast<PrefillQ8Ctrl*>(p_s + 2 * L::kP);
  const int warp = warp_idx_uniform(), lane = threadIdx.x & 31;
  if (smem_u32(p8_smem) & 1023) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, ERR_BAD_ARGUMENT);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ctrl->raw_full[i], 4);                   // one arrival for each page
      mbar_init(&ctrl->raw_empty[i], 4);                  // one from each converting warp, as below
      mbar_init(&ctrl->kv_full[i], 4);                    // one arrival from each converting warp
      mbar_init(&ctrl->kv_empty[i], 2);                   // one from each query tile's issuer
    }
    for (int i = 0; i < kP8Works; ++i) {
      mbar_init(&ctrl->w_full[i], 1);
      mbar_init(&ctrl->w_empty[i], kP8Readers);
    }
    for (int i = 0; i < kP8Slots; ++i) {
      mbar_init(&ctrl->e_full[i], 1);
      mbar_init(&ctrl->e_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctrl->q_full[i], 4);
      mbar_init(&ctrl->s_full[i], 1);
      mbar_init(&ctrl->s_empty[i], 4);
      mbar_init(&ctrl->p_full[i], 4);
      mbar_init(&ctrl->o_full[i], 1);
      mbar_init(&ctrl->o_empty[i], 4);
      for (int q = 0; q < 4; ++q) mbar_init(&ctrl->turn[i][q], 1);
    }
    mbar_init(&ctrl->done, 9);
    ctrl->abort = 0;
    ctrl->again = -1;
    mbar_fence_init();
    fence_proxy_async();
  }
  if (warp == 12) {
    tmem_alloc(&ctrl->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(kAll, ctrl->tmem_base, 0);
  volatile int* abort_flag = &ctrl->abort;
  griddep_wait();
  griddep_launch();

  if (warp < 4) {
    // ---------------------------------------------------------------- conversion
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    constexpr int kRows = 512 / D, kSteps = kQ8Page / kRows;       // tokens per sixteen-byte load of the warp, loads per page
    constexpr int kLanes = D / 16;                                 // lanes that share a token
    const int piece = lane % kLanes, row_of = lane / kLanes;
    // where the lane's two chunks of a row go: where eight lanes have one row (D = 128), those of its second half take their eight-byte halves
    // the other way round, so that all banks are used
    const int odd = NH == 2 ? piece >> 2 : 0;
    const uint32_t to0 = smem_u32(kv_s) + (piece >> 2) * kHalf + (warp * kQ8Page + row_of) * 128 + ((((piece & 3) * 2 + odd) ^ row_of) << 4);
    const uint8_t* from0 = raw_s + warp * L::kPageBytes + lane * 16;
    uint32_t item0 = 0, tiles0 = 0;                                // ring items and tiles of the works before
    uint32_t n_works = 0;
    bool alive = true;
    P8Work k;
#pragma unroll 1
    while (alive && p8_next(ctrl, n_works, k, false, p.status)) {
      int vis_lo, vis_hi;
      p8_seen(p, k, vis_lo, vis_hi);
      const int items = 2 * k.n_union;
#pragma unroll 1
      for (int i = 0; i < items; ++i) {
        const bool v_item = p8_is_v(i, items);
        const int x = p8_tile(i, items), st = (item0 + i) % kStages, slot = (tiles0 + x) % kP8Slots;
        const uint32_t ph = (item0 + i) / kStages & 1u;
        bool ok = v_item || p8_wait(&ctrl->e_full[slot], (tiles0 + x) / kP8Slots & 1u, abort_flag, p.status, ERR_WAIT_SMEM_FULL);
        ok = ok && p8_wait(&ctrl->raw_full[st], ph, abort_flag, p.status, ERR_WAIT_SMEM_FULL);
        ok = ok && p8_wait(&ctrl->kv_empty[st], ph ^ 1u, abort_flag, p.status, ERR_WAIT_SMEM_EMPTY);
        if (!__all_sync(kAll, ok)) {
          alive = false;
          break;
        }
        // factor of token `lane` of the page
        const int pages = ctrl->pages[slot], byte = ctrl->bytes[slot][v_item][warp * kQ8Page + lane];
        const bool whole = pages & 16;
        uint32_t fac = f16x2_pow2(q8_log2_of(byte) - (v_item ? ctrl->e_v[slot] : ctrl->e_k[slot]) + int(kP8Lift));
        const int tok0 = (k.u_lo + x) * kP8Tile + warp * kQ8Page;
        if (!whole) {
          // NaN, K's or V's, is one of the scores: a row that does not see the token must not meet it in a product
          const bool none = byte == 255 || ctrl->bytes[slot][!v_item][warp * kQ8Page + lane] == 255;
          if (none) fac = v_item ? 0u : 0x7fff7fffu;
          if (tok0 + lane < vis_lo || tok0 + lane >= vis_hi) fac = 0u;
        }
        const int lo = vis_lo - tok0 - row_of, hi = (pages >> warp) & 1 ? vis_hi - tok0 - row_of : -kQ8Page;
        const uint8_t* from = from0 + st * 4 * L::kPageBytes;
        const uint32_t to = to0 + st * L::kTile;
        // four loads at a time, then their stores (a load behind a store would wait for it)
        constexpr int kAhead = 4;
#pragma unroll
        for (int j0 = 0; j0 < kSteps; j0 += kAhead) {
          uint2 ra[kAhead], rc[kAhead];
          uint32_t f[kAhead];
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            const uint8_t* at = from + (j0 + j) * 512;
            const uint4 both = *reinterpret_cast<const uint4*>(at);
            ra[j] = odd ? make_uint2(both.z, both.w) : make_uint2(both.x, both.y);
            rc[j] = odd ? make_uint2(both.x, both.y) : make_uint2(both.z, both.w);
          }
#pragma unroll
          for (int j = 0; j < kAhead; ++j) f[j] = __shfl_sync(kAll, fac, (j0 + j) * kRows + row_of);
          if (!whole) {                                              // what no row sees may be anything
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
              if ((j0 + j) * kRows < lo || (j0 + j) * kRows >= hi) ra[j] = rc[j] = make_uint2(0u, 0u);
          }
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            const uint4 a = make_uint4(hmul2(e4m3x2_to_f16x2(uint16_t(ra[j].x)), f[j]), hmul2(e4m3x2_to_f16x2(uint16_t(ra[j].x >> 16)), f[j]),
                                       hmul2(e4m3x2_to_f16x2(uint16_t(ra[j].y)), f[j]), hmul2(e4m3x2_to_f16x2(uint16_t(ra[j].y >> 16)), f[j]));
            const uint4 c = make_uint4(hmul2(e4m3x2_to_f16x2(uint16_t(rc[j].x)), f[j]), hmul2(e4m3x2_to_f16x2(uint16_t(rc[j].x >> 16)), f[j]),
                                       hmul2(e4m3x2_to_f16x2(uint16_t(rc[j].y)), f[j]), hmul2(e4m3x2_to_f16x2(uint16_t(rc[j].y >> 16)), f[j]));
            // rows four on: bit 2 of the swizzle
            const uint32_t at = (to ^ (kRows == 4 && (j & 1) ? 64u : 0u)) + (j0 + j) * kRows * 128;
            st_shared_16(at, a);
            st_shared_16(at ^ 16u, c);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ctrl->kv_full[st]);
          mbar_arrive(&ctrl->raw_empty[st]);
          if (v_item) mbar_arrive(&ctrl->e_empty[slot]);
        }
      }
      item0 += items;
      tiles0 += k.n_union;
    }
    alive = p8_wait(&ctrl->done, 0, abort_flag, p.status, ERR_WAIT_SOFTMAX);
    if (__all_sync(kAll, alive) && !*abort_flag) p8_again<D>(p, ctrl->again, warp, lane);
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 15) {
      // -------------------------------------------------------------- pages: lanes 0 to 3 a page of the item each
      // and the works: a CTA's first has its number, the others come from a counter of the grid.  The last rows of all sequences first, those
      // with the longest contexts ahead.
      const int across = p.nkv * p.batch * p.parts;
      int order = lane;                                   // (up to 32 sequences) the sequence of rank `lane`
      if (p.batch > 1 && p.batch <= 32) {
        const int ctx = lane < p.batch ? p.context_lens[lane] : INT_MIN;
        int rank = 0;
        for (int j = 0; j < p.batch; ++j) {
          const int c = __shfl_sync(kAll, ctx, j);
          rank += c > ctx || (c == ctx && j < lane);
        }
        for (int j = 0; j < p.batch; ++j)
          if (__shfl_sync(kAll, rank, j) == lane) order = j;
      }
      auto take = [&]() {
        unsigned int w = 0;
        if (lane == 0) w = gridDim.x + atomicAdd(p.sched, 1u);
        return w;
      };
      uint32_t item0 = 0, n_works = 0;
      unsigned int taken = blockIdx.x;
      bool alive = true;
      P8Work k;
#pragma unroll 1
      while (alive) {
        const unsigned int w = __shfl_sync(kAll, taken, 0), level = w / across;
        k.b = -1;
        k.n_union = 0;
        if (level < unsigned(p.q_blocks)) {
          const int rest = int(w % across), head = rest / p.parts, b = head / p.nkv;
          if (!p8_work(p, p.batch <= 32 ? __shfl_sync(kAll, order, b & 31) : b, head % p.nkv, (p.q_blocks - 1 - int(level)) * 2 * kP8Tile,
                       rest % p.parts, k)) {
            taken = take();
            continue;
          }
        }
        const int items = 2 * k.n_union;
        int blk = items > 0 && lane < 4 ? p8_block(p, k, 0, lane) : -1;
        const bool free_slot = p8_wait(&ctrl->w_empty[n_works % kP8Works], (n_works / kP8Works & 1u) ^ 1u, abort_flag, p.status, ERR_WAIT_SMEM_EMPTY);
        if (!__all_sync(kAll, free_slot)) break;
        if (lane == 0) {
          ctrl->works[n_works % kP8Works] = k;
          mbar_arrive(&ctrl->w_full[n_works % kP8Works]);
        }
        __syncwarp();
        ++n_works;
        if (k.b < 0) break;
#pragma unroll 1
        for (int i = 0; i < items; ++i, ++item0) {
          if (i == max(items - 3, 0)) taken = take();     // late, so that works go to who is free, and early enough to be there
          const int st = item0 % kStages;
          const int next = i + 1 < items && lane < 4 ? p8_block(p, k, p8_tile(i + 1, items), lane) : -1;
          const bool ok = p8_wait(&ctrl->raw_empty[st], (item0 / kStages & 1u) ^ 1u, abort_flag, p.status, ERR_WAIT_SMEM_EMPTY);
          if (!__all_sync(kAll, ok)) {
            alive = false;
            break;
          }
          if (lane < 4) {
            uint64_t* bar = &ctrl->raw_full[st];
            if (blk >= 0) {
              mbar_expect_tx(bar, L::kPageBytes);
              bulk_load_1d(raw_s + (st * 4 + lane) * L::kPageBytes,
                           (p8_is_v(i, items) ? p.v_values : p.k_values) + ((long long)blk * p.nkv + k.kvh) * L::kPageBytes, L::kPageBytes, bar);
            } else {
              mbar_arrive(bar);
            }
          }
          __syncwarp();
          blk = next;
        }
        if (items == 0) taken = take();
      }
    } else if (warp == 14) {
      // -------------------------------------------------------------- scales: a lane has tokens 4 lane .. 4 lane + 3 of a tile
      uint32_t tiles0 = 0, n_works = 0;
      bool alive = true;
      P8Work k;
#pragma unroll 1
      while (alive && p8_next(ctrl, n_works, k, false, p.status)) {
        auto scales_of = [&](const uint8_t* at, int blk) {
          // (a page that is not there has no say in the tile's scale)
          return blk >= 0 ? *reinterpret_cast<const uint32_t*>(at + ((long long)blk * p.nkv + k.kvh) * kQ8Page + (lane & 7) * 4) : 0u;
        };
        int vis_lo, vis_hi;
        p8_seen(p, k, vis_lo, vis_hi);
        // tokens [all_lo, all_hi) are seen by all rows, whose positions are less than 256 apart
        const int all_hi = p.causal ? vis_hi - 2 * kP8Tile : vis_hi, all_lo = p.chunk > 0 ? INT_MAX : (p.window > 0 ? vis_lo + 2 * kP8Tile : 0);
        // for p8_again: largest scales of tiles that all rows see, and of others; this lane's least of the others; V's ends
        constexpr int kNone = 1000;
        int in_k = -kNone, in_v = -kNone, at_k = -2 * kNone, at_v = -2 * kNone;
        uint32_t k_low = 0x00ff00ffu, v_low = 0x00ff00ffu;
        int v_most = -kNone, v_least = kNone;
        int blk = p8_block(p, k, 0, lane >> 3), blk_n = p8_block(p, k, 1, lane >> 3);
        uint32_t kb = scales_of(p.k_scales, blk), vb = scales_of(p.v_scales, blk);
#pragma unroll 1
        for (int x = 0; x < k.n_union; ++x, ++tiles0) {
          const uint32_t kb_n = scales_of(p.k_scales, blk_n), vb_n = scales_of(p.v_scales, blk_n);
          const int blk_2 = p8_block(p, k, x + 2, lane >> 3), slot = tiles0 % kP8Slots, tile0 = (k.u_lo + x) * kP8Tile;
          // The tile eight before had this slot.  Its V, and with it its softmax, is behind the V of four tiles before, which is converted
          // after that of six before has been used.
          if (tiles0 >= kP8Lead) {
            const uint32_t past = tiles0 - kP8Lead;
            const bool ok = p8_wait(&ctrl->e_empty[past % kP8Slots], past / kP8Slots & 1u, abort_flag, p.status, ERR_WAIT_SMEM_EMPTY);
            if (!__all_sync(kAll, ok)) {
              alive = false;
              break;
            }
          }
          uint32_t k4 = kb, v4 = vb, k_up = blk >= 0 ? kb : 0xffffffffu, v_up = blk >= 0 ? vb : 0xffffffffu;
          bool all = blk >= 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int tok = tile0 + lane * 4 + j;
            if (tok >= vis_hi || tok < vis_lo || ((kb >> (8 * j)) & 255) == 255 || ((vb >> (8 * j)) & 255) == 255) {
              k4 &= ~(255u << (8 * j));                   // such a token has no say in the tile's scale
              v4 &= ~(255u << (8 * j));
              k_up |= 255u << (8 * j);
              v_up |= 255u << (8 * j);
              all = false;
            }
          }
          const uint32_t k2 = __vmaxu2(k4 & 0x00ff00ffu, (k4 >> 8) & 0x00ff00ffu), v2 = __vmaxu2(v4 & 0x00ff00ffu, (v4 >> 8) & 0x00ff00ffu);
          const int ek = q8_log2_of(int(__reduce_max_sync(kAll, max(k2 & 0xffffu, k2 >> 16))));
          const int ev = q8_log2_of(int(__reduce_max_sync(kAll, max(v2 & 0xffffu, v2 >> 16))));
          const uint32_t there = __ballot_sync(kAll, blk >= 0);
          const bool whole = __all_sync(kAll, all);
          *reinterpret_cast<uint32_t*>(&ctrl->bytes[slot][0][lane * 4]) = kb;
          *reinterpret_cast<uint32_t*>(&ctrl->bytes[slot][1][lane * 4]) = vb;
          if (lane == 0) {
            ctrl->e_k[slot] = ek;
            ctrl->e_v[slot] = ev;
            ctrl->pages[slot] = int((there & 1) | ((there >> 7) & 2) | ((there >> 14) & 4) | ((there >> 21) & 8)) | (whole ? 16 : 0);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctrl->e_full[slot]);
          v_most = max(v_most, ev);
          v_least = min(v_least, ev);
          if (tile0 >= all_lo && tile0 + kP8Tile <= all_hi) {
            in_k = max(in_k, ek);
            in_v = max(in_v, ev);
          } else {
            at_k = max(at_k, ek);
            at_v = max(at_v, ev);
            k_low = __vminu2(__vminu2(k_low, k_up & 0x00ff00ffu), (k_up >> 8) & 0x00ff00ffu);
            v_low = __vminu2(__vminu2(v_low, v_up & 0x00ff00ffu), (v_up >> 8) & 0x00ff00ffu);
          }
          kb = kb_n;
          vb = vb_n;
          blk = blk_n;
          blk_n = blk_2;
        }
        // (a lane's own least tokens: where there are any so small, some lane has them)
        const int k_least = q8_log2_of(int(min(k_low & 0xffffu, k_low >> 16))), v_least_at = q8_log2_of(int(min(v_low & 0xffffu, v_low >> 16)));
        const bool apart = v_most - v_least > kP8Apart;
        const bool again = apart || at_k > max(in_k, k_least) + kP8MoreK || at_v > max(in_v, v_least_at) + kP8MoreV;
        if (__any_sync(kAll, again) && lane == 0) {
          const int id = k.block * p.parts + (k.part & 255);
          p.again[id] = ctrl->again;
          ctrl->again = 2 * id + (apart ? 1 : 0);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctrl->done);
    }
    // ---------------------------------------------------------------- MMA issuers, one per query tile (see attn_prefill.cu)
    constexpr uint32_t idesc_qk = p8_idesc(128, kP8Tile, 0), idesc_pv = p8_idesc(128, D, 1);
    const int t = warp - 12;
    if (t < 2 && elect_one()) {
      const uint32_t q_lo = uint32_t(make_smem_desc_sw128(smem_u32(q_s + t * L::kTile), 0, 1024));
      const uint32_t kv_lo = uint32_t(make_smem_desc_sw128(smem_u32(kv_s), 0, 1024));
      const uint32_t p_lo = uint32_t(make_smem_desc_sw128(smem_u32(p_s + t * L::kP), 0, 1024));
      const uint64_t hk = uint64_t(uint32_t(make_smem_desc_sw128(0, 0, 1024) >> 32)) << 32;
      const uint32_t lbo_v = (uint32_t(kHalf) >> 4) << 16;
      const uint32_t s_tmem = tmem_base + kSCol + t * 128, o_tmem = tmem_base + kOCol + t * 128;
      bool ok = true;
      uint32_t item = 0, tiles = 0;                       // ring items, and tiles that this query tile attended to
      uint32_t results = 0;                               // works in which it had any
      int a_lo = 0, a_hi = 0, n_union = 0;
      auto do_k = [&](int x) {
        if (x >= n_union || !ok) return;
        const uint32_t st = item % kStages, ph = item / kStages & 1u;
        ++item;
        ok = p8_wait(&ctrl->kv_full[st], ph, abort_flag, p.status, ERR_WAIT_SMEM_FULL);
        if (!ok) return;
        if (x >= a_lo && x < a_hi) {
          ok = p8_wait(&ctrl->s_empty[t], (tiles + uint32_t(x - a_lo) & 1u) ^ 1u, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY);
          if (!ok) return;
          tc_fence_after();
          const uint32_t kvd = kv_lo + uint32_t(st * L::kTile >> 4);
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            uint64_t da[4], db[4];
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              da[k4] = hk | (q_lo + uint32_t(h * (kHalf >> 4) + k4 * 2));
              db[k4] = hk | (kvd + uint32_t(h * (kHalf >> 4) + k4 * 2));
            }
            umma4_ss(s_tmem, da, db, idesc_qk, h > 0 ? 1u : 0u);
          }
          umma_commit(&ctrl->s_full[t]);
        }
        umma_commit(&ctrl->kv_empty[st]);
      };
      auto do_v = [&](int x) {
        if (!ok) return;
        const uint32_t st = item % kStages, ph = item / kStages & 1u;
        ++item;
        ok = p8_wait(&ctrl->kv_full[st], ph, abort_flag, p.status, ERR_WAIT_SMEM_FULL);
        if (!ok) return;
        if (x >= a_lo && x < a_hi) {
          // O_t of the work before has been read
          if (x == a_lo) ok = p8_wait(&ctrl->o_empty[t], (results & 1u) ^ 1u, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY);
          ok = ok && p8_wait(&ctrl->p_full[t], tiles + uint32_t(x - a_lo) & 1u, abort_flag, p.status, ERR_WAIT_SOFTMAX);
          if (!ok) return;
          tc_fence_after();
          const uint32_t kvd = kv_lo + uint32_t(st * L::kTile >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint64_t da[4], db[4];
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              db[k4] = hk | ((kvd + uint32_t((h * 4 + k4) * 128)) | lbo_v);
              da[k4] = hk | (p_lo + uint32_t(h * (kHalf >> 4) + k4 * 2));
            }
            umma4_ss(o_tmem, da, db, idesc_pv, (x > a_lo || h > 0) ? 1u : 0u);
          }
          umma_commit(&ctrl->o_full[t]);
        }
        umma_commit(&ctrl->kv_empty[st]);
      };
      uint32_t n_works = 0;
      P8Work k;
#pragma unroll 1
      while (ok && p8_next(ctrl, n_works, k, true, p.status)) {
        const P8Range tr = t == 0 ? k.tr0 : k.tr1;
        n_union = k.n_union;
        a_lo = a_hi = 0;
        if (tr.hi > tr.lo) {
          a_lo = tr.lo - k.u_lo;
          a_hi = tr.hi - k.u_lo;
          ok = p8_wait(&ctrl->q_full[t], results & 1u, abort_flag, p.status, ERR_WAIT_SMEM_FULL);
        }
        do_k(0);
#pragma unroll 1
        for (int u = 0; u < n_union && ok; ++u) {
          do_k(u + 1);
          do_v(u);
        }
        tiles += a_hi - a_lo;
        results += a_hi > a_lo;
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax, one thread per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int t = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_off = uint32_t(quad * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + kSCol + t * 128, o_addr = tmem_base + lane_off + kOCol + t * 128;
    uint8_t* my_p = p_s + t * L::kP + r * 128;
    const P8Rows<D> q_rows(q_s + t * L::kTile + quad * 32 * 128, lane);
    // a row of a work: (token, head of the group)
    struct Row {
      int tile_lo, n_tiles, lo_pos, hi_pos, head, x0;     // x0: walk position of its first tile
      int paired;                                         // tiles whose exponentials the two query tiles take turns with
      int block, part;
      long long at;                                       // row of q and out (of heads), < 0: none
      float raw_log2;                                     // raw score -> exponent of two, without 2^K
      uint32_t tiles0;                                    // tiles of the works before
    };
    Row cur{}, next{};
    bool have = false, alive = true;
    uint32_t tiles_seen = 0, done = 0, pairs = 0;         // tiles of all works; this query tile's; paired ones
    uint32_t n_works = 0;
    bool last = false;                                    // no more works
#pragma unroll 1
    while (true) {
      float m = -INFINITY, l = 0.f;
      if (have) {
        const int n_tiles = cur.n_tiles, hi_pos = cur.hi_pos, lo_pos = cur.lo_pos;
        for (int it = 0; it < n_tiles; ++it) {
          const uint32_t x = cur.tiles0 + cur.x0 + it;
          const int kv0 = (cur.tile_lo + it) * kP8Tile;
          bool ok = p8_wait(&ctrl->e_full[x % kP8Slots], x / kP8Slots & 1u, abort_flag, p.status, ERR_WAIT_SMEM_FULL);
          ok = ok && p8_wait(&ctrl->s_full[t], done + it & 1u, abort_flag, p.status, ERR_WAIT_TMEM_FULL);
          if (!__all_sync(kAll, ok)) { alive = false; break; }
          const int e_k = *(volatile int*)&ctrl->e_k[x % kP8Slots], e_v = *(volatile int*)&ctrl->e_v[x % kP8Slots];
          // not zero, for rows of zeros or next to it: masked scores are -infinity
          const float to_log2 = fmaxf(cur.raw_log2 * exp2_int(e_k - int(kP8Lift)), FLT_MIN), add = float(e_v);
          tc_fence_after();
          uint32_t v[kP8Tile];
          constexpr int kFirst = 64;                          // scores whose maximum is taken while the others come
          float mx4[4];
          auto largest = [&](int i0, int i1) {
            if (i0 == 0) {
#pragma unroll
              for (int i = 0; i < 4; ++i) mx4[i] = fmaxf(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
              i0 = 8;
            }
#pragma unroll
            for (int i = i0; i < i1; i += 2) mx4[(i >> 1) & 3] = fmax3(mx4[(i >> 1) & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          };
#pragma unroll
          for (int c = 0; c < kFirst / 32; ++c) tmem_ld_32x32(s_addr + c * 32, reinterpret_cast<uint32_t(&)[32]>(v[c * 32]));
          tmem_ld_wait();
#pragma unroll
          for (int c = kFirst / 32; c < kP8Tile / 32; ++c) tmem_ld_32x32(s_addr + c * 32, reinterpret_cast<uint32_t(&)[32]>(v[c * 32]));
          const bool edge = __any_sync(kAll, kv0 + kP8Tile - 1 > hi_pos || kv0 < lo_pos);
          if (!edge) {
            largest(0, kFirst);
            asm volatile("" : "+f"(mx4[0]), "+f"(mx4[1]), "+f"(mx4[2]), "+f"(mx4[3]));
          }
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctrl->s_empty[t]);      // the scores (and the tile's exponents) are in registers
          if (edge) {
            const int hi_rel = hi_pos - kv0, lo_rel = lo_pos - kv0;
#pragma unroll
            for (int i = 0; i < kP8Tile; ++i)
              if (i > hi_rel || i < lo_rel) v[i] = 0xff800000u;
            largest(0, kFirst);
          }
          largest(kFirst, kP8Tile);
          const float mx = fmaf(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), to_log2, add);
          bool p_free = it == 0;
          if (it == 0) {
            m = mx;
          } else {
            const bool grow = mx > m + kP8Grow;
            if (__any_sync(kAll, grow)) {
              ok = p8_wait(&ctrl->o_full[t], done + it - 1 & 1u, abort_flag, p.status, ERR_WAIT_TMEM_FULL);
              if (!__all_sync(kAll, ok)) { alive = false; break; }
              p_free = true;
              tc_fence_after();
              const float alpha = grow ? exp2f(m - mx) : 1.f;
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32(o_addr + c * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st_32x32(o_addr + c * 32, o);
              }
              tmem_st_wait();
              l *= alpha;
              if (grow) m = mx;
            }
          }
          const float less = add + kP8Lift - (m == -INFINITY ? 0.f : m);
          const float2 sc2 = make_float2(to_log2, to_log2), nb2 = make_float2(less, less);
          // The other query tile's turn comes ahead of this one's end: while its exponentials start, this one's last weights are stored and published.
          // A quarter later, us: 16 prompts of 1024 165 (157 here), 2 of 8000 786 (741); a quarter earlier 159 and 747, and 247 for 241 at 64 columns.
          constexpr int kHand = NH == 2 ? 2 : 3;
          float2 sum2[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum2[i] = make_float2(0.f, 0.f);
          if (!p_free) {
            ok = p8_wait(&ctrl->o_full[t], done + it - 1 & 1u, abort_flag, p.status, ERR_WAIT_TMEM_FULL);
            if (!__all_sync(kAll, ok)) { alive = false; break; }
          }
          // turns with the exponentials, where both query tiles have one: tile 0 (it), tile 1 (it), tile 0 (it + 1), ..., over all works
          if (it < cur.paired && (t == 1 || pairs + it > 0)) {
            ok = p8_wait(&ctrl->turn[t][quad], pairs + it - (t == 0 ? 1 : 0) & 1u, abort_flag, p.status, ERR_WAIT_SOFTMAX);
            if (!__all_sync(kAll, ok)) { alive = false; break; }
          }
#pragma unroll
          for (int c = 0; c < kP8Tile / 32; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int k = c * 32 + 2 * i;
              const float2 y = ffma2(make_float2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), sc2, nb2);
              const float2 e = make_float2(exp2f(y.x), exp2f(y.y));
              sum2[i & 3] = fadd2(sum2[i & 3], e);
              pk[i] = p8_pack_f16x2(e.x, e.y);
            }
            if (c == kHand) {
              __syncwarp();
              if (lane == 0 && it < cur.paired) mbar_arrive(&ctrl->turn[1 - t][quad]);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint4*>(my_p + (c >> 1) * kHalf + ((((c & 1) * 4 + q) ^ (r & 7)) << 4)) =
                  make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
          }
          fence_proxy_async();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctrl->p_full[t]);
          const float2 s4 = fadd2(fadd2(sum2[0], sum2[1]), fadd2(sum2[2], sum2[3]));
          l = fmaf(s4.x + s4.y, exp2_int(-e_v), l);
        }
      }
      // ---- queries of the next work, ahead of this one's result: the products of this one with Q have been read
      bool more = false;
      P8Work k;
#pragma unroll 1
      while (alive && !last && !more) {
        if (!p8_next(ctrl, n_works, k, false, p.status)) {
          last = true;
          break;
        }
        const P8Range tr = t == 0 ? k.tr0 : k.tr1;
        next.tiles0 = tiles_seen;
        tiles_seen += k.n_union;
        if (tr.rows == 0) continue;                       // (a work's second query tile may have none)
        more = true;
        const int row = k.row0 + t * kP8Tile + r, token = row / p.group;
        const long long q_row = (long long)k.q_start + token;
        next.head = k.kvh * p.group + row % p.group;
        next.at = r < tr.rows && q_row >= 0 && q_row < p.total_q ? q_row * p.nq + next.head : -1;
        next.tile_lo = tr.lo;
        next.x0 = tr.lo - k.u_lo;
        next.n_tiles = tr.hi - tr.lo;
        next.paired = k.paired();
        next.block = k.block;
        next.part = k.part;
        const int q_pos = k.ctx - k.q_len + token;
        next.hi_pos = p.causal ? min(k.ctx - 1, q_pos) : k.ctx - 1;
        next.lo_pos = nkb_first_visible(q_pos, p.window, p.chunk);
        uint4 v[D / 8];
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const long long at = __shfl_sync(kAll, next.at, i * q_rows.kRows + q_rows.row);
          v[i] = at >= 0 ? reinterpret_cast<const uint4*>(p.q + at * D)[q_rows.piece] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) *q_rows.wide(i * q_rows.kRows) = v[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < D / 8; ++i) v[i] = *q_rows.own(i);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t q4[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_bf16x2(q4[j]);
            mx = fmax3(mx, fabsf(f.x), fabsf(f.y));
          }
        }
        const int e = max((__float_as_int(mx) >> 23) - 127, -100);
        const float up = copysignf(exp2_int(14 - e), p.scale_log2);       // the largest score has the largest exponent so
        next.raw_log2 = fabsf(p.scale_log2) * exp2_int(e - 14);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t q4[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
          uint32_t h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_bf16x2(q4[j]);
            h[j] = p8_pack_f16x2(f.x * up, f.y * up);
          }
          *q_rows.own(i) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0 && next.n_tiles > 0) mbar_arrive(&ctrl->q_full[t]);
      }
      // ---- O / l
      if (have) {
        bool have_o = false;
        if (alive && cur.n_tiles > 0) {
          const bool ok = p8_wait(&ctrl->o_full[t], done + cur.n_tiles - 1 & 1u, abort_flag, p.status, ERR_WAIT_TMEM_FULL);
          have_o = __all_sync(kAll, ok);
          alive = have_o;
          if (have_o) tc_fence_after();
        }
        const bool whole = cur.part >> 8 == 1;
        // the weights are behind their last product.  The lane goes through an empty asm, since addresses that are computed ahead of the loop
        // over tiles take registers there (267 us for 251 at 64 columns).
        int lane_o = lane;
        asm volatile("" : "+r"(lane_o));
        const P8Rows<D> rows(p_s + t * L::kP + quad * 32 * 128, lane_o);
        const float inv = whole ? p8_inverse(p, cur.head, m, l) : 0.f;
        const bool store = !*abort_flag;
        constexpr long long kPart = 2 * kP8Tile * (D + 2);
        float* first = p.partials + (long long)cur.block * p.parts * kPart;
        float* mine = first + (cur.part & 255) * kPart + (t * kP8Tile + r) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (have_o) {
            tmem_ld_32x32(o_addr + c * 32, reinterpret_cast<uint32_t(&)[32]>(o));
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *rows.own(c * 4 + i) =
                  make_uint4(pack_bf16x2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf16x2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                             pack_bf16x2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_bf16x2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
          } else if (have_o) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(mine + c * 32 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (have_o) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctrl->o_empty[t]);
        }
        if (whole) {
          __syncwarp();
#pragma unroll 4
          for (int j = 0; j < 32; j += rows.kRows) {
            const long long at = __shfl_sync(kAll, cur.at, j + rows.row);
            const uint4 x = *rows.wide(j);
            if (at >= 0 && store) reinterpret_cast<uint4*>(p.out + at * D)[rows.piece] = x;
          }
          __syncwarp();
        }
        if (!whole) {
          float* tail = first + (cur.part & 255) * kPart + 2 * kP8Tile * D + t * kP8Tile + r;
          tail[0] = have_o ? m : -INFINITY;
          tail[2 * kP8Tile] = have_o ? l : 0.f;
        }
        if (p.parts > 1 && t == 0 && r == 0) p.counts[cur.block] = cur.part >> 8;
        done += cur.n_tiles;
        pairs += cur.paired;
      }
      if (!more || !alive) break;
      cur = next;
      have = true;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctrl->done);
  }

  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  if (threadIdx.x == 15 * 32) {                           // this warp has taken its last work
    __threadfence();
    if (atomicAdd(p.sched + 1, 1u) == gridDim.x - 1) {
      p.sched[0] = 0u;
      p.sched[1] = 0u;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// Puts the parts of divided blocks together: a warp per row, D / 32 columns a lane
template <int D>
__global__ void __launch_bounds__(256) attn_q8_join_kernel(const PrefillQ8Params p) {
  constexpr int N = D / 32, kAhead = 4;
  constexpr long long kPart = 2 * kP8Tile * (D + 2);
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, block = blockIdx.y, r = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int head_of = block % p.nkv, b = block / p.nkv % p.batch, row = block / (p.nkv * p.batch) * 2 * kP8Tile + r;
  const int q_len = p.q_lens[b], token = row / p.group, head = head_of * p.group + row % p.group;
  const long long q_row = (long long)p.q_start[b] + token;
  if (token >= q_len || q_row < 0 || q_row >= p.total_q) return;
  const float* first = p.partials + (long long)block * p.parts * kPart;
  // lane = part, of those that there may be until it is known
  const int parts = min(__ldcg(p.counts + block), p.parts);
  float mine = lane < p.parts ? __ldcg(first + lane * kPart + 2 * kP8Tile * D + r) : 0.f;
  float sum = lane < p.parts ? __ldcg(first + lane * kPart + 2 * kP8Tile * (D + 1) + r) : 0.f;
  if (parts == 1) return;                                 // the results are there
  if (lane >= parts) {
    mine = -INFINITY;
    sum = 0.f;
  }
  const float m = warp_max(mine), weight = mine == m ? 1.f : exp2f(mine - m);
  // (a part of small values counts in the denominator where its weight may be below the least normal number)
  const float counts = mine - m < -60.f && sum > 0.f ? exp2f(mine - m + log2f(sum)) : sum * weight;
  const uint32_t there = __ballot_sync(0xffffffffu, mine != -INFINITY || sum != 0.f);      // the others had no tile, or saw nothing
  const float inv = p8_inverse(p, head, m, warp_sum(counts));
  float o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  for (int s0 = 0; s0 < parts; s0 += kAhead) {
    float x[kAhead][N];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[s][i] = there >> (s0 + s) & 1 ? __ldcg(first + (s0 + s) * kPart + r * D + i * 32 + lane) : 0.f;
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const float w = __shfl_sync(0xffffffffu, weight, s0 + s);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = there >> (s0 + s) & 1 ? fmaf(w, x[s][i], o[i]) : o[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) p.out[(q_row * p.nq + head) * D + i * 32 + lane] = __float2bfloat16(o[i] * inv);
}

template <int D>
static int launch_prefill_q8(const PrefillQ8Params& p, cudaStream_t s) {
  using L = PrefillQ8Smem<D>;
  static bool attr_set[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!attr_set[dev]) {
    // the register split would wait for registers that a smaller launch does not have
    cudaFuncAttributes a;
    if (cudaError_t e = cudaFuncGetAttributes(&a, attn_q8_prefill_kernel<D>)) return int(e);
    if (a.numRegs != kP8Regs) return -3;
    if (cudaError_t e = cudaFuncSetAttribute(attn_q8_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes)) return int(e);
    attr_set[dev] = true;
  }
  const long long works = (long long)p.q_blocks * p.nkv * p.batch * p.parts;
  if (int rc = launch_pdl(attn_q8_prefill_kernel<D>, dim3(unsigned(works < num_sms() ? works : num_sms())), dim3(kP8Threads), size_t(L::kBytes), s, p))
    return rc;
  return p.parts == 1 ? 0 : launch_pdl(attn_q8_join_kernel<D>, dim3(2 * kP8Tile / 8, unsigned(works / p.parts)), dim3(256), 0, s, p);
}

}  // namespace nkb

using namespace nkb;

// How many works a block's tiles are divided into at most: where there are no more blocks than half the SMs, and four tiles that they may see
static int p8_parts(long long blocks, int table_width) {
  const long long fit = blocks > 0 ? num_sms() / blocks : 1, tiles = (table_width + 3) / 4;
  const long long parts = fit < tiles ? fit : tiles;
  return int(parts < 2 || tiles < kP8Least ? 1 : (parts > 16 ? 16 : parts));
}
static long long p8_blocks(int batch, int max_q_len, int nq, int nkv) {
  return ((long long)max_q_len * (nq / nkv) + 2 * kP8Tile - 1) / (2 * kP8Tile) * nkv * batch;
}

static long long p8_again_ints(long long works) { return (works + 3) / 4 * 4; }

// Negative: there is no device.
extern "C" long long nkb_q8_attn_prefill_scratch_floats(int batch, int max_q_len, int nq, int nkv, int head_dim, int table_width) {
  if (batch <= 0 || nkv < 1 || nq < nkv || max_q_len < 1 || (!status_word() && nkb_init() != 0)) return -1;
  const long long blocks = p8_blocks(batch, max_q_len, nq, nkv);
  const int parts = p8_parts(blocks, table_width);
  return kQ8Counters + p8_again_ints(blocks * parts) + (parts > 1 ? kP8Counts + blocks * parts * 2 * kP8Tile * (head_dim + 2) : 0);
}
// 2 where parts of blocks are joined, else 1
extern "C" int nkb_q8_attn_prefill_launches(int batch, int max_q_len, int nq, int nkv, int table_width) {
  if (batch <= 0 || nkv < 1 || nq < nkv || max_q_len < 1 || (!status_word() && nkb_init() != 0)) return -1;
  return p8_parts(p8_blocks(batch, max_q_len, nq, nkv), table_width) > 1 ? 2 : 1;
}

extern "C" int nkb_q8_attn_prefill(const NkbQ8Attn* arg) {
  const NkbQ8Attn& g = *arg;
  if (g.batch <= 0 || g.total_q <= 0) return 0;
  if (g.batch > 65535 || g.nkv > 65535 || g.nkv < 1 || g.nq < g.nkv || g.nq % g.nkv || g.q_len < 1) return -2;
  if (!status_word() && nkb_init() != 0) return -1;
  PrefillQ8Params p{};
  p.q = (const __nv_bfloat16*)g.q;
  p.k_values = (const uint8_t*)g.k_values; p.k_scales = (const uint8_t*)g.k_scales;
  p.v_values = (const uint8_t*)g.v_values; p.v_scales = (const uint8_t*)g.v_scales;
  p.block_table = g.block_table; p.q_start = g.q_start; p.q_lens = g.q_lens; p.context_lens = g.context_lens;
  p.out = (__nv_bfloat16*)g.out;
  p.sinks = g.sinks;
  p.status = status_word();
  const long long blocks = p8_blocks(g.batch, g.q_len, g.nq, g.nkv);
  p.parts = p8_parts(blocks, g.table_width);
  if (!g.scratch || blocks * p.parts > 0x3fffffffll) return -2;
  if (g.scratch_floats < nkb_q8_attn_prefill_scratch_floats(g.batch, g.q_len, g.nq, g.nkv, g.head_dim, g.table_width)) return -2;
  p.sched = reinterpret_cast<unsigned int*>(g.scratch);
  p.again = reinterpret_cast<int*>(g.scratch + kQ8Counters);
  p.counts = p.again + p8_again_ints(blocks * p.parts);
  p.partials = reinterpret_cast<float*>(p.counts + kP8Counts);
  p.batch = g.batch; p.q_blocks = int(blocks / ((long long)g.nkv * g.batch));
  p.total_q = g.total_q; p.nq = g.nq; p.nkv = g.nkv; p.group = g.nq / g.nkv; p.num_blocks = g.num_blocks; p.table_width = g.table_width;
  p.causal = g.causal; p.window = g.window; p.chunk = g.chunk;
  p.table_stride = g.table_stride;
  p.scale_log2 = g.scale * 1.4426950408889634f;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(g.stream);
  if (g.head_dim == 128) return launch_prefill_q8<128>(p, s);
  if (g.head_dim == 64) return launch_prefill_q8<64>(p, s);
  return -2;
}
