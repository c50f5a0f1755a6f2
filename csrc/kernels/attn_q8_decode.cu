// Decode attention over 8-bit pages (kv_quant.cuh): the new tokens of every sequence, up to sixteen query rows per kv head.
//
//   o = sum_j 2^{s_j + v_j} v8_j / sum_j 2^{s_j},    s_j = (scale / ln 2) 2^{k_j} (q . k8_j)
//
// with 2^{k_j} and 2^{v_j} the powers of two that token j's key and value are kept with.  The sums run over t_j = s_j + v_j: weights
// 2^{t_j - M}, M near the largest t so far, multiply the values as they are kept, and 2^{-v_j} takes a weight back to the denominator.  So
// values of any size meet weights that f16 holds: a weight below 2^-30 of the largest contribution is all that rounds to nothing.  In the
// denominator a token counts by its score alone: where v_j is so small that 2^{t_j - M} may be below the least normal number while the
// token still counts (a row of zeros beside values of 2^40 or more), it gets an exponential of its own, and factors of the denominator go
// on in two steps.
//
// The op is bound by the bytes of the pages, half of a bf16 cache's, and next by what a warp does per page.  Four bytes are two
// conversions to f16 (exact; e4m3 has no matrix instruction with 16-bit queries).  Keys and columns of values are the 16-row side of the
// products, query rows the side of eight: S^T = K Q^T, O^T = V^T P^T, so that a group of up to eight rows costs half the products and a
// lane half the exponentials that rows padded to sixteen would.  Queries are f16 too, each row brought below 2^15 by a power of two, which
// loses nothing that 32-bit sums would keep.  Fragments come from shared memory with ldmatrix in units of two bytes: a lane then holds
// four neighbouring columns of a key, which the queries are permuted to match, and of a value pairs of neighbouring columns, which a byte
// permutation turns into pairs of tokens.
//
// The grid, the page plan and the merge are those of decode attention over bf16 pages (attn_decode.cu); a page is half as large, so
// an SM holds the rings of twice as many warps.
//
// Measured, beside the bytes at the copy bandwidth (6.56 TB/s) and bf16 pages: 32 heads of 128 on 8, 64 sequences of 1024 24.8 us (21.0, 46.0), 7 of
// 3500 to 7000 23.4 (15.6, 36.7; its CTAs' ends and the merge), one of 203 4.2 (latency); 64 heads of 64 on 8 with two new tokens, 37 of 1000 to
// 2000 18.7 (9.1, 27.4): sixteen rows, half the bytes per conversion, and issue slots at half use.
#include "api.h"
#include "kv_quant.cuh"
#include "mma_frag.cuh"
#include "page_plan.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace nkb {

constexpr int kQ8Stages = 3;
// warps whose rings an SM holds
template <int D>
constexpr int kQ8SmWarps = 1024 / D;
constexpr float kQ8Lift = 6.f;         // log2 of the weight at M; t may grow by kQ8Grow above M before M follows: f16 ends at 2^16
constexpr int kQ8Tiny = -40;            // log2 of a value's scale: 2^-126 (f32) 2^40 is 2^-28 of the least that a token at M adds
constexpr float kQ8Grow = 8.f;

struct DecodeQ8Params {
  const __nv_bfloat16* q;              // may be out: all warps have read their queries before a result of their sequence and kv head is written
  const int *block_table, *context_lens;
  __nv_bfloat16* out;
  float* scratch;
  unsigned int* counters;
  const float* sinks;
  const float* qkv_partials;           // null: the newest tokens are in the pages
  int* status;
  int batch, q_len, nq, nkv, group, table_width, window, chunk;
  int units;
  // The kernel before writes queries and the newest token's page (at position context - 1) and nothing else that is read here: the other pages
  // are fetched without waiting for it.  Append and attention, us: 64 sequences of 1024 29.2 -> 28.2, 7 of 3500 to 7000 27.5 -> 24.9, 128 of 512
  // on 4 heads 21.1 -> 19.1, one of 203 7.1 -> 6.4.
  int early;
  long long table_stride;
  float scale_log2;
  __device__ __forceinline__ int context(int b) const { return min(context_lens[b], table_width * kPage); }
};

__device__ __forceinline__ void mma_16816_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// the transpose of an 8 x 8 matrix of 16-bit values that the warp holds
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(v));
  return v;
}

// Byte of a 16-byte piece in a [32][D] page, as the load's swizzle places it: 128-byte rows piece ^ row, 64-byte rows piece ^ row / 2
template <int D>
__device__ __forceinline__ uint32_t q8_piece(int row, int piece) {
  return D == 128 ? row * 128 + ((piece ^ (row & 7)) << 4) : row * 64 + ((piece ^ ((row >> 1) & 3)) << 4);
}

template <int D, int W>
struct DecodeQ8Smem {
  static constexpr int kMat = kPage * D, kStage = 2 * kMat, kScales = 256;       // K and V scales, on 128 bytes each
  static constexpr int kRings = W * kQ8Stages * kStage, kScaleAt = kRings;
  static constexpr int kBytes = kScaleAt + W * kQ8Stages * kScales + 1024;
  static constexpr int kPitch = D + 8;                                           // floats between the rows of merged results
  static_assert(kRings >= W * (16 * kPitch + 32) * 4, "merge space must fit in the rings");
};

// NT: query rows of a kv head in eights
template <int D, int W, int NT>
__global__ void __launch_bounds__(W * 32, kQ8SmWarps<D> / W)
attn_q8_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ CUtensorMap tmKS, const __grid_constant__ CUtensorMap tmVS, const DecodeQ8Params p) {
  using L = DecodeQ8Smem<D, W>;
  constexpr uint32_t kAll = 0xffffffffu;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[W][kQ8Stages];
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, rows = p.q_len * p.group;
  if (threadIdx.x == 0) {
    for (int w = 0; w < W; ++w)
      for (int s = 0; s < kQ8Stages; ++s) mbar_init(&bars[w][s], 1);
    abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmKS);
    tma_prefetch_desc(&tmVS);
  }
  __syncthreads();
  if (!p.early) {
    griddep_wait();
    griddep_launch();
  }
  PagePlan plan{int(blockIdx.z), 0, 1, 0x3fffffff};
  if (p.units && !plan_pages<false>(p, blockIdx.x, 2 * W, lane, plan)) return;     // (a grid waits for the one before until its last CTA ends)
  const int b = plan.b, split = plan.split;
  // what does not depend on the context's length is on its way beside it
  uint2 q_raw[NT][D / 16];
  auto load_q = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const __nv_bfloat16* src = p.q + (((long long)b * p.q_len + r / p.group) * p.nq + kvh * p.group + r % p.group) * D + 4 * t;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) q_raw[nt][ks] = r < rows ? *reinterpret_cast<const uint2*>(src + 16 * ks) : make_uint2(0u, 0u);
    }
  };
  const int* table = p.block_table + b * p.table_stride;
  const bool from_start = !p.units && p.window == 0 && p.chunk == 0;     // this CTA's pages begin with the first
  int blks[kQ8Stages];
  if (from_start) {
#pragma unroll
    for (int s = 0; s < kQ8Stages; ++s) blks[s] = table[min(warp + s * W, p.table_width - 1)];
  }
  if (!p.early) load_q();
  const int ctx = p.context(b);
  int page_lo, kept;
  const int npages = pages_of<false>(p, ctx, page_lo, kept);
  const int p0 = page_lo + split * (plan.splits > 1 ? plan.per : 0), p1 = min(page_lo + npages, p0 + plan.per);

  uint8_t* my_ring = smem + warp * kQ8Stages * L::kStage;
  uint8_t* my_scales = smem + L::kScaleAt + warp * kQ8Stages * L::kScales;
  const uint64_t policy = l2_evict_first();
  // A block outside the pool lies outside the tensor maps, which read zeros there.
  auto issue = [&](int blk, int stage) {
    if (lane == 0) {
      uint8_t* dst = my_ring + stage * L::kStage;
      uint64_t* bar = &bars[warp][stage];
      mbar_expect_tx(bar, L::kStage + 2 * kPage);
      tma_load_4d_as(dst, &tmK, bar, 0, 0, kvh, blk, policy);
      tma_load_4d_as(dst + L::kMat, &tmV, bar, 0, 0, kvh, blk, policy);
      tma_load_3d_as(my_scales + stage * L::kScales, &tmKS, bar, 0, kvh, blk, policy);
      tma_load_3d_as(my_scales + stage * L::kScales + 128, &tmVS, bar, 0, kvh, blk, policy);
    }
  };
  if (!from_start) {
#pragma unroll
    for (int s = 0; s < kQ8Stages; ++s) blks[s] = p0 + warp + s * W < p1 ? table[p0 + warp + s * W] : 0;
  }
  const int late = p.early ? (ctx - 1) / kPage : -1;      // the page that has to wait
#pragma unroll
  for (int s = 0; s < kQ8Stages; ++s)
    if (p0 + warp + s * W < p1 && p0 + warp + s * W != late) issue(blks[s], s);
  if (p.early) {
    griddep_wait();
    griddep_launch();
#pragma unroll
    for (int s = 0; s < kQ8Stages; ++s)
      if (p0 + warp + s * W < p1 && p0 + warp + s * W == late) issue(blks[s], s);
    load_q();
  }

  // ---- query fragments (the first pages are on their way): lane (g, t) has columns 16 ks + 4 t ... of row g, as the keys come.
  // rs: raw score -> exponent of two, without the key's factor, of rows 2 t and 2 t + 1
  uint32_t qf[NT][D / 16][2];
  float rs[NT][2];
  int pos[NT][2], low[NT][2];            // last and first visible position
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint2(&v)[D / 16] = q_raw[nt];
    float mx = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const float2 x = unpack_bf16x2(v[ks].x), y = unpack_bf16x2(v[ks].y);
      mx = fmaxf(fmaxf(fmaxf(mx, fabsf(x.x)), fmaxf(fabsf(x.y), fabsf(y.x))), fabsf(y.y));
    }
    mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 2));
    const int e = max((__float_as_int(mx) >> 23) - 127, -100);
    const float up = exp2_int(14 - e), down = p.scale_log2 * exp2_int(e - 14);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const float2 x = unpack_bf16x2(v[ks].x), y = unpack_bf16x2(v[ks].y);
      qf[nt][ks][0] = pack_f16x2(x.x * up, x.y * up);
      qf[nt][ks][1] = pack_f16x2(y.x * up, y.y * up);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      rs[nt][i] = __shfl_sync(kAll, down, (2 * t + i) * 4);
      const int row = nt * 8 + 2 * t + i;
      pos[nt][i] = ctx - p.q_len + (row < rows ? row / p.group : 0);
      low[nt][i] = nkb_first_visible(pos[nt][i], p.window, p.chunk);
    }
  }
  const int all_hi = ctx - p.q_len, all_lo = nkb_first_visible(ctx - 1, p.window, p.chunk);      // what every row sees
  const int any_lo = nkb_first_visible(ctx - p.q_len, p.window, p.chunk);                        // and what one does, up to ctx

  // lane (g, t): rows 2 t, 2 t + 1 of columns 16 c + 2 g, 16 c + 2 g + 1
  float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[nt][c][0] = o[nt][c][1] = o[nt][c][2] = o[nt][c][3] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }

  int stage = 0;
  uint32_t phase = 0;
  for (int pg = p0 + warp; pg < p1; pg += W) {
    const int next = pg + kQ8Stages * W;
    const int next_blk = next < p1 ? table[next] : 0;
    const bool ok = mbar_wait(&bars[warp][stage], phase, &abort_flag, p.status, ERR_WAIT_SMEM_FULL);
    if (!__all_sync(kAll, ok)) break;
    const uint32_t kbase = smem_u32(my_ring + stage * L::kStage), vbase = kbase + L::kMat;
    // lane = token: its factors, for the lanes that hold its scores
    const int kb = my_scales[stage * L::kScales + lane], vb = my_scales[stage * L::kScales + 128 + lane];
    const int v_log2 = q8_log2_of(vb);
    const float my_kf = q8_factor_of(kb), my_ve = vb == 255 ? __int_as_float(0x7fc00000) : float(v_log2), my_back = exp2_int(-v_log2);

    // fragments of the page ahead of their use, a wait for shared memory each otherwise
    uint32_t kr[D / 32][2][4], vr[2][D / 32][4];         // pieces 2 c and 2 c + 1 of tokens 0 to 7 and 8 to 15 of each sixteen
#pragma unroll
    for (int c2 = 0; c2 < D / 32; ++c2) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
        ldsm_x4(kbase + q8_piece<D>(mt * 16 + (lane & 15), 2 * c2 + (lane >> 4)), kr[c2][mt][0], kr[c2][mt][1], kr[c2][mt][2], kr[c2][mt][3]);
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int c2 = 0; c2 < D / 32; ++c2)
        ldsm_x4_t(vbase + q8_piece<D>(mt * 16 + (lane & 15), 2 * c2 + (lane >> 4)), vr[mt][c2][0], vr[mt][c2][1], vr[mt][c2][2], vr[mt][c2][3]);
    }
    // S^T: keys 16 mt + g and + 8, rows 2 t and 2 t + 1
    float s[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
    }
#pragma unroll
    for (int c2 = 0; c2 < D / 32; ++c2) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const uint32_t(&r)[4] = kr[c2][mt];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a[4] = {e4m3x2_to_f16x2(uint16_t(r[2 * i])), e4m3x2_to_f16x2(uint16_t(r[2 * i + 1])),
                                 e4m3x2_to_f16x2(uint16_t(r[2 * i] >> 16)), e4m3x2_to_f16x2(uint16_t(r[2 * i + 1] >> 16))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816_f16(s[mt][nt], a, qf[nt][2 * c2 + i][0], qf[nt][2 * c2 + i][1]);
        }
      }
    }
    // t = s + v, the mask only where a page crosses an edge
    const int tok0 = pg * kPage;
    const bool edge = tok0 + kPage - 1 > all_hi || tok0 < all_lo;
    float mx[NT][2], back[2][2];
    bool grow = false;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = mt * 16 + h * 8 + g;
        const float kf = __shfl_sync(kAll, my_kf, key), ve = __shfl_sync(kAll, my_ve, key);
        back[mt][h] = __shfl_sync(kAll, my_back, key);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            s[mt][nt][2 * h + i] = fmaf(s[mt][nt][2 * h + i] * rs[nt][i], kf, ve);
          }
        }
      }
    }
    if (edge) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = tok0 + mt * 16 + (e >> 1) * 8 + g;
            if (tok > pos[nt][e & 1] || tok < low[nt][e & 1]) s[mt][nt][e] = -INFINITY;
          }
        }
      }
      // what no row sees may be anything: a lane's values are of tokens 2 t and 2 t + 1 of each eight
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int tok = tok0 + mt * 16 + h * 8 + 2 * t;
          const uint32_t keep = (tok >= any_lo && tok < ctx ? 0xffffu : 0u) | (tok + 1 >= any_lo && tok + 1 < ctx ? 0xffff0000u : 0u);
#pragma unroll
          for (int c2 = 0; c2 < D / 32; ++c2) {
            vr[mt][c2][h] &= keep;
            vr[mt][c2][2 + h] &= keep;
          }
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) mx[nt][i] = fmaxf(fmax3(s[0][nt][i], s[0][nt][2 + i], s[1][nt][i]), s[1][nt][2 + i]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) grow = grow || mx[nt][0] > m[nt][0] + kQ8Grow || mx[nt][1] > m[nt][1] + kQ8Grow;
    // M follows the largest t when that has grown by more than kQ8Grow
    if (__any_sync(kAll, grow || v_log2 < kQ8Tiny)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float keep[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = mx[nt][i];
          x = fmaxf(x, __shfl_xor_sync(kAll, x, 4));
          x = fmaxf(x, __shfl_xor_sync(kAll, x, 8));
          x = fmaxf(fmaxf(x, __shfl_xor_sync(kAll, x, 16)), m[nt][i]);
          const float root = m[nt][i] == x ? 1.f : exp2f(0.5f * (m[nt][i] - x));
          keep[i] = root * root;
          m[nt][i] = x;
          l[nt][i] = l[nt][i] * root * root;
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          o[nt][c][0] *= keep[0]; o[nt][c][1] *= keep[1];
          o[nt][c][2] *= keep[0]; o[nt][c][3] *= keep[1];
        }
      }
      if (__any_sync(kAll, v_log2 < kQ8Tiny)) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ve = __shfl_sync(kAll, v_log2, mt * 16 + h * 8 + g);
            if (ve >= kQ8Tiny) continue;
            back[mt][h] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int i = 0; i < 2; ++i) l[nt][i] += exp2f(s[mt][nt][2 * h + i] - (m[nt][i] == -INFINITY ? 0.f : m[nt][i]) + (kQ8Lift - float(ve)));
            }
          }
        }
      }
    }
    uint32_t pb[2][NT][2];               // P^T: row g, tokens 2 t and 2 t + 1 of each eight
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float base0 = (m[nt][0] == -INFINITY ? 0.f : m[nt][0]) - kQ8Lift, base1 = (m[nt][1] == -INFINITY ? 0.f : m[nt][1]) - kQ8Lift;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w0 = exp2f(s[mt][nt][2 * h] - base0), w1 = exp2f(s[mt][nt][2 * h + 1] - base1);
          l[nt][0] = fmaf(w0, back[mt][h], l[nt][0]);
          l[nt][1] = fmaf(w1, back[mt][h], l[nt][1]);
          pb[mt][nt][h] = transposed_8x8(pack_f16x2(w0, w1));
        }
      }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int c2 = 0; c2 < D / 32; ++c2) {
        const uint32_t(&r)[4] = vr[mt][c2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t lo = __byte_perm(r[2 * i], 0u, 0x3120), hi = __byte_perm(r[2 * i + 1], 0u, 0x3120);   // pairs of tokens
          const uint32_t a[4] = {e4m3x2_to_f16x2(uint16_t(lo)), e4m3x2_to_f16x2(uint16_t(lo >> 16)),
                                 e4m3x2_to_f16x2(uint16_t(hi)), e4m3x2_to_f16x2(uint16_t(hi >> 16))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816_f16(o[nt][2 * c2 + i], a, pb[mt][nt][0], pb[mt][nt][1]);
        }
      }
    }
    __syncwarp();
    if (next < p1) issue(next_blk, stage);
    if (++stage == kQ8Stages) { stage = 0; phase ^= 1u; }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[nt][i] += __shfl_xor_sync(kAll, l[nt][i], x);
    }
  }

  if (abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  __syncthreads();  // every load consumed: the rings are merge space now

  float* mo = reinterpret_cast<float*>(smem);             // [warp][16][pitch]
  float* mm = mo + W * 16 * L::kPitch;                    // [warp][16]
  float* ml = mm + W * 16;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = nt * 8 + 2 * t + i;
      if (row < rows) {
        float* dst = mo + (warp * 16 + row) * L::kPitch + 2 * g;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) *reinterpret_cast<float2*>(dst + 16 * c) = make_float2(o[nt][c][i], o[nt][c][2 + i]);
      }
      if (g == 0) {
        mm[warp * 16 + row] = m[nt][i];
        ml[warp * 16 + row] = l[nt][i];
      }
    }
  }
  __syncthreads();
  // o and l carry 2^(lift - M); merged values 2^(lift - mf)
  auto finish = [&](int r, int d, float mf, float l, float4 acc) {
    const int head = kvh * p.group + r % p.group;
    if (p.sinks) {
      const float sk = p.sinks[head] * 1.4426950408889634f, m2 = fmaxf(mf, sk), sc = mf == -INFINITY ? 0.f : exp2f(mf - m2);
      const float add = sk == -INFINITY ? 0.f : exp2f(sk - m2 + kQ8Lift);
      acc.x *= sc; acc.y *= sc; acc.z *= sc; acc.w *= sc;
      l = l * sc + add;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint2 v;
    v.x = pack_bf16x2(acc.x * inv, acc.y * inv);
    v.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(p.out + (((long long)b * p.q_len + r / p.group) * p.nq + head) * D + d) = v;
  };
  float* part = plan.splits > 1 ? p.scratch + ((long long)kvh * p.units + blockIdx.x) * (16 * D + 32) : nullptr;
  for (int idx = threadIdx.x; idx < rows * (D / 4); idx += W * 32) {
    const int r = idx / (D / 4), d = idx % (D / 4) * 4;
    float mf = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) mf = fmaxf(mf, mm[w * 16 + r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = mm[w * 16 + r], root = mw == -INFINITY && mf != -INFINITY ? 0.f : exp2f(mw == mf ? 0.f : 0.5f * (mw - mf)), sc = root * root;
      const float4 x = *reinterpret_cast<const float4*>(mo + (w * 16 + r) * L::kPitch + d);
      acc.x += sc * x.x; acc.y += sc * x.y; acc.z += sc * x.z; acc.w += sc * x.w;
      l += root * ml[w * 16 + r] * root;
    }
    if (plan.splits == 1) {
      finish(r, d, mf, l, acc);
    } else {
      *reinterpret_cast<float4*>(part + r * D + d) = acc;
      if (d == 0) {
        part[16 * D + r] = mf;
        part[16 * D + 16 + r] = l;
      }
    }
  }
  if (plan.splits == 1) return;

  // ---- merge by the CTA that arrives last at this (sequence, kv head)'s counter
  __shared__ int is_last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned int* ctr = p.counters + (long long)b * p.nkv + kvh;
    const int last = atomicAdd(ctr, 1u) == unsigned(plan.splits - 1);
    if (last) *ctr = 0u;                 // ready for the next call (the next kernel starts after this grid)
    is_last = last;
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  const float* base = p.scratch + ((long long)kvh * p.units + blockIdx.x - split) * (16 * D + 32);
  constexpr int kAhead = 8;              // partials on their way together: the merge is a chain of latencies
  for (int idx = threadIdx.x; idx < rows * (D / 4); idx += W * 32) {
    const int r = idx / (D / 4), d = idx % (D / 4) * 4;
    float mf = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < plan.splits; s0 += kAhead) {
      float ms[kAhead], ls[kAhead];
      float4 x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float* ps = base + (long long)min(s0 + i, plan.splits - 1) * (16 * D + 32);
        ms[i] = __ldcg(ps + 16 * D + r);
        ls[i] = __ldcg(ps + 16 * D + 16 + r);
        x[i] = __ldcg(reinterpret_cast<const float4*>(ps + r * D + d));
      }
      float mn = mf;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) mn = fmaxf(mn, ms[i]);
      const float kept = mf == mn ? 1.f : exp2f(0.5f * (mf - mn)), keep = kept * kept;
      acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
      l = l * kept * kept;
      mf = mn;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (s0 + i >= plan.splits) break;
        const float root = ms[i] == mn ? 1.f : exp2f(0.5f * (ms[i] - mn)), sc = root * root;
        acc.x += sc * x[i].x; acc.y += sc * x[i].y; acc.z += sc * x[i].z; acc.w += sc * x[i].w;
        l += root * ls[i] * root;
      }
    }
    finish(r, d, mf, l, acc);
  }
}

template <int D, int W, int NT>
static int launch_decode_q8(const CUtensorMap (&m)[4], const DecodeQ8Params& p, cudaStream_t s) {
  using L = DecodeQ8Smem<D, W>;
  static bool attr_set[64] = {false};    // the attribute is per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_q8_decode_kernel<D, W, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (e != cudaSuccess) return int(e);
    attr_set[dev] = true;
  }
  const dim3 grid = p.units ? dim3(p.units, p.nkv, 1) : dim3(1, p.nkv, p.batch);
  return launch_pdl(attn_q8_decode_kernel<D, W, NT>, grid, dim3(W * 32), size_t(L::kBytes), s, m[0], m[1], m[2], m[3], p);
}

template <int D, int NT>
static int dispatch_decode_q8(const CUtensorMap (&m)[4], const DecodeQ8Params& p, cudaStream_t s) {
  constexpr int most = kQ8SmWarps<D>;
  const long long ctas = (long long)(p.units ? p.units : p.batch) * p.nkv, sms = num_sms();
  if (ctas <= sms) return launch_decode_q8<D, most, NT>(m, p, s);
  if (ctas <= 2 * sms) return launch_decode_q8<D, most / 2, NT>(m, p, s);
  if (ctas <= 4 * sms) return launch_decode_q8<D, most / 4, NT>(m, p, s);
  return launch_decode_q8<D, most / 8, NT>(m, p, s);
}

// Tensor maps of K and V pages and of their scales
static int q8_maps(CUtensorMap (&m)[4], const void* const (&at)[4], int dim, int nkv, int num_blocks) {
  const uint64_t dims[4] = {uint64_t(dim), uint64_t(kPage), uint64_t(nkv), uint64_t(num_blocks)};
  const uint64_t strides[3] = {uint64_t(dim), uint64_t(dim) * kPage, uint64_t(dim) * kPage * nkv};
  const uint32_t box[4] = {uint32_t(dim), uint32_t(kPage), 1, 1};
  const uint64_t sdims[3] = {uint64_t(kPage), uint64_t(nkv), uint64_t(num_blocks)};
  const uint64_t sstrides[2] = {uint64_t(kPage), uint64_t(kPage) * nkv};
  const uint32_t sbox[3] = {uint32_t(kPage), 1, 1};
  for (int i = 0; i < 2; ++i)
    if (encode_tmap_u8(&m[i], at[i], 4, dims, strides, box, dim) || encode_tmap_u8(&m[2 + i], at[2 + i], 3, sdims, sstrides, sbox, 0)) return -4;
  return 0;
}

}  // namespace nkb

using namespace nkb;

// Needs the device (the plan rounds up to waves of its SMs); negative: there is none.
extern "C" long long nkb_q8_attn_decode_scratch_floats(int batch, int nkv, int head_dim, int group, int num_splits) {
  if (num_splits <= 1) return 0;
  if (batch < 1 || nkv < 1 || group < 1 || (!status_word() && nkb_init() != 0)) return -1;
  return kQ8Counters + (long long)plan_units(batch, nkv, group, num_splits) * nkv * (16 * head_dim + 32);
}

static int attn_q8_decode(const NkbQ8Attn& g, int early) {
  if (g.batch <= 0) return 0;
  const int group = g.nkv > 0 ? g.nq / g.nkv : 0;
  if (group < 1 || g.nq % g.nkv || g.q_len < 1 || (long long)g.q_len * group > 16 || g.nkv > 65535 || g.batch > 65535) return -2;
  if (g.num_splits > 1 && (!g.scratch || (long long)g.batch * g.nkv > kQ8Counters)) return -2;
  if (!status_word() && nkb_init() != 0) return -1;
  if (g.num_splits > 1 && g.scratch_floats < nkb_q8_attn_decode_scratch_floats(g.batch, g.nkv, g.head_dim, group, g.num_splits)) return -2;
  DecodeQ8Params p{};
  p.q = (const __nv_bfloat16*)g.q;
  p.block_table = g.block_table; p.context_lens = g.context_lens;
  p.out = (__nv_bfloat16*)g.out;
  p.scratch = g.num_splits > 1 ? g.scratch + kQ8Counters : nullptr;
  p.counters = reinterpret_cast<unsigned int*>(g.scratch);
  p.sinks = g.sinks;
  p.status = status_word();
  p.batch = g.batch; p.q_len = g.q_len; p.nq = g.nq; p.nkv = g.nkv; p.group = group; p.table_width = g.table_width;
  p.window = g.window; p.chunk = g.chunk; p.early = early;
  p.units = plan_units(g.batch, g.nkv, group, g.num_splits);
  p.table_stride = g.table_stride;
  p.scale_log2 = g.scale * 1.4426950408889634f;
  CUtensorMap m[4];
  if (int rc = q8_maps(m, {g.k_values, g.v_values, g.k_scales, g.v_scales}, g.head_dim, g.nkv, g.num_blocks)) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(g.stream);
  const bool eight = g.q_len * group <= 8;
  if (g.head_dim == 128) return eight ? dispatch_decode_q8<128, 1>(m, p, s) : dispatch_decode_q8<128, 2>(m, p, s);
  if (g.head_dim == 64) return eight ? dispatch_decode_q8<64, 1>(m, p, s) : dispatch_decode_q8<64, 2>(m, p, s);
  return -2;
}

// At most 16 query rows per kv head (q_len * nq / nkv).  num_splits > 1: parts of a sequence on average, with scratch.
extern "C" int nkb_q8_attn_decode(const NkbQ8Attn* arg) { return attn_q8_decode(*arg, 0); }

// One new token per sequence: append, and behind it attention of its queries, which fetches all pages but the new token's while the append
// runs.  append.slots[b] is the place of position context_lens[b] - 1, or negative.
extern "C" int nkb_q8_step(const NkbQ8Append* append, const NkbQ8Attn* attn) {
  if (attn->nkv < 1 || attn->nq % attn->nkv || attn->nq / attn->nkv > 16 || attn->q_len != 1 || append->tokens != attn->batch) return -2;
  if (int rc = nkb_q8_append(append)) return rc;
  return attn_q8_decode(*attn, pdl_enabled() ? 1 : 0);
}
