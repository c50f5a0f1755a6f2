// Decode attention over 8-bit pages (kv_quant.cuh): the new tokens of every sequence, up to sixteen query rows per kv head.
//
//   o = sum_j 2^{s_j + v_j} v8_j / sum_j 2^{s_j},    s_j = (scale / ln 2) 2^{k_j} (q . k8_j)
//
// with 2^{k_j} and 2^{v_j} the powers of two that token j's key and value are kept with.  The sums run over t_j = s_j + v_j: weights
// 2^{t_j - M}, M near the largest t so far, multiply the values as they are kept, and 2^{-v_j} takes a weight back to the denominator.  So
// values of any size meet weights that f16 holds: a weight below 2^-30 of the largest contribution is all that rounds to nothing.
//
// The op is bound by the bytes of the pages, half of a bf16 cache's, and next by the instructions per byte: four bytes are two
// conversions to f16 (exact; e4m3 has no matrix instruction with 16-bit queries) and one (V: two) bytes permutation.  Queries are f16 too, each
// row brought below 2^15 by a power of two, which loses nothing that 32-bit sums would keep.  Fragments come from shared memory with
// ldmatrix in units of two bytes: a lane then holds four neighbouring columns of a key, which the queries are permuted to match, and of a
// value pairs of neighbouring columns, which a byte permutation turns into pairs of tokens.
//
// The grid, the page plan and the merge are those of decode attention over bf16 pages (attn_decode.cu); a page is half as large, so
// an SM holds the rings of eight warps.
#include "api.h"
#include "kv_quant.cuh"
#include "mma_frag.cuh"
#include "page_plan.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace nkb {

constexpr int kQ8Stages = 3;
constexpr int kQ8SmWarps = 8;          // warps whose rings an SM holds
constexpr int kQ8Counters = 16384;     // the scratch starts with as many arrival counters
constexpr float kQ8Lift = 6.f;         // log2 of the weight at M; t may grow by kQ8Grow above M before M follows: f16 ends at 2^16
constexpr float kQ8Grow = 8.f;

struct DecodeQ8Params {
  const __nv_bfloat16* q;
  const int *block_table, *context_lens;
  __nv_bfloat16* out;
  float* scratch;
  unsigned int* counters;
  const float* sinks;
  const float* qkv_partials;           // null: the newest tokens are in the pages
  int* status;
  int batch, q_len, nq, nkv, group, table_width, window, chunk;
  int units;
  long long table_stride;
  float scale_log2;
  __device__ __forceinline__ int context(int b) const { return min(context_lens[b], table_width * kPage); }
};

__device__ __forceinline__ void mma_16816_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Byte of a 16-byte piece in a [32][D] page, as the load's swizzle places it: 128-byte rows piece ^ row, 64-byte rows piece ^ row / 2
template <int D>
__device__ __forceinline__ uint32_t q8_piece(int row, int piece) {
  return D == 128 ? row * 128 + ((piece ^ (row & 7)) << 4) : row * 64 + ((piece ^ ((row >> 1) & 3)) << 4);
}

template <int D, int W>
struct DecodeQ8Smem {
  static constexpr int kMat = kPage * D, kStage = 2 * kMat, kScales = 256;       // K and V scales, on 128 bytes each
  static constexpr int kRings = W * kQ8Stages * kStage, kScaleAt = kRings, kFactorAt = kScaleAt + W * kQ8Stages * kScales;
  static constexpr int kBytes = kFactorAt + W * 3 * kPage * 4 + 1024;
  static_assert(kRings >= W * (16 * D + 32) * 4, "merge space must fit in the rings");
};

template <int D, int W>
__global__ void __launch_bounds__(W * 32, kQ8SmWarps / W)
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
  griddep_wait();
  griddep_launch();
  PagePlan plan{int(blockIdx.z), 0, 1, 0x3fffffff};
  if (p.units && !plan_pages<false>(p, blockIdx.x, 2 * W, lane, plan)) return;
  const int b = plan.b, split = plan.split, ctx = p.context(b);
  int page_lo, kept;
  const int npages = pages_of<false>(p, ctx, page_lo, kept);
  const int p0 = page_lo + split * (plan.splits > 1 ? plan.per : 0), p1 = min(page_lo + npages, p0 + plan.per);
  const int* table = p.block_table + b * p.table_stride;

  uint8_t* my_ring = smem + warp * kQ8Stages * L::kStage;
  uint8_t* my_scales = smem + L::kScaleAt + warp * kQ8Stages * L::kScales;
  float* my_factors = reinterpret_cast<float*>(smem + L::kFactorAt) + warp * 3 * kPage;
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
  int blks[kQ8Stages];
#pragma unroll
  for (int s = 0; s < kQ8Stages; ++s) {
    const int pg = p0 + warp + s * W;
    blks[s] = pg < p1 ? table[pg] : 0;
  }
#pragma unroll
  for (int s = 0; s < kQ8Stages; ++s)
    if (p0 + warp + s * W < p1) issue(blks[s], s);

  // ---- query fragments (the first pages are on their way): four neighbouring columns per lane and step, as the keys come
  uint32_t qf[D / 16][4];
  float rs0, rs1;                        // raw score -> exponent of two, without the key's factor
  {
    const __nv_bfloat16* q0 = p.q + (((long long)b * p.q_len + g / p.group) * p.nq + kvh * p.group + g % p.group) * D + 4 * t;
    const __nv_bfloat16* q1 = p.q + (((long long)b * p.q_len + (g + 8) / p.group) * p.nq + kvh * p.group + (g + 8) % p.group) * D + 4 * t;
    auto load_row = [&](const __nv_bfloat16* src, bool on, float& rs, int half) {
      uint2 v[D / 16];
      float mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        v[ks] = on ? *reinterpret_cast<const uint2*>(src + 16 * ks) : make_uint2(0u, 0u);
        const float2 a = unpack_bf16x2(v[ks].x), c = unpack_bf16x2(v[ks].y);
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(a.x)), fmaxf(fabsf(a.y), fabsf(c.x))), fabsf(c.y));
      }
      mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 2));
      const int e = max((__float_as_int(mx) >> 23) - 127, -100);
      const float up = exp2_int(14 - e);
      rs = p.scale_log2 * exp2_int(min(e - 14, 127));
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const float2 a = unpack_bf16x2(v[ks].x), c = unpack_bf16x2(v[ks].y);
        qf[ks][half] = pack_f16x2(a.x * up, a.y * up);
        qf[ks][2 + half] = pack_f16x2(c.x * up, c.y * up);
      }
    };
    load_row(q0, g < rows, rs0, 0);
    load_row(q1, g + 8 < rows, rs1, 1);
  }
  // last and first visible position of the rows this lane has, and of all rows
  const int pos0 = ctx - p.q_len + (g < rows ? g / p.group : 0), pos1 = ctx - p.q_len + (g + 8 < rows ? (g + 8) / p.group : 0);
  const int low0 = nkb_first_visible(pos0, p.window, p.chunk), low1 = nkb_first_visible(pos1, p.window, p.chunk);
  const int all_hi = ctx - p.q_len, all_lo = nkb_first_visible(ctx - 1, p.window, p.chunk);

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  int stage = 0;
  uint32_t phase = 0;
  for (int pg = p0 + warp; pg < p1; pg += W) {
    const int next = pg + kQ8Stages * W;
    const int next_blk = next < p1 ? table[next] : 0;
    const bool ok = mbar_wait(&bars[warp][stage], phase, &abort_flag, p.status, ERR_WAIT_SMEM_FULL);
    if (!__all_sync(kAll, ok)) break;
    const uint32_t kbase = smem_u32(my_ring + stage * L::kStage), vbase = kbase + L::kMat;
    {
      // lane = token: its factors, for the lanes that hold its scores
      const int kb = my_scales[stage * L::kScales + lane], vb = my_scales[stage * L::kScales + 128 + lane];
      const float ve = float(q8_log2_of(vb));
      my_factors[lane] = q8_factor_of(kb);
      my_factors[kPage + lane] = vb == 255 ? __int_as_float(0x7fc00000) : ve;
      my_factors[2 * kPage + lane] = exp2_int(-q8_log2_of(vb));
    }
    __syncwarp();

    float s[4][4];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int kp = 0; kp < D / 64; ++kp) {
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        uint32_t r[4];
        ldsm_x4(kbase + q8_piece<D>(nt * 8 + (lane & 7), 4 * kp + (lane >> 3)), r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mma_16816_f16(s[nt], qf[4 * kp + i], e4m3x2_to_f16x2(uint16_t(r[i])), e4m3x2_to_f16x2(uint16_t(r[i] >> 16)));
      }
    }
    // t = s + v, the mask only where a page crosses an edge
    const int tok0 = pg * kPage;
    const bool edge = tok0 + kPage - 1 > all_hi || tok0 < all_lo;
    float mx0 = -INFINITY, mx1 = -INFINITY;
    float back[4][2];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
      const float2 kf = *reinterpret_cast<const float2*>(my_factors + nt * 8 + 2 * t);
      const float2 ve = *reinterpret_cast<const float2*>(my_factors + kPage + nt * 8 + 2 * t);
      const float2 bk = *reinterpret_cast<const float2*>(my_factors + 2 * kPage + nt * 8 + 2 * t);
      back[nt][0] = bk.x;
      back[nt][1] = bk.y;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v0 = fmaf(s[nt][e] * rs0, e ? kf.y : kf.x, e ? ve.y : ve.x);
        float v1 = fmaf(s[nt][2 + e] * rs1, e ? kf.y : kf.x, e ? ve.y : ve.x);
        if (edge) {
          const int tok = tok0 + nt * 8 + 2 * t + e;
          if (tok > pos0 || tok < low0) v0 = -INFINITY;
          if (tok > pos1 || tok < low1) v1 = -INFINITY;
        }
        s[nt][e] = v0;
        s[nt][2 + e] = v1;
        mx0 = fmaxf(mx0, v0);
        mx1 = fmaxf(mx1, v1);
      }
    }
    // M follows the largest t when that has grown by more than kQ8Grow
    if (__any_sync(kAll, mx0 > m0 + kQ8Grow || mx1 > m1 + kQ8Grow)) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(kAll, mx0, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(kAll, mx0, 2));
      mx1 = fmaxf(mx1, __shfl_xor_sync(kAll, mx1, 1));
      mx1 = fmaxf(mx1, __shfl_xor_sync(kAll, mx1, 2));
      const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
      const float a0 = m0 == -INFINITY ? 0.f : exp2f(m0 - mn0), a1 = m1 == -INFINITY ? 0.f : exp2f(m1 - mn1);
      m0 = mn0;
      m1 = mn1;
      l0 *= a0;
      l1 *= a1;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= a0; o[i][1] *= a0;
        o[i][2] *= a1; o[i][3] *= a1;
      }
    }
    const float base0 = (m0 == -INFINITY ? 0.f : m0) - kQ8Lift, base1 = (m1 == -INFINITY ? 0.f : m1) - kQ8Lift;
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[nt][e] = exp2f(s[nt][e] - base0);
        s[nt][2 + e] = exp2f(s[nt][2 + e] - base1);
        l0 = fmaf(s[nt][e], back[nt][e], l0);
        l1 = fmaf(s[nt][2 + e], back[nt][e], l1);
      }
    }
    // O += P V
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t pa[4] = {pack_f16x2(s[2 * j][0], s[2 * j][1]), pack_f16x2(s[2 * j][2], s[2 * j][3]),
                              pack_f16x2(s[2 * j + 1][0], s[2 * j + 1][1]), pack_f16x2(s[2 * j + 1][2], s[2 * j + 1][3])};
#pragma unroll
      for (int cp = 0; cp < D / 32; ++cp) {
        uint32_t r[4];
        ldsm_x4_t(vbase + q8_piece<D>(16 * j + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * cp + (lane >> 4)), r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __byte_perm(r[i], 0u, 0x3120);     // pairs of tokens: column 2g below, 2g + 1 above
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mma_16816_f16(o[4 * cp + 2 * c], pa, e4m3x2_to_f16x2(uint16_t(r[2 * c])), e4m3x2_to_f16x2(uint16_t(r[2 * c + 1])));
          mma_16816_f16(o[4 * cp + 2 * c + 1], pa, e4m3x2_to_f16x2(uint16_t(r[2 * c] >> 16)), e4m3x2_to_f16x2(uint16_t(r[2 * c + 1] >> 16)));
        }
      }
    }
    __syncwarp();
    if (next < p1) issue(next_blk, stage);
    if (++stage == kQ8Stages) { stage = 0; phase ^= 1u; }
  }
  l0 += __shfl_xor_sync(kAll, l0, 1);
  l0 += __shfl_xor_sync(kAll, l0, 2);
  l1 += __shfl_xor_sync(kAll, l1, 1);
  l1 += __shfl_xor_sync(kAll, l1, 2);

  if (abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  __syncthreads();  // every load consumed: the rings are merge space now

  float* mo = reinterpret_cast<float*>(smem);             // [warp][16][D]
  float* mm = mo + W * 16 * D;                            // [warp][16]
  float* ml = mm + W * 16;
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    // column 16 c + 4 t + i: even ones in one tile, odd ones in the next
    if (g < rows)
      *reinterpret_cast<float4*>(mo + (warp * 16 + g) * D + 16 * c + 4 * t) = make_float4(o[2 * c][0], o[2 * c + 1][0], o[2 * c][1], o[2 * c + 1][1]);
    if (g + 8 < rows)
      *reinterpret_cast<float4*>(mo + (warp * 16 + g + 8) * D + 16 * c + 4 * t) = make_float4(o[2 * c][2], o[2 * c + 1][2], o[2 * c][3], o[2 * c + 1][3]);
  }
  if (t == 0) {
    mm[warp * 16 + g] = m0; mm[warp * 16 + g + 8] = m1;
    ml[warp * 16 + g] = l0; ml[warp * 16 + g + 8] = l1;
  }
  __syncthreads();
  // o and l carry 2^(lift - M); merged values 2^(lift - mf)
  auto finish = [&](int r, int d, float mf, float l, float4 acc) {
    const int head = kvh * p.group + r % p.group;
    if (p.sinks) {
      const float sk = p.sinks[head] * 1.4426950408889634f, m2 = fmaxf(mf, sk), sc = mf == -INFINITY ? 0.f : exp2f(mf - m2);
      acc.x *= sc; acc.y *= sc; acc.z *= sc; acc.w *= sc;
      l = l * sc + exp2f(sk - m2 + kQ8Lift);
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
      const float mw = mm[w * 16 + r], sc = mw == -INFINITY && mf != -INFINITY ? 0.f : exp2f(mw == mf ? 0.f : mw - mf);
      const float4 x = *reinterpret_cast<const float4*>(mo + (w * 16 + r) * D + d);
      acc.x += sc * x.x; acc.y += sc * x.y; acc.z += sc * x.z; acc.w += sc * x.w;
      l += sc * ml[w * 16 + r];
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
      const float keep = mf == mn ? 1.f : exp2f(mf - mn);
      acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
      l *= keep;
      mf = mn;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (s0 + i >= plan.splits) break;
        const float sc = ms[i] == mn ? 1.f : exp2f(ms[i] - mn);
        acc.x += sc * x[i].x; acc.y += sc * x[i].y; acc.z += sc * x[i].z; acc.w += sc * x[i].w;
        l += sc * ls[i];
      }
    }
    finish(r, d, mf, l, acc);
  }
}

template <int D, int W>
static int launch_decode_q8(const CUtensorMap (&m)[4], const DecodeQ8Params& p, cudaStream_t s) {
  using L = DecodeQ8Smem<D, W>;
  static bool attr_set[64] = {false};    // the attribute is per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_q8_decode_kernel<D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (e != cudaSuccess) return int(e);
    attr_set[dev] = true;
  }
  const dim3 grid = p.units ? dim3(p.units, p.nkv, 1) : dim3(1, p.nkv, p.batch);
  return launch_pdl(attn_q8_decode_kernel<D, W>, grid, dim3(W * 32), size_t(L::kBytes), s, m[0], m[1], m[2], m[3], p);
}

template <int D>
static int dispatch_decode_q8(const CUtensorMap (&m)[4], const DecodeQ8Params& p, cudaStream_t s) {
  const long long ctas = (long long)(p.units ? p.units : p.batch) * p.nkv, sms = num_sms();
  if (ctas <= sms) return launch_decode_q8<D, 8>(m, p, s);
  if (ctas <= 2 * sms) return launch_decode_q8<D, 4>(m, p, s);
  if (ctas <= 4 * sms) return launch_decode_q8<D, 2>(m, p, s);
  return launch_decode_q8<D, 1>(m, p, s);
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

extern "C" long long nkb_q8_attn_decode_scratch_floats(int batch, int nkv, int head_dim, int group, int num_splits) {
  if (num_splits <= 1) return 0;
  return kQ8Counters + (long long)plan_units(batch, nkv, group, num_splits) * nkv * (16 * head_dim + 32);
}

// At most 16 query rows per kv head (q_len * nq / nkv).  num_splits > 1: scratch as large as the function above says, its first kQ8Counters
// words zero before the first call (a call leaves them at zero).
extern "C" int nkb_q8_attn_decode(const void* q, const void* k_values, const void* k_scales, const void* v_values, const void* v_scales,
                                  const int* block_table, const int* context_lens, void* out, float* scratch, int batch, int q_len, int nq,
                                  int nkv, int head_dim, int num_blocks, int table_width, long long table_stride, float scale, int window,
                                  int chunk, const float* sinks, int num_splits, void* stream) {
  if (batch <= 0) return 0;
  if (nkv < 1 || nq % nkv || q_len * (nq / nkv) > 16 || nkv > 65535 || batch > 65535) return -2;
  if (num_splits > 1 && (!scratch || (long long)batch * nkv > kQ8Counters)) return -2;
  if (!status_word() && nkb_init() != 0) return -1;
  DecodeQ8Params p{};
  p.q = (const __nv_bfloat16*)q;
  p.block_table = block_table; p.context_lens = context_lens;
  p.out = (__nv_bfloat16*)out;
  p.scratch = num_splits > 1 ? scratch + kQ8Counters : nullptr;
  p.counters = reinterpret_cast<unsigned int*>(scratch);
  p.sinks = sinks;
  p.status = status_word();
  p.batch = batch; p.q_len = q_len; p.nq = nq; p.nkv = nkv; p.group = nq / nkv; p.table_width = table_width;
  p.window = window; p.chunk = chunk;
  p.units = plan_units(batch, nkv, p.group, num_splits);
  p.table_stride = table_stride;
  p.scale_log2 = scale * 1.4426950408889634f;
  CUtensorMap m[4];
  if (int rc = q8_maps(m, {k_values, v_values, k_scales, v_scales}, head_dim, nkv, num_blocks)) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (head_dim == 128) return dispatch_decode_q8<128>(m, p, s);
  if (head_dim == 64) return dispatch_decode_q8<64>(m, p, s);
  return -2;
}
