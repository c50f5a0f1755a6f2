// Products of rows and weights in 8-bit whole numbers: y[m, n] = sx[m] * sw[n] * sum_k x[m, k] w[n, k], both operands K-major.
//
// The sums are whole numbers of 32 bits (at most 128 * 128 * k, so k is up to 131071), exact whatever their order; the only roundings are
// those of the epilogue: sum -> fp32, times sx, times sw, gate, + bias, + residual, -> bf16, the same operations in every kernel (i8_epilogue.cuh).  So every
// variant below, and the kernel for few tokens, gives a token the same bits, whatever else is in the step.
//
// Two kernels:
//   pairs  D[tokens, features] on CTA pairs (tcgen05.mma.cta_group::2.kind::i8, tiles of 256 tokens by up to 256 features), for prompts;
//          see gemm_2cta.cu for the scheme, which this one shares: a slab is 128 bytes of k, 64 bf16 there and 128 numbers here.
//   swap   D[features, tokens] for few tokens: 128 features fill the M side, up to 128 tokens the narrow one.  One tile per CTA and several CTAs per SM, so
//          that one's start and end lie under another's loads; k may be divided among the CTAs of a cluster, whose sums are joined through distributed
//          shared memory, or left as partial sums.
#include "api.h"
#include "gemm_tcgen05.cuh"
#include "i8_args.h"
#include "i8_epilogue.cuh"

namespace nkb {

constexpr int kI8Slab = 128;                       // bytes (numbers) of k per stage: one swizzled row
constexpr int kI8ATile = 128 * kI8Slab;            // 16 KB
constexpr int kI8MaxK = 131071;                    // 128 * 128 * k < 2^31

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::i8: signed numbers, sums in 32 bits, both operands K-major.
__host__ __device__ constexpr uint32_t make_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// (Argument blocks: small ones, see GemmArgs.)
struct I8Out {                // what the epilogues write
  int m, n;                   // tokens, features; the up half of w and its scales begin at n
  int act, fp32;
  long long ldo;
  void* out;
  const float *sx, *sw;
  const __nv_bfloat16 *bias, *residual;
};
struct I8SwapArgs {
  I8Out o;
  int kb_total, kb_per_split, splits, stages;
  int join;                   // the CTAs of a cluster (as many as splits) join their sums; otherwise splits leave partial sums
  int static_w;
  long long split_stride;
  int* status;
};
struct I8PairArgs {
  I8Out o;
  int kb_total, stages;
  int tiles_m, tiles_n, tile_n, group_m;
  int splits, kb_per_split;   // more than one: partial sums in 32 bits, split s at o.out + s * split_stride
  short static_w, gated;
  int apart;                  // rows of results or of the residual do not start on sixteen bytes
  long long split_stride;
  int* status;
};
static_assert(sizeof(I8SwapArgs) <= 112 && sizeof(I8PairArgs) <= 128, "argument blocks grew past the fast kernel-parameter size");

// ------------------------------------------------------------------------------------------------ swap
struct I8Ctrl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t done;
  uint32_t tmem_base;
  int abort;
};

// Scales and bias of the four features from f on (those past the last one read its); they stay with a thread for all of its tokens.
template <bool GATED>
struct Features4 {
  float sw[4], su[4], bias[4];
  __device__ __forceinline__ Features4(const I8Out& a, bool first, int f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int fj = min(f + j, a.n - 1);
      sw[j] = __ldg(a.sw + fj);
      su[j] = GATED ? __ldg(a.sw + a.n + fj) : 0.f;
      bias[j] = !GATED && a.bias && first ? __bfloat162float(a.bias[fj]) : 0.f;
    }
  }
};

// Four finished features (whole sums s, up half u) of one token, from feature f on; at: where the results begin.
template <bool GATED>
__device__ __forceinline__ void i8_store4(const I8Out& a, const Features4<GATED>& w, long long at, int tok, int f, const int4& s, const int4& u) {
  const float sx = a.sx[tok];
  const int sv[4] = {s.x, s.y, s.z, s.w}, uv[4] = {u.x, u.y, u.z, u.w};
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = i8_scaled(sv[j], sx, w.sw[j]);
    if constexpr (GATED) y[j] = i8_gated(y[j], i8_scaled(uv[j], sx, w.su[j]), a.act);
    else if (a.bias) y[j] = add_rn(y[j], w.bias[j]);
  }
  at += (long long)tok * a.ldo + f;
  const bool whole = f + 4 <= a.n;
  if (!GATED && a.residual) {
    const __nv_bfloat16* r = a.residual + at;
    if (whole && (reinterpret_cast<uintptr_t>(r) & 7) == 0) {
      const uint2 v = *reinterpret_cast<const uint2*>(r);
      const float2 lo = unpack_bf16x2(v.x), hi = unpack_bf16x2(v.y);
      y[0] = add_rn(y[0], lo.x); y[1] = add_rn(y[1], lo.y); y[2] = add_rn(y[2], hi.x); y[3] = add_rn(y[3], hi.y);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f + j < a.n) y[j] = add_rn(y[j], __bfloat162float(r[j]));
    }
  }
  if (a.fp32) {
    float* o = reinterpret_cast<float*>(a.out) + at;
    if (whole && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
      *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f + j < a.n) o[j] = y[j];
    }
  } else {
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
    if (whole && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
      *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f + j < a.n) o[j] = __float2bfloat16(y[j]);
    }
  }
}

// Grid: x = feature tiles * splits (the splits of a tile follow one another; joined ones are a cluster), y = token tiles of BN.
template <int BN, bool GATED>
__global__ void __launch_bounds__(128)
i8_swap_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const I8SwapArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ I8Ctrl ctrl;
  constexpr int kW = GATED ? 2 : 1;
  constexpr int kStage = kW * kI8ATile + BN * kI8Slab;
  constexpr uint32_t kCols = (kW * BN) < 32 ? 32 : kW * BN;
  const int warp = warp_idx_uniform(), lane = threadIdx.x & 31;
  const int tile = blockIdx.x / args.splits, split = blockIdx.x - tile * args.splits;
  const int f0 = tile * 128, tok0 = blockIdx.y * BN;
  const int kb0 = split * args.kb_per_split, kb1 = min(args.kb_total, kb0 + args.kb_per_split);
  const int slabs = kb1 - kb0, stages = args.stages;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&ctrl.full[s], 1);
      mbar_init(&ctrl.empty[s], 1);
    }
    mbar_init(&ctrl.done, 1);
    ctrl.abort = 0;
    mbar_fence_init();
    fence_proxy_async();
  }
  if (warp == 2) {
    tmem_alloc(&ctrl.tmem_base, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctrl.tmem_base;
  volatile int* abort_flag = &ctrl.abort;
  griddep_launch();

  if (warp == 0) {
    if (lane == 0) {
      auto load_w = [&](int stage, int kb) {
        uint8_t* p = tiles + stage * kStage;
        tma_load_2d(p, &tmW, &ctrl.full[stage], kb * kI8Slab, f0);
        if (GATED) tma_load_2d(p + kI8ATile, &tmW, &ctrl.full[stage], kb * kI8Slab, args.o.n + f0);
      };
      auto load_x = [&](int stage, int kb) {
        tma_load_2d(tiles + stage * kStage + kW * kI8ATile, &tmX, &ctrl.full[stage], kb * kI8Slab, tok0);
      };
      // weights do not depend on the kernel before this one: the first turn of the ring takes them ahead of the wait
      const int pre = args.static_w ? min(stages, slabs) : 0;
      for (int i = 0; i < pre; ++i) {
        mbar_expect_tx(&ctrl.full[i], kStage);
        load_w(i, kb0 + i);
      }
      griddep_wait();
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < slabs; ++i) {
        if (!mbar_wait(&ctrl.empty[stage], phase ^ 1u, abort_flag, args.status, ERR_WAIT_SMEM_EMPTY)) break;
        if (i >= pre) {
          mbar_expect_tx(&ctrl.full[stage], kStage);
          load_w(stage, kb0 + i);
        }
        load_x(stage, kb0 + i);
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_i8(128, BN);
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      const uint64_t d_tiles = make_smem_desc_sw128(smem_u32(tiles), 0, 1024);
      const uint64_t d_hi = d_tiles & 0xffffffff00000000ull;
      const uint32_t w_lo0 = uint32_t(d_tiles);
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(&ctrl.full[stage], phase, abort_flag, args.status, ERR_WAIT_SMEM_FULL);
        if (!ok) break;
        tc_fence_after();
        const uint32_t w_lo = w_lo0 + uint32_t(stage) * uint32_t(kStage >> 4);
        const uint64_t dw = d_hi | w_lo, du = d_hi | (w_lo + uint32_t(kI8ATile >> 4)), dx = d_hi | (w_lo + uint32_t(kW * kI8ATile >> 4));
#pragma unroll
        for (int k = 0; k < 4; ++k) {          // 32 numbers per instruction
          const uint32_t acc = (kb > kb0 || k > 0) ? 1u : 0u;
          umma_i8(tmem_base, dw + uint64_t(2 * k), dx + uint64_t(2 * k), idesc, acc);
          if (GATED) umma_i8(tmem_base + BN, du + uint64_t(2 * k), dx + uint64_t(2 * k), idesc, acc);
        }
        umma_commit(&ctrl.empty[stage]);
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
      if (ok) umma_commit(&ctrl.done);
    }
    __syncwarp();
  }

  // ---- all four warps: warp w holds features 32 w .. 32 w + 31 of the tile
  griddep_wait();
  bool ok = mbar_wait(&ctrl.done, 0, abort_flag, args.status, ERR_WAIT_TMEM_FULL);
  ok = __all_sync(0xffffffffu, ok);
  tc_fence_after();
  int* stg = reinterpret_cast<int*>(tiles);      // [kW][BN tokens][128 features], over the ring that is done with
  if (ok) {
    const uint32_t t0 = tmem_base + (uint32_t(warp * 32) << 16);
#pragma unroll 1
    for (int c = 0; c < kW * BN; c += 16) {
      uint32_t v[16];
      tmem_ld_32x16(t0 + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) stg[(c + j) * 128 + warp * 32 + lane] = int(v[j]);
    }
  }
  const int joined = args.join ? args.splits : 1;
  ok = __syncthreads_and(ok);
  if (joined > 1) cluster_sync_all();            // (a CTA that gave up takes part too)
  if (ok) {
    // A lane has four features, a warp goes from token to token; the CTAs of a cluster share the tokens, or the features of fewer tokens than CTAs.
    const int toks = min(BN, args.o.m - tok0), rank = joined > 1 ? split : 0, f = lane * 4;
    const bool by_token = toks >= joined;
    const bool mine = f0 + f < args.o.n && (by_token || lane / (32 / joined) == rank);
    const int step = by_token ? 4 * joined : 4, first_tok = by_token ? warp * joined + rank : warp;
    if (mine) {
      const Features4<GATED> w(args.o, args.join || split == 0, f0 + f);
      const long long at = args.join ? 0 : split * args.split_stride;
      for (int t = first_tok; t < toks; t += step) {
        const int* p = stg + t * 128 + f;
        int4 s, u = make_int4(0, 0, 0, 0);
        if (joined > 1) {
          int4 v[8], q[GATED ? 8 : 1];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r < joined) {
              v[r] = ld_cluster_v4(map_to_cta(p, r));
              if (GATED) q[r] = ld_cluster_v4(map_to_cta(p + BN * 128, r));
            }
          s = v[0];
          if (GATED) u = q[0];
#pragma unroll
          for (int r = 1; r < 8; ++r)
            if (r < joined) {
              s.x += v[r].x; s.y += v[r].y; s.z += v[r].z; s.w += v[r].w;
              if (GATED) {
                u.x += q[r].x; u.y += q[r].y; u.z += q[r].z; u.w += q[r].w;
              }
            }
        } else {
          s = *reinterpret_cast<const int4*>(p);
          if (GATED) u = *reinterpret_cast<const int4*>(p + BN * 128);
        }
        i8_store4<GATED>(args.o, w, at, tok0 + t, f0 + f, s, u);
      }
    }
  }
  if (joined > 1) cluster_sync_all();            // shared memory stays until every CTA of the cluster has read it
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kCols);
  }
}

// ------------------------------------------------------------------------------------------------ pairs
constexpr int kPairTileN = 256;
constexpr int kPairStage = 2 * kI8ATile;
constexpr int kPairStages = 7, kApartStages = 6;   // (without and with the epilogue's tiles)
// Warps of the epilogue.  1024 tokens by 4096 x 4096, us, with four and eight at the widths 128, 192 and 256: 21.1 and 20.7, 24.5 and 22.6, 21.9 and 20.5;
// 414 by 2 x 14336 x 4096 54.7 and 62.0, 50.0 and 53.7, 52.1 and 51.7; 4096 tokens by it 359 and 399, 314 and 333, 297 and 296.
__host__ __device__ constexpr int pair_warps(bool gated) { return gated ? 4 : 8; }
constexpr int kApartBytes = pair_warps(false) * 32 * 33 * 4;      // a tile of 32 x 32 sums for each
constexpr int kPairSmem = 232448;
static_assert(2048 + kApartStages * kPairStage + kApartBytes <= kPairSmem && 2048 + kPairStages * kPairStage <= kPairSmem, "more than an SM's shared memory");

struct WorkI8 {
  int tm, tn, sp, kb0, kb1;
};
// group_m row tiles share a sweep over the column tiles, so that both operands are read again from L2; the splits of a tile follow one another.
//
// The slabs' bounds come from the split even where there is one.  With a loop from zero to a kernel argument (nvcc 12.9) an MMA takes 65 cycles to issue and not
// 16, and 200 tokens by 4096 x 14336 40 us and not 25.
__device__ __forceinline__ WorkI8 i8_work(const I8PairArgs& a, int w) {
  WorkI8 o;
  o.sp = w % a.splits;
  const int t = w / a.splits;
  const int per_group = a.group_m * a.tiles_n;
  const int gr = t / per_group, first = gr * a.group_m;
  const int gsz = min(a.tiles_m - first, a.group_m), in = t - gr * per_group;
  o.tm = first + in % gsz;
  o.tn = in / gsz;
  o.kb0 = o.sp * a.kb_per_split;
  o.kb1 = min(a.kb_total, o.kb0 + a.kb_per_split);
  return o;
}

// 32 finished columns of a row from column c on, cols_end at most; at: where the results begin.
template <bool GATED>
__device__ __forceinline__ void i8_store_row(const I8Out& a, bool first, long long at, int row, int c, int cols_end, float (&y)[32]) {
  at += (long long)row * a.ldo + c;
  if (!GATED && a.bias && first) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c + j < cols_end) y[j] = add_rn(y[j], __bfloat162float(__ldg(a.bias + c + j)));
  }
  if (!GATED && a.residual) {
    const __nv_bfloat16* r = a.residual + at;
    const bool r16 = (reinterpret_cast<uintptr_t>(r) & 15) == 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (r16 && c + 8 * q + 8 <= cols_end) {
        const uint4 rr = reinterpret_cast<const uint4*>(r)[q];
        const uint32_t rw[4] = {rr.x, rr.y, rr.z, rr.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack_bf16x2(rw[e]);
          y[8 * q + 2 * e] = add_rn(y[8 * q + 2 * e], f.x);
          y[8 * q + 2 * e + 1] = add_rn(y[8 * q + 2 * e + 1], f.y);
        }
      } else {
#pragma unroll
        for (int j = 8 * q; j < 8 * q + 8; ++j)
          if (c + j < cols_end) y[j] = add_rn(y[j], __bfloat162float(r[j]));
      }
    }
  }
  if (a.fp32) {
    float* o = reinterpret_cast<float*>(a.out) + at;
    const bool o16 = (reinterpret_cast<uintptr_t>(o) & 15) == 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (o16 && c + 4 * q + 4 <= cols_end) {
        reinterpret_cast<float4*>(o)[q] = make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
      } else {
#pragma unroll
        for (int j = 4 * q; j < 4 * q + 4; ++j)
          if (c + j < cols_end) o[j] = y[j];
      }
    }
    return;
  }
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
  const bool o16 = (reinterpret_cast<uintptr_t>(o) & 15) == 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (o16 && c + 8 * q + 8 <= cols_end) {
      reinterpret_cast<uint4*>(o)[q] = make_uint4(pack_bf16x2(y[8 * q], y[8 * q + 1]), pack_bf16x2(y[8 * q + 2], y[8 * q + 3]),
                                                  pack_bf16x2(y[8 * q + 4], y[8 * q + 5]), pack_bf16x2(y[8 * q + 6], y[8 * q + 7]));
    } else {
#pragma unroll
      for (int j = 8 * q; j < 8 * q + 8; ++j)
        if (c + j < cols_end) o[j] = __float2bfloat16(y[j]);
    }
  }
}

// The same of the warp's 32 rows from row0 on where they do not start on sixteen bytes: through shared memory, so that the lanes store neighbouring columns of
// a row (848 tokens by 2 x 10726 x 100, whose rows start on four bytes: 118 us lane by lane, each with a row of its own).
template <bool GATED>
__device__ __forceinline__ void i8_store_rows(const I8Out& a, bool first, long long at, int row0, int c, int cols_end, const float (&y)[32], float* tile) {
  const int lane = threadIdx.x & 31, col = c + lane;
#pragma unroll
  for (int j = 0; j < 32; ++j) tile[lane * 33 + j] = y[j];
  __syncwarp();
  if (col < cols_end) {
    const float bias = !GATED && a.bias && first ? __bfloat162float(__ldg(a.bias + col)) : 0.f;
    const int rows = min(32, a.m - row0);
    at += (long long)row0 * a.ldo + col;
#pragma unroll 8
    for (int r = 0; r < rows; ++r, at += a.ldo) {
      float v = tile[r * 33 + lane];
      if (!GATED && a.bias) v = add_rn(v, bias);
      if (!GATED && a.residual) v = add_rn(v, __bfloat162float(a.residual[at]));
      if (a.fp32) reinterpret_cast<float*>(a.out)[at] = v;
      else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16(v);
    }
  }
  __syncwarp();
}

// Scales of the columns from c on; those from cols_end on are another's.
__device__ __forceinline__ void i8_scales(const float* sw, int c, int cols_end, float (&s)[32]) {
  const bool s16 = (reinterpret_cast<uintptr_t>(sw + c) & 15) == 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if (s16 && c + 4 * q + 4 <= cols_end) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(sw + c) + q);
      s[4 * q] = f.x; s[4 * q + 1] = f.y; s[4 * q + 2] = f.z; s[4 * q + 3] = f.w;
    } else {
#pragma unroll
      for (int j = 4 * q; j < 4 * q + 4; ++j) s[j] = __ldg(sw + min(c + j, cols_end - 1));
    }
  }
}

template <bool GATED>
__device__ __forceinline__ void i8_pair_body(const CUtensorMap& tmX, const CUtensorMap& tmW, const I8PairArgs& args) {
  constexpr int W = pair_warps(GATED);
  extern __shared__ uint8_t smem_raw[];
  // identical layout in both CTAs: [control 1 KB][ring]
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  GemmCtrl* ctrl = reinterpret_cast<GemmCtrl*>(base);
  uint8_t* tiles = base + 1024;
  const int warp = warp_idx_uniform();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();        // 0 = issues the MMAs
  const int stages = args.stages;
  constexpr uint32_t tmem_cols = 2 * kPairTileN;     // two accumulators of 256 columns
  const int tile_n = args.tile_n, half_n = tile_n / 2;     // half_n: rows of B per CTA
  const uint32_t stage_tx = 2u * uint32_t(kI8ATile + half_n * kI8Slab);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&ctrl->full[s], 1);
      mbar_init(&ctrl->empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctrl->tfull[i], 1);
      mbar_init(&ctrl->tempty[i], 2 * W);
    }
    ctrl->abort = 0;
    mbar_fence_init();
    fence_proxy_async();
  }
  if (warp == 1) {
    tmem_alloc_pair(&ctrl->tmem_base, tmem_cols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                              // both CTAs' barriers exist before anything remote arrives
  tc_fence_after();
  const uint32_t tmem_base = ctrl->tmem_base;
  volatile int* abort_flag = &ctrl->abort;

  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int total_work = args.tiles_m * args.tiles_n * args.splits;
  griddep_launch();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    auto b_row_of = [&](const WorkI8& t) {
      return args.gated ? int(rank) * args.o.n + t.tn * half_n : t.tn * tile_n + int(rank) * half_n;
    };
    // Weight tiles do not depend on the preceding kernel: the first fill of the ring takes them before the wait.  (The second
    // CTA's bytes may arrive before the first one has announced them: a barrier's phase ends only with the announcement.)
    int pre = 0;
    if (args.static_w && pair < total_work) {
      const WorkI8 t = i8_work(args, pair);
      pre = min(stages, t.kb1 - t.kb0);
      if (lane == 0)
        for (int i = 0; i < pre; ++i) {
          if (rank == 0) mbar_expect_tx(&ctrl->full[i], stage_tx);
          tma_load_2d_pair(tiles + i * kPairStage + kI8ATile, &tmW, map_to_cta(&ctrl->full[i], 0), (t.kb0 + i) * kI8Slab,
                           b_row_of(t));
        }
      __syncwarp();
    }
    griddep_wait();
    int stage = 0;
    uint32_t phase = 0;
    bool alive = true;
    for (int w = pair; w < total_work && alive; w += npairs) {
      const WorkI8 t = i8_work(args, w);
      const int a_row = t.tm * 256 + int(rank) * 128;
      const int b_row = b_row_of(t);
      for (int kb = t.kb0; kb < t.kb1; ++kb) {
        bool ok = mbar_wait(&ctrl->empty[stage], phase ^ 1u, abort_flag, args.status, ERR_WAIT_SMEM_EMPTY);
        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        if (lane == 0) {
          const uint32_t full0 = map_to_cta(&ctrl->full[stage], 0);
          uint8_t* a_ptr = tiles + stage * kPairStage;
          // the first CTA announces the bytes of both CTAs; the second only lets its loads complete there
          // (its loads of this phase cannot start before the barrier entered the phase: they wait for the
          // stage to be released, which follows the previous phase's completion)
          const bool ahead = w == pair && kb - t.kb0 < pre;
          if (rank == 0 && !ahead) mbar_expect_tx(&ctrl->full[stage], stage_tx);
          tma_load_2d_pair(a_ptr, &tmX, full0, kb * kI8Slab, a_row);
          if (!ahead) tma_load_2d_pair(a_ptr + kI8ATile, &tmW, full0, kb * kI8Slab, b_row);
        }
        __syncwarp();
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issuer (first CTA of the pair)
    // One elected thread runs the whole loop alone: the tensor pipe queues only a few MMAs, so warp votes,
    // reconvergence and descriptor arithmetic between two k-blocks are time in which it drains.
    const uint32_t idesc = make_idesc_i8(256, tile_n);
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      const uint64_t d_tiles = make_smem_desc_sw128(smem_u32(tiles), 0, 1024);
      const uint64_t d_hi = d_tiles & 0xffffffff00000000ull;
      const uint32_t a_lo0 = uint32_t(d_tiles);
      const uint32_t empty0 = map_to_cta(&ctrl->empty[0], 0), empty1 = map_to_cta(&ctrl->empty[0], 1);
      bool ok = true;
      for (int w = pair; w < total_work && ok; w += npairs) {
        ok = mbar_wait(&ctrl->tempty[acc], acc_phase ^ 1u, abort_flag, args.status, ERR_WAIT_TMEM_EMPTY);
        if (!ok) break;
        const uint32_t d0 = tmem_base + uint32_t(acc * kPairTileN);
        const WorkI8 t = i8_work(args, w);
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          ok = mbar_wait(&ctrl->full[stage], phase, abort_flag, args.status, ERR_WAIT_SMEM_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + uint32_t(stage) * uint32_t(kPairStage >> 4);
          const uint64_t da = d_hi | a_lo, db = d_hi | (a_lo + uint32_t(kI8ATile >> 4));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_i8_pair(d0, da + uint64_t(k * 2), db + uint64_t(k * 2), idesc, (kb > t.kb0 || k > 0) ? 1u : 0u);
          umma_commit_pair(empty0 + uint32_t(stage) * 8u);
          umma_commit_pair(empty1 + uint32_t(stage) * 8u);
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair(map_to_cta(&ctrl->tfull[acc], 0));
        umma_commit_pair(map_to_cta(&ctrl->tfull[acc], 1));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    __syncwarp();
  } else if (warp >= 2) {
    // ------------------------------------------------------------------ epilogue (warps 2.., both CTAs): 32 rows, all 32 columns or every second
    const int quad = warp & 3, part = (warp - 2) >> 2;
    float* apart = reinterpret_cast<float*>(tiles + kApartStages * kPairStage) + (warp - 2) * (32 * 33);
    griddep_wait();
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int w = pair; w < total_work; w += npairs) {
      const WorkI8 t = i8_work(args, w);
      const int row = t.tm * 256 + int(rank) * 128 + quad * 32 + lane;
      const float sx = args.o.sx[min(row, args.o.m - 1)];
      bool ok = mbar_wait(&ctrl->tfull[acc], acc_phase, abort_flag, args.status, ERR_WAIT_TMEM_FULL);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t t0 = tmem_base + (uint32_t(quad * 32) << 16) + uint32_t(acc * kPairTileN);
      const int width = GATED ? half_n : tile_n;
      const int col0 = t.tn * width, cols_end = min(args.o.n, col0 + width);
      // (tiles have at least 64 columns, so every warp has some)
#pragma unroll 1
      for (int c = part * 32; c < width; c += 8 * W) {
        const bool some = col0 + c < cols_end;
        float y[32], s[32];
        uint32_t v[32];
        tmem_ld_32x32(t0 + c, v);
        if (some) i8_scales(args.o.sw, col0 + c, cols_end, s);          // (while the sums are on their way)
        const float2 sx2 = make_float2(sx, sx);
        if constexpr (GATED) {
          uint32_t u[32];
          float su[32];
          tmem_ld_32x32(t0 + half_n + c, u);
          if (some) i8_scales(args.o.sw + args.o.n, col0 + c, cols_end, su);
          tmem_ld_wait();
          if (some) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 g = i8_scaled2(v[j], v[j + 1], sx2, s[j], s[j + 1]), up = i8_scaled2(u[j], u[j + 1], sx2, su[j], su[j + 1]);
              const float2 r = i8_gated2(g, up, args.o.act);
              y[j] = r.x;
              y[j + 1] = r.y;
            }
          }
        } else {
          tmem_ld_wait();
          if (some) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 r = i8_scaled2(v[j], v[j + 1], sx2, s[j], s[j + 1]);
              y[j] = r.x;
              y[j + 1] = r.y;
            }
          }
        }
        if (c + 8 * W >= width) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_cta(&ctrl->tempty[acc], 0));
        }
        if (!some) continue;
        if (args.apart) i8_store_rows<GATED>(args.o, t.sp == 0, t.sp * args.split_stride, row - lane, col0 + c, cols_end, y, apart);
        else if (row < args.o.m) i8_store_row<GATED>(args.o, t.sp == 0, t.sp * args.split_stride, row, col0 + c, cols_end, y);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // neither CTA leaves (and frees shared / tensor memory) while its peer still works
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, tmem_cols);
  }
}

template <bool GATED>
__global__ void __launch_bounds__(64 + 32 * pair_warps(GATED), 1)
i8_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const I8PairArgs args) {
  i8_pair_body<GATED>(tmX, tmW, args);
}

constexpr int kMaxDev = 64;

static int i8_maps(const NkbGemmI8& g, CUtensorMap* x, uint32_t x_box, CUtensorMap* w, uint32_t w_box) {
  const uint64_t xd[2] = {uint64_t(g.k), uint64_t(g.m)}, wd[2] = {uint64_t(g.k), uint64_t(g.gated ? 2 : 1) * uint64_t(g.n)};
  const uint64_t xs[1] = {uint64_t(g.ldx)}, ws[1] = {uint64_t(g.ldw)};
  const uint32_t xb[2] = {uint32_t(kI8Slab), x_box}, wb[2] = {uint32_t(kI8Slab), w_box};
  return encode_tmap_u8(x, g.x, 2, xd, xs, xb, 128) || encode_tmap_u8(w, g.w, 2, wd, ws, wb, 128);
}

template <int BN, bool GATED>
static int launch_swap(const NkbGemmI8& g, I8SwapArgs a) {
  constexpr int kW = GATED ? 2 : 1, kStage = kW * kI8ATile + BN * kI8Slab, kStaging = kW * BN * 128 * 4;
  // Two CTAs per SM where a round is all there is; where tiles come in several rounds, four (three of 128 tokens, whose sums are staged in 64 KB), whose
  // starts and ends lie under one another's loads.  Vocabulary of 128256 x 4096, us: 64 tokens 106 with two per SM and 96 with four, one token 81 and 78.
  const long long ctas = (long long)((g.n + 127) / 128) * a.splits * ((g.m + BN - 1) / BN);
  const int ring = ctas <= 2 * num_sms() ? 110 : (BN == 128 ? 75 : 56);
  int stages = (ring * 1024) / kStage;
  stages = stages > a.kb_per_split ? a.kb_per_split : stages;
  stages = stages < 1 ? 1 : (stages > kMaxStages ? kMaxStages : stages);
  a.stages = stages;
  const int smem = 1024 + (stages * kStage > kStaging ? stages * kStage : kStaging);
  static bool ready[kMaxDev] = {false};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return -1;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(i8_swap_kernel<BN, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return int(e);
    ready[dev] = true;
  }
  CUtensorMap tx, tw;
  if (i8_maps(g, &tx, BN, &tw, 128)) return -4;
  const dim3 grid(unsigned((g.n + 127) / 128 * a.splits), unsigned((g.m + BN - 1) / BN));
  return launch_pdl_cluster(i8_swap_kernel<BN, GATED>, grid, dim3(128), size_t(smem), reinterpret_cast<cudaStream_t>(g.stream),
                            a.join ? a.splits : 1, tw, tx, a);
}

// k divided into whole slabs, none of them empty: at most `want` parts.
template <typename A>
static void divide(A& a, int want) {
  want = want < 1 ? 1 : (want > a.kb_total ? a.kb_total : want);
  a.kb_per_split = (a.kb_total + want - 1) / want;
  a.splits = (a.kb_total + a.kb_per_split - 1) / a.kb_per_split;
}

// CTA pairs that can be resident at once on the current device; negative: an error.
template <bool GATED>
static int resident_pairs(int dev, cudaLaunchConfig_t cfg) {
  static int known[kMaxDev] = {0};
  if (known[dev] == 0) {
    if (cudaFuncSetAttribute(i8_pair_kernel<GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return -1;
    int n = 0;
    cfg.gridDim = dim3(2 * (num_sms() / 2));
    cfg.numAttrs = 1;
    known[dev] = cudaOccupancyMaxActiveClusters(&n, i8_pair_kernel<GATED>, &cfg) == cudaSuccess && n > 0 ? n : num_sms() / 4;
  }
  return known[dev];
}

// Columns of a tile.  A pair takes its tiles one after another, so a narrower tile wins where it makes the rounds come out even.  us per slab of a tile
// (taken at 200 tokens by 4096 x 14336): at 256 columns both operands' 32 KB per CTA and slab are what L2 gives an SM (52 bytes per clock), narrower
// ones wait for the MMAs' and loads' latencies.  us at every width; the rule's choice is within 3 % of the best one:
//   columns                              256    224    192    160    128     96     64   chosen
//    200 tokens by 14336 x 4096         20.4   19.6   22.6   22.2   20.7   24.8   29.2     19.6
//    300 by 6144 x 4096                 18.4   17.3   15.7   19.6   18.9   18.2   22.3     15.7
//    414 by 2 x 14336 x 4096            48.0   49.1   47.4   48.5   52.6   61.6   80.6     48.4
//   1024 by 4096 x 4096                 18.3   20.3   20.5   19.6   18.8   23.4   27.5     18.2
//   1024 by 2 x 14336 x 4096            86.1   88.7   87.9   93.4   97.2  115.5  148.7     88.8
//   2048 by 4096 x 14336                78.6   90.2   85.0   81.8   92.1  106.4  137.1     79.0
static int pair_width(int tiles_m, int splits, int slabs, int columns, bool gated, int pairs, float* us_out) {
  static const struct { int width; float us; } kSlab[] = {{256, 0.326f}, {224, 0.287f}, {192, 0.250f}, {160, 0.224f}, {128, 0.207f}, {96, 0.200f}, {64, 0.192f}};
  int best = 256;
  float best_us = 0.f;
  for (const auto& t : kSlab) {
    const long long tiles = (long long)tiles_m * ((columns + t.width - 1) / t.width) * splits;
    // (a tile of few slabs takes as long as what comes behind its sums: 848 tokens by 2 x 10720 x 100 59 us at 64 columns, 37 at 256)
    const float tile = fmaxf(float(slabs) * t.us, gated ? 0.8f + 1.6f * float(t.width / 64) : 0.7f + 0.95f * float((t.width + 63) / 64));
    const float us = float((tiles + pairs - 1) / pairs) * tile + 4.f + 0.012f * float(t.width);
    if (t.width == 256 || us < 0.97f * best_us) {
      best = t.width;
      best_us = us;
    }
  }
  if (us_out) *us_out = best_us;
  return best;
}

template <bool GATED>
static int launch_i8_pairs(const NkbGemmI8& g, const I8Out& o) {
  I8PairArgs a{};
  a.o = o;
  a.kb_total = (g.k + kI8Slab - 1) / kI8Slab;
  a.static_w = g.static_w;
  a.gated = GATED;
  a.group_m = 16;
  a.split_stride = g.split_stride;
  divide(a, g.splits);
  const int size = g.fp32 ? 4 : 2;
  a.apart = ((reinterpret_cast<uintptr_t>(g.out) | uintptr_t(g.ldo * size) | uintptr_t(g.split_stride * size)) & 15) != 0 ||
            (g.residual && ((reinterpret_cast<uintptr_t>(g.residual) | uintptr_t(g.ldo * 2)) & 15) != 0);
  a.status = status_word();
  a.tiles_m = (g.m + 255) / 256;
  a.stages = a.apart ? kApartStages : kPairStages;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(64 + 32 * pair_warps(GATED));
  cfg.dynamicSmemBytes = size_t(kPairSmem);
  cfg.stream = reinterpret_cast<cudaStream_t>(g.stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  const int pairs = resident_pairs<GATED>(dev, cfg);
  if (pairs < 0) return -1;
  const int columns = (GATED ? 2 : 1) * g.n;
  a.tile_n = pair_width(a.tiles_m, a.splits, a.kb_per_split, columns, GATED, pairs, nullptr);
  a.tiles_n = (columns + a.tile_n - 1) / a.tile_n;
  if (GATED) a.tiles_n = (g.n + a.tile_n / 2 - 1) / (a.tile_n / 2);
  CUtensorMap tx, tw;
  if (i8_maps(g, &tx, 128, &tw, uint32_t(a.tile_n / 2))) return -4;
  const int total = a.tiles_m * a.tiles_n * a.splits;
  cfg.gridDim = dim3(2 * unsigned(pairs < total ? pairs : total));
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return int(cudaLaunchKernelEx(&cfg, i8_pair_kernel<GATED>, tx, tw, a));
}

// CTAs of a cluster that share a tile's k in the swap kernel: doubled while the grid stays within two CTAs per SM and each keeps two slabs.
static int pick_join(int tiles, int kb) {
  int s = 1;
  while (s < 8 && tiles * s * 2 <= 2 * num_sms() && kb / (s * 2) >= 2) s *= 2;
  return s;
}

// Whether pairs take a whole product of more than 32 tokens: the times of both kernels by their models.  That of the swap kernel is a start, an end with its
// staging (6 us at 64 tokens, 8.3 at 128), and 0.33 us per slab and CTA of an SM.  Swap and pairs, us: 64 tokens by 6144 x 4096 9.9 and 12.0, by 4096 x
// 14336 14.9 and 25.5, by 2 x 14336 x 4096 30.8 and 32.9, by 2048 x 768 7.5 and 4.8; 128 by 6144 x 4096 13.1 and 12.8, by 4096 x 14336 17.9 and 25.7, by 128256
// x 4096 121 and 99; 256 by 1500 x 8000 12.3 and 19.9, by 6144 x 4096 19.0 and 13.3.
static bool pairs_first(const NkbGemmI8& g, int bn, int tiles, int splits) {
  const int slabs = (g.k + kI8Slab - 1) / kI8Slab, weights = g.gated ? 2 : 1;
  const long long per_sm = ((long long)tiles * splits + num_sms() - 1) / num_sms();
  const float swap_us = (bn <= 64 ? 6.f : 8.3f) + 0.33f * float(per_sm) * float((slabs + splits - 1) / splits) * float(weights);
  float pair_us = 0.f;
  pair_width((g.m + 255) / 256, 1, slabs, weights * g.n, g.gated, num_sms() / 2, &pair_us);
  return pair_us < swap_us;
}

template <bool GATED>
static int launch_i8(const NkbGemmI8& g, const I8Out& o) {
  const int bn = g.m <= 16 ? 16 : (g.m <= 32 ? 32 : (g.m <= 64 || GATED ? 64 : 128));
  const long long tiles = (long long)((g.n + 127) / 128) * ((g.m + bn - 1) / bn);
  I8SwapArgs a{};
  a.o = o;
  a.kb_total = (g.k + kI8Slab - 1) / kI8Slab;
  a.split_stride = g.split_stride;
  a.static_w = g.static_w;
  a.status = status_word();
  if (g.splits > 0) {
    if (g.m > 128) return launch_i8_pairs<GATED>(g, o);
    divide(a, g.splits);
  } else {
    if (tiles > 64 * num_sms()) return launch_i8_pairs<GATED>(g, o);
    // (a cluster wants as many CTAs as it is launched with, and a power of two of them)
    for (int s = pick_join(int(tiles), a.kb_total);; s /= 2) {
      divide(a, s);
      if (a.splits == s) break;
    }
    a.join = a.splits > 1;
    if (g.m > 32 && pairs_first(g, bn, int(tiles), a.splits)) return launch_i8_pairs<GATED>(g, o);
  }
  if (bn == 16) return launch_swap<16, GATED>(g, a);
  if (bn == 32) return launch_swap<32, GATED>(g, a);
  if (bn == 64) return launch_swap<64, GATED>(g, a);
  if constexpr (!GATED) return launch_swap<128, GATED>(g, a);
  return -2;
}

}  // namespace nkb

using namespace nkb;

// Splits that a product asked for `splits` of them really has.
extern "C" int nkb_gemm_i8_splits(int k, int splits) {
  I8SwapArgs a{};
  a.kb_total = (k + kI8Slab - 1) / kI8Slab;
  divide(a, splits);
  return a.splits;
}

extern "C" int nkb_gemm_i8(const void* packed) {
  const NkbGemmI8& g = *reinterpret_cast<const NkbGemmI8*>(packed);
  if (!status_word() && nkb_init() != 0) return -1;
  if (g.m <= 0 || g.n <= 0) return 0;
  if (g.k <= 0 || g.k > kI8MaxK || (g.ldx & 15) || (g.ldw & 15) || g.ldx < g.k || g.ldw < g.k || g.ldo < g.n) return -2;
  if ((reinterpret_cast<uintptr_t>(g.x) | reinterpret_cast<uintptr_t>(g.w)) & 15) return -2;
  if (g.gated && (g.bias || g.residual || g.fp32 || g.splits)) return -2;
  if (g.splits < 0 || (g.splits > 0 && (!g.fp32 || g.residual))) return -2;
  if ((g.n + 127) / 128 > 0x7fffffff / 1024 || (g.m + 15) / 16 > 65535 * 8) return -2;
  I8Out o{};
  o.m = g.m;
  o.n = g.n;
  o.act = g.act;
  o.fp32 = g.fp32;
  o.ldo = g.ldo;
  o.out = g.out;
  o.sx = g.x_scale;
  o.sw = g.w_scale;
  o.bias = reinterpret_cast<const __nv_bfloat16*>(g.bias);
  o.residual = reinterpret_cast<const __nv_bfloat16*>(g.residual);
  return g.gated ? launch_i8<true>(g, o) : launch_i8<false>(g, o);
}

// Rows brought into 8 bits (null: they are), and their product.
extern "C" int nkb_linear_i8(const void* rows, const void* gemm) {
  if (rows) {
    const int rc = nkb_quant_rows(rows);
    if (rc) return rc;
  }
  return nkb_gemm_i8(gemm);
}
