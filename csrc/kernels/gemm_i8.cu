// Products of rows and weights in 8-bit whole numbers: y[m, n] = sx[m] * sw[n] * sum_k x[m, k] w[n, k], both operands K-major.
//
// The sums are whole numbers of 32 bits (at most 127 * 127 * k, so k is up to 133144), exact whatever their order; the only roundings are
// those of the epilogue: sum -> fp32, times sx, times sw, + bias, + residual, -> bf16.  So every variant below gives the same bits.
//
// Two kernels:
//   pairs  D[tokens, features] on CTA pairs (tcgen05.mma.cta_group::2.kind::i8, tiles of 256 tokens by up to 256 features), for prompts;
//          see gemm_2cta.cu for the scheme, which this one shares: a slab is 128 bytes of k, 64 bf16 there and 128 numbers here.
//   swap   D[features, tokens] for few tokens: 128 features fill the M side, up to 128 tokens the narrow one.  One tile per CTA and several CTAs per SM, so
//          that one's start and end lie under another's loads; k may be divided among the CTAs of a cluster, whose sums are joined through distributed
//          shared memory, or left as partial sums.
#include <stdlib.h>
#include "api.h"
#include "gemm_tcgen05.cuh"
#include "i8_args.h"

namespace nkb {

constexpr int kI8Slab = 128;                       // bytes (numbers) of k per stage: one swizzled row
constexpr int kI8ATile = 128 * kI8Slab;            // 16 KB
constexpr int kI8MaxK = 133144;                    // 127 * 127 * k < 2^31

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
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

struct I8Args {               // <= 128 bytes (see GemmArgs)
  int m, n, k;                // tokens, features
  int kb_total, stages;
  int splits, kb_per_split;
  int gate_off;               // row offset of the up half of w
  int act;
  int fp32;
  int join;                   // swap: the CTAs of a cluster (as many as splits) join their sums; otherwise splits leave partial sums
  int static_w;
  int tiles_m, tiles_n, tile_n, group_m;   // pairs
  long long ldo, split_stride;
  void* out;
  const float *sx, *sw;
  const __nv_bfloat16 *bias, *residual;
  int* status;
};
static_assert(sizeof(I8Args) <= 128, "I8Args grew past the fast kernel-parameter size");

__device__ __forceinline__ float gate_act(float g, int act) { return act ? gelu_tanh_f(g) : silu_f(g); }

// ------------------------------------------------------------------------------------------------ swap
struct I8Ctrl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t done;
  uint32_t tmem_base;
  int abort;
};

// Four finished features (whole sums s, up half u) of one token, from feature f on.
template <bool GATED>
__device__ __forceinline__ void i8_store4(const I8Args& a, int split, int tok, int f, const int4& s, const int4& u) {
  const float sx = a.sx[tok];
  const int sv[4] = {s.x, s.y, s.z, s.w}, uv[4] = {u.x, u.y, u.z, u.w};
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int fj = min(f + j, a.n - 1);
    y[j] = float(sv[j]) * sx * a.sw[fj];
    if constexpr (GATED) y[j] = gate_act(y[j], a.act) * (float(uv[j]) * sx * a.sw[a.gate_off + fj]);
    if (!GATED && a.bias && split == 0) y[j] += __bfloat162float(a.bias[fj]);
  }
  const long long at = (long long)tok * a.ldo + f;
  if (!GATED && a.residual) {
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] += __bfloat162float(a.residual[at + min(j, a.n - 1 - f)]);
  }
  if (a.fp32) {
    float* o = reinterpret_cast<float*>(a.out) + split * a.split_stride + at;
    if (f + 4 <= a.n && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
      *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f + j < a.n) o[j] = y[j];
    }
  } else {
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
    if (f + 4 <= a.n && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
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
i8_swap_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const I8Args args) {
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
        if (GATED) tma_load_2d(p + kI8ATile, &tmW, &ctrl.full[stage], kb * kI8Slab, args.gate_off + f0);
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
      bool ok = true;
      for (int i = 0; i < slabs && ok; ++i) {
        ok = mbar_wait(&ctrl.full[stage], phase, abort_flag, args.status, ERR_WAIT_SMEM_FULL);
        if (!ok) break;
        tc_fence_after();
        const uint32_t w = smem_u32(tiles + stage * kStage);
        const uint64_t dw = make_smem_desc_sw128(w, 0, 1024), du = make_smem_desc_sw128(w + kI8ATile, 0, 1024);
        const uint64_t dx = make_smem_desc_sw128(w + kW * kI8ATile, 0, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) {          // 32 numbers per instruction
          const uint32_t acc = (i > 0 || k > 0) ? 1u : 0u;
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
    const int toks = min(BN, args.m - tok0), groups = toks * 32;         // pieces of four features
    const int share = (groups + joined - 1) / joined, rank = joined > 1 ? split : 0;
    const int g1 = min(groups, (rank + 1) * share);
    for (int g = rank * share + threadIdx.x; g < g1; g += 128) {
      const int t = g >> 5, f = (g & 31) * 4;
      if (f0 + f >= args.n) continue;
      int4 s, u = make_int4(0, 0, 0, 0);
      const int* p = stg + t * 128 + f;
      if (joined > 1) {
        s = make_int4(0, 0, 0, 0);
        for (int r = 0; r < joined; ++r) {
          const int4 v = ld_cluster_v4(map_to_cta(p, r));
          s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
          if (GATED) {
            const int4 q = ld_cluster_v4(map_to_cta(p + BN * 128, r));
            u.x += q.x; u.y += q.y; u.z += q.z; u.w += q.w;
          }
        }
      } else {
        s = *reinterpret_cast<const int4*>(p);
        if (GATED) u = *reinterpret_cast<const int4*>(p + BN * 128);
      }
      i8_store4<GATED>(args, args.join ? 0 : split, tok0 + t, f0 + f, s, u);
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

struct WorkI8 {
  int tm, tn;
};
// group_m row tiles share a sweep over the column tiles so that tiles of both operands are read again from L2
__device__ __forceinline__ WorkI8 i8_work(const I8Args& a, int t) {
  const int per_group = a.group_m * a.tiles_n;
  const int gr = t / per_group, first = gr * a.group_m;
  const int gsz = min(a.tiles_m - first, a.group_m), in = t - gr * per_group;
  return {first + in % gsz, in / gsz};
}

// 32 finished columns of a row from column c on, cols_end at most; y in fp32.
template <bool GATED>
__device__ __forceinline__ void i8_store_row(const I8Args& a, int row, int c, int cols_end, float (&y)[32]) {
  const long long at = (long long)row * a.ldo + c;
  const bool whole = c + 32 <= cols_end;
  if (!GATED && a.bias) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (whole || c + j < cols_end) y[j] += __bfloat162float(a.bias[c + j]);
  }
  if (a.fp32) {
    float* o = reinterpret_cast<float*>(a.out) + at;
    if (!GATED && a.residual) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (whole || c + j < cols_end) y[j] += __bfloat162float(a.residual[at + j]);
    }
    if (whole && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        reinterpret_cast<float4*>(o)[j] = make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j < cols_end) o[j] = y[j];
    }
    return;
  }
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
  const bool r16 = !GATED && a.residual && (reinterpret_cast<uintptr_t>(a.residual + at) & 15) == 0;
  if (whole && (reinterpret_cast<uintptr_t>(o) & 15) == 0 && (GATED || !a.residual || r16)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!GATED && a.residual) {
        const uint4 rr = reinterpret_cast<const uint4*>(a.residual + at)[q];
        const uint32_t rw[4] = {rr.x, rr.y, rr.z, rr.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack_bf16x2(rw[e]);
          y[8 * q + 2 * e] += f.x;
          y[8 * q + 2 * e + 1] += f.y;
        }
      }
      reinterpret_cast<uint4*>(o)[q] = make_uint4(pack_bf16x2(y[8 * q], y[8 * q + 1]), pack_bf16x2(y[8 * q + 2], y[8 * q + 3]),
                                                  pack_bf16x2(y[8 * q + 4], y[8 * q + 5]), pack_bf16x2(y[8 * q + 6], y[8 * q + 7]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c + j < cols_end) {
        if (!GATED && a.residual) y[j] += __bfloat162float(a.residual[at + j]);
        o[j] = __float2bfloat16(y[j]);
      }
  }
}

// y[j] = v[j] * sx * sw[c + j]; columns from cols_end on read the last scale.
__device__ __forceinline__ void i8_scale_row(const uint32_t (&v)[32], float sx, const float* sw, int c, int cols_end, float (&y)[32]) {
  if (c + 32 <= cols_end && (reinterpret_cast<uintptr_t>(sw + c) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 s = __ldg(reinterpret_cast<const float4*>(sw + c) + j);
      y[4 * j] = float(int(v[4 * j])) * sx * s.x;
      y[4 * j + 1] = float(int(v[4 * j + 1])) * sx * s.y;
      y[4 * j + 2] = float(int(v[4 * j + 2])) * sx * s.z;
      y[4 * j + 3] = float(int(v[4 * j + 3])) * sx * s.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = float(int(v[j])) * sx * __ldg(sw + min(c + j, cols_end - 1));
  }
}

template <bool GATED>
__global__ void __launch_bounds__(kGemmThreads, 1)
i8_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const I8Args args) {
  extern __shared__ uint8_t smem_raw[];
  // identical layout in both CTAs: [control 1 KB][ring]
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  GemmCtrl* ctrl = reinterpret_cast<GemmCtrl*>(base);
  uint8_t* tiles = base + 1024;
  const int warp = warp_idx_uniform();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();        // 0 = issues the MMAs
  const int stages = args.stages;
  constexpr uint32_t tmem_cols = 2 * kPairTileN;
  const int tile_n = args.tile_n, half_n = tile_n / 2;     // half_n: rows of w per CTA
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
      mbar_init(&ctrl->tempty[i], 8);
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
  const int total = args.tiles_m * args.tiles_n;
  griddep_launch();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    auto w_row_of = [&](int tn) {
      return GATED ? int(rank) * args.gate_off + tn * half_n : tn * tile_n + int(rank) * half_n;
    };
    int pre = 0;
    if (args.static_w && pair < total) {
      const WorkI8 t = i8_work(args, pair);
      pre = min(stages, args.kb_total);
      if (lane == 0)
        for (int i = 0; i < pre; ++i) {
          if (rank == 0) mbar_expect_tx(&ctrl->full[i], stage_tx);
          tma_load_2d_pair(tiles + i * kPairStage + kI8ATile, &tmW, map_to_cta(&ctrl->full[i], 0), i * kI8Slab, w_row_of(t.tn));
        }
      __syncwarp();
    }
    griddep_wait();
    int stage = 0;
    uint32_t phase = 0;
    bool alive = true;
    for (int w = pair; w < total && alive; w += npairs) {
      const WorkI8 t = i8_work(args, w);
      const int x_row = t.tm * 256 + int(rank) * 128, w_row = w_row_of(t.tn);
      for (int kb = 0; kb < args.kb_total; ++kb) {
        bool ok = mbar_wait(&ctrl->empty[stage], phase ^ 1u, abort_flag, args.status, ERR_WAIT_SMEM_EMPTY);
        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        if (lane == 0) {
          const uint32_t full0 = map_to_cta(&ctrl->full[stage], 0);
          uint8_t* p = tiles + stage * kPairStage;
          const bool ahead = w == pair && kb < pre;
          if (rank == 0 && !ahead) mbar_expect_tx(&ctrl->full[stage], stage_tx);
          tma_load_2d_pair(p, &tmX, full0, kb * kI8Slab, x_row);
          if (!ahead) tma_load_2d_pair(p + kI8ATile, &tmW, full0, kb * kI8Slab, w_row);
        }
        __syncwarp();
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issuer (first CTA of the pair)
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
      for (int w = pair; w < total && ok; w += npairs) {
        ok = mbar_wait(&ctrl->tempty[acc], acc_phase ^ 1u, abort_flag, args.status, ERR_WAIT_TMEM_EMPTY);
        if (!ok) break;
        const uint32_t d0 = tmem_base + uint32_t(acc * kPairTileN);
        for (int kb = 0; kb < args.kb_total; ++kb) {
          ok = mbar_wait(&ctrl->full[stage], phase, abort_flag, args.status, ERR_WAIT_SMEM_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + uint32_t(stage) * uint32_t(kPairStage >> 4);
          const uint64_t da = d_hi | a_lo, db = d_hi | (a_lo + uint32_t(kI8ATile >> 4));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_i8_pair(d0, da + uint64_t(k * 2), db + uint64_t(k * 2), idesc, (kb > 0 || k > 0) ? 1u : 0u);
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
    // ------------------------------------------------------------------ epilogue (warps 2..5, both CTAs)
    const int quad = warp & 3;
    griddep_wait();
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int w = pair; w < total; w += npairs) {
      const WorkI8 t = i8_work(args, w);
      const int row = t.tm * 256 + int(rank) * 128 + quad * 32 + lane;
      const float sx = args.sx[min(row, args.m - 1)];
      bool ok = mbar_wait(&ctrl->tfull[acc], acc_phase, abort_flag, args.status, ERR_WAIT_TMEM_FULL);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t t0 = tmem_base + (uint32_t(quad * 32) << 16) + uint32_t(acc * kPairTileN);
      const int width = GATED ? half_n : tile_n;
      const int col0 = t.tn * width, cols_end = min(args.n, col0 + width);
#pragma unroll 1
      for (int c = 0; c < width; c += 32) {
        float y[32];
        uint32_t v[32];
        tmem_ld_32x32(t0 + c, v);
        if constexpr (GATED) {
          uint32_t u[32];
          tmem_ld_32x32(t0 + half_n + c, u);
          tmem_ld_wait();
          if (col0 + c < cols_end) {
            float up[32];
            i8_scale_row(v, sx, args.sw, col0 + c, cols_end, y);
            i8_scale_row(u, sx, args.sw + args.gate_off, col0 + c, cols_end, up);
            if (args.act) {
#pragma unroll
              for (int j = 0; j < 32; ++j) y[j] = gelu_tanh_f(y[j]) * up[j];
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) y[j] = silu_f(y[j]) * up[j];
            }
          }
        } else {
          tmem_ld_wait();
          if (col0 + c < cols_end) i8_scale_row(v, sx, args.sw, col0 + c, cols_end, y);
        }
        if (c + 32 >= width) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_cta(&ctrl->tempty[acc], 0));
        }
        if (row < args.m && col0 + c < cols_end) i8_store_row<GATED>(args, row, col0 + c, cols_end, y);
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

constexpr int kMaxDev = 64;

static int i8_maps(const NkbGemmI8& g, CUtensorMap* x, uint32_t x_box, CUtensorMap* w, uint32_t w_box) {
  const uint64_t xd[2] = {uint64_t(g.k), uint64_t(g.m)}, wd[2] = {uint64_t(g.k), uint64_t(g.gated ? 2 : 1) * uint64_t(g.n)};
  const uint64_t xs[1] = {uint64_t(g.ldx)}, ws[1] = {uint64_t(g.ldw)};
  const uint32_t xb[2] = {uint32_t(kI8Slab), x_box}, wb[2] = {uint32_t(kI8Slab), w_box};
  return encode_tmap_u8(x, g.x, 2, xd, xs, xb, 128) || encode_tmap_u8(w, g.w, 2, wd, ws, wb, 128);
}

template <int BN, bool GATED>
static int launch_swap(const NkbGemmI8& g, I8Args a, int join) {
  constexpr int kW = GATED ? 2 : 1, kStage = kW * kI8ATile + BN * kI8Slab, kStaging = kW * BN * 128 * 4;
  // two CTAs per SM at least where the staging leaves room
  int stages = (110 * 1024) / kStage;
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
                            join ? a.splits : 1, tw, tx, a);
}

template <bool GATED>
static int launch_i8_pairs(const NkbGemmI8& g, I8Args a, int tile_n) {
  a.tile_n = tile_n;
  a.tiles_m = (g.m + 255) / 256;
  a.tiles_n = GATED ? (g.n + tile_n / 2 - 1) / (tile_n / 2) : (g.n + tile_n - 1) / tile_n;
  a.group_m = 16;
  a.stages = (232448 - 2048) / kPairStage;
  const int smem = a.stages * kPairStage + 2048;
  CUtensorMap tx, tw;
  if (i8_maps(g, &tx, 128, &tw, uint32_t(tile_n / 2))) return -4;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (num_sms() / 2));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = reinterpret_cast<cudaStream_t>(g.stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static int resident[kMaxDev] = {0};
  if (resident[dev] == 0) {
    const cudaError_t e = cudaFuncSetAttribute(i8_pair_kernel<GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return int(e);
    int n = 0;
    resident[dev] = cudaOccupancyMaxActiveClusters(&n, i8_pair_kernel<GATED>, &cfg) == cudaSuccess && n > 0 ? n : num_sms() / 4;
  }
  const int total = a.tiles_m * a.tiles_n;
  cfg.gridDim = dim3(2 * unsigned(resident[dev] < total ? resident[dev] : total));
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return int(cudaLaunchKernelEx(&cfg, i8_pair_kernel<GATED>, tx, tw, a));
}

// k divided into whole slabs, none of them empty: at most `want` parts.
static void divide(I8Args& a, int want) {
  want = want < 1 ? 1 : (want > a.kb_total ? a.kb_total : want);
  a.kb_per_split = (a.kb_total + want - 1) / want;
  a.splits = (a.kb_total + a.kb_per_split - 1) / a.kb_per_split;
}

// CTAs of a cluster that share a tile's k in the swap kernel: doubled while the grid stays within two CTAs per SM and each keeps four slabs.
static int pick_join(int tiles, int kb) {
  int s = 1;
  while (s < 8 && tiles * s * 2 <= 2 * num_sms() && kb / (s * 2) >= 4) s *= 2;
  return s;
}

template <bool GATED>
static int launch_i8(const NkbGemmI8& g, const I8Args& a0) {
  I8Args a = a0;
  if (g.m > 128 && g.splits == 0) {
    divide(a, 1);
    return launch_i8_pairs<GATED>(g, a, 256);
  }
  const int bn = g.m <= 16 ? 16 : (g.m <= 32 ? 32 : (g.m <= 64 || GATED ? 64 : 128));
  const int tiles = (g.n + 127) / 128 * ((g.m + bn - 1) / bn);
  int join = 0;
  if (g.splits > 0) {
    divide(a, g.splits);
  } else {
    // (a cluster wants as many CTAs as it is launched with, and a power of two of them)
    for (int s = pick_join(tiles, a.kb_total);; s /= 2) {
      divide(a, s);
      if (a.splits == s) break;
    }
    join = a.splits > 1;
  }
  a.join = join;
  if (bn == 16) return launch_swap<16, GATED>(g, a, join);
  if (bn == 32) return launch_swap<32, GATED>(g, a, join);
  if (bn == 64) return launch_swap<64, GATED>(g, a, join);
  if constexpr (!GATED) return launch_swap<128, GATED>(g, a, join);
  return -2;
}

}  // namespace nkb

using namespace nkb;

// Splits that a product asked for `splits` of them really has.
extern "C" int nkb_gemm_i8_splits(int k, int splits) {
  I8Args a{};
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
  I8Args a{};
  a.m = g.m; a.n = g.n; a.k = g.k;
  a.kb_total = (g.k + kI8Slab - 1) / kI8Slab;
  a.gate_off = g.n;
  a.act = g.act;
  a.fp32 = g.fp32;
  a.static_w = g.static_w;
  a.ldo = g.ldo;
  a.split_stride = g.split_stride;
  a.out = g.out;
  a.sx = g.x_scale;
  a.sw = g.w_scale;
  a.bias = reinterpret_cast<const __nv_bfloat16*>(g.bias);
  a.residual = reinterpret_cast<const __nv_bfloat16*>(g.residual);
  a.status = status_word();
  return g.gated ? launch_i8<true>(g, a) : launch_i8<false>(g, a);
}
