// Gated projection of a feed-forward block, forward and backward:
//   h = act(x . Wg^T) * (x . Wu^T)                  x [N, H], Wg and Wu [F, H], h [N, F]
//   act(g) = g * sig(v): silu v = g; gelu (tanh form) v = 2 sqrt(2/pi) (g + 0.044715 g^3),
//   which is 0.5 g (1 + tanh(v / 2)) without the cancellation of 1 + tanh
// (the reference runs two cuBLAS products and its SwiGLU kernels,
// solution/kernels.py:355-446, with g and u in memory between them).
// Backward, from dh and the forward's g and u:
//   dg = dh * u * act'(g),  du = dh * act(g)        rounded to the inputs' type (tensor-core operands)
//   dx = dg . Wg + du . Wu,  dWg = dg^T . x,  dWu = du^T . x
//
// Forward (gated_fwd_kernel): both products of a tile share one accumulator: its columns
// [0, FT) are gate features, [128, 128 + FT) the same features of up, so a thread finds both
// values of a feature in its own TMEM lane and the epilogue forms h in registers; g and u never
// leave the SM unless the backward needs them. On CTA pairs (N > 128: 256 tokens x 128
// features) the pair UMMA takes half of its B rows from each CTA: the leader stages the gate
// rows, its peer the up rows. Up to 128 tokens (gated_few_kernel, gated_token_kernel) the weights'
// read is all that counts. Stages, loads (one 256-byte-row box per operand) and roles are those of the head's
// kernels (lmce_engine.cuh, lmce_bwd_pair.cuh).
//
// With training the epilogue also keeps g and u, the upper 24 bits of their fp32 values, in
// blocks of 32 tokens x 32 features laid out as the accumulator is read: for each of g and u the
// upper 16 bits [4 groups of 8 features][32 tokens][8] and the next 8 bits [2 groups of 16][32
// tokens][16], one contiguous piece of 3 KB each. That leaves an error of at most 2^-15, a
// sixteenth of fp16's 2^-11. dg and du are rounded once already, so a gradient's error is sqrt(2) times that of its
// own rounding alone; with g and u in the inputs' type it would be 1.8 times. 6 bytes per token and
// feature; an eager block keeps 8 (g, u, act(g) and h). The pieces leave by bulk stores from
// shared memory: with 16-byte stores from registers the warps waited on the SM's path to L2 (one
// B200, 8192 x 4096 x 14336 1500 us without, 1633 with register stores, 1556 with bulk stores; 2048
// x 1536 x 8960 96, 113 and 105; 4096 x 896 x 4864 63, 84 and 81).
//
// e4m3 operands (serving): the same kernel with kind::f8f6f4, K = 256 per stage in the same
// bytes; g and u are scaled by the row's and the feature's scale in the epilogue.
#pragma once

#include <cuda_fp8.h>

#include "lmce_bwd_pair.cuh"
#include "lmce_rmsnorm.cuh"

namespace lmce {

constexpr int GT_GROUP = 16;       // row blocks that share a sweep over the column blocks
// One 32 x 32 block of saved g and u: 2 KB of upper halves and 1 KB of third bytes for each.
constexpr int GATED_SAVE_HI = 32 * 32 * 2;
constexpr int GATED_SAVE_LO = 32 * 32;
constexpr int GATED_SAVE_PART = GATED_SAVE_HI + GATED_SAVE_LO;
constexpr int GATED_SAVE_BLOCK = 2 * GATED_SAVE_PART;

enum : int { ACT_SILU = 0, ACT_GELU_TANH = 1 };

struct GatedParams {
  int N, H, F;
  int act;
  int b_rows;            // up to 128 tokens: token rows per stage, N rounded up to 16
  uint8_t* saved;        // SAVE: blocks of GATED_SAVE_BLOCK bytes
  const float* x_scale;  // e4m3: [N]
  const float* g_scale;  // e4m3: [F]
  const float* u_scale;
  int* err;
  unsigned long long timeout_ns;
};

// ------------------------------------------------------------- activation ---

// sig(v) = 1 / (1 + exp(-v)); exp overflows to infinity and sig to 0 far out.
__device__ __forceinline__ float act_sigmoid(float g, int act) {
  const float v = act == ACT_SILU ? g : 1.5957691216057308f * fmaf(0.044715f * g * g, g, g);
  return rcp_approx(1.0f + ex2_approx(-LOG2E * v));
}

__device__ __forceinline__ float act_value(float g, int act) { return g * act_sigmoid(g, act); }

// act(g) and act'(g) = sig + g sig (1 - sig) v'. With a = g sig, a - a sig in one rounding keeps
// the small a (1 - sig) of large g, and is 0 once sig is 1.
__device__ __forceinline__ void act_both(float g, int act, float& a, float& da) {
  const float s = act_sigmoid(g, act);
  a = g * s;
  const float t = fmaf(-a, s, a);
  if (act == ACT_SILU) {
    da = t + s;
  } else {
    const float dv = 1.5957691216057308f * fmaf(0.134145f * g, g, 1.0f);
    da = t == 0.f ? s : fmaf(t, dv, s);  // far out v' may be infinite
  }
}

// One token's 32 values in a saved block's layout (`dst`: the token's first 16 bytes).
__device__ __forceinline__ void save_part(uint8_t* dst, const uint32_t (&v)[32]) {
  uint4* hi = reinterpret_cast<uint4*>(dst);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    hi[i * 32] = make_uint4(
        __byte_perm(v[8 * i], v[8 * i + 1], 0x7632), __byte_perm(v[8 * i + 2], v[8 * i + 3], 0x7632),
        __byte_perm(v[8 * i + 4], v[8 * i + 5], 0x7632), __byte_perm(v[8 * i + 6], v[8 * i + 7], 0x7632));
  uint4* lo = reinterpret_cast<uint4*>(dst + GATED_SAVE_HI);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = 16 * i + 4 * k;
      w[k] = __byte_perm(__byte_perm(v[j], v[j + 1], 0x0051), __byte_perm(v[j + 2], v[j + 3], 0x0051), 0x5410);
    }
    lo[i * 32] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The 16 values that two 16-byte pieces of upper halves and one of third bytes hold. The third
// byte stands in for the lost fourth as well: as good as random, it leaves the values without a
// bias (an error of at most 2^-15, 0.41 * 2^-15 rms), and zeros, infinities and NaNs as they were.
__device__ __forceinline__ void load_part(const uint4 (&hi)[2], const uint4& lo, float* f) {
  const uint32_t h[8] = {hi[0].x, hi[0].y, hi[0].z, hi[0].w, hi[1].x, hi[1].y, hi[1].z, hi[1].w};
  const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const uint32_t sel = ((j & 1) ? 0x3200u : 0x1000u) | ((4u + (j & 3)) * 0x11u);
    f[j] = __uint_as_float(__byte_perm(h[j >> 1], l[j >> 2], sel));
  }
}

// ------------------------------------------------------------ few tokens ---

// One token without a backward: one warp per feature reads its gate and its up row once, 16
// bytes per lane, and multiplies both with the token in fp32 (the token, a few KB, comes from
// L1). The weights' read is all that counts, and it has no pipeline to fill: 32 lanes x 2 x
// GT_UNROLL loads of 16 bytes are in flight per warp from its first instruction on. One B200,
// 16 bits: 1536 x 8960 10.5 us (floor 8.6, gated_few_kernel 13.2), 3584 x 18944 41.3 us (floor
// 42.2, 43.9). A second token costs this kernel as many instructions again (14.1 and 48.4 us)
// and the other one nothing, so it has one only. In e4m3, with twice the conversions per byte, it is
// still the faster one: 896 x 4864 4.0 us (gated_few_kernel 6.1, floor 1.4), 1536 x 8960 7.7 (8.8,
// floor 4.3), 3584 x 18944 24.9 (25.3, floor 21.1), 4096 x 14336 21.7 (23.5, floor 18.2).
constexpr int GT_WARPS = 4;
constexpr int GT_UNROLL = 4;

template <bool BF16, bool E4M3>
__device__ __forceinline__ void unpack_operand(const uint4& u, float* f) {
  if constexpr (E4M3) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const __half2_raw hr =
            __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w[i] >> (16 * k)) & 0xffffu), __NV_E4M3);
        const float2 v = __half22float2(__half2(hr));
        f[4 * i + 2 * k] = v.x;
        f[4 * i + 2 * k + 1] = v.y;
      }
    }
  } else {
    unpack8<BF16>(u, f);
  }
}

// vec: 16-byte units per row.
template <bool BF16, bool E4M3>
__global__ void __launch_bounds__(32 * GT_WARPS)
    gated_token_kernel(const uint4* __restrict__ x, const uint4* __restrict__ wg, const uint4* __restrict__ wu,
                       int vec, const GatedParams p, uint16_t* __restrict__ h) {
  constexpr int PER = E4M3 ? 16 : 8;
  const int lane = threadIdx.x & 31;
  const int f = blockIdx.x * GT_WARPS + threadIdx.x / 32;
  if (f >= p.F) return;
  const uint4* rg = wg + static_cast<size_t>(f) * vec;
  const uint4* ru = wu + static_cast<size_t>(f) * vec;
  float g = 0.f, u = 0.f;
  for (int c0 = lane; c0 < vec; c0 += 32 * GT_UNROLL) {
    uint4 a[GT_UNROLL], b[GT_UNROLL];
#pragma unroll
    for (int i = 0; i < GT_UNROLL; ++i) {
      const int c = c0 + 32 * i;
      a[i] = b[i] = make_uint4(0u, 0u, 0u, 0u);
      if (c < vec) {
        a[i] = __ldcs(rg + c);
        b[i] = __ldcs(ru + c);
      }
    }
#pragma unroll
    for (int i = 0; i < GT_UNROLL; ++i) {
      const int c = c0 + 32 * i;
      if (c >= vec) break;
      float fa[PER], fb[PER], fx[PER];
      unpack_operand<BF16, E4M3>(a[i], fa);
      unpack_operand<BF16, E4M3>(b[i], fb);
      unpack_operand<BF16, E4M3>(__ldg(x + c), fx);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        g = fmaf(fx[j], fa[j], g);
        u = fmaf(fx[j], fb[j], u);
      }
    }
  }
  g = warp_sum(g);
  u = warp_sum(u);
  if (lane != 0) return;
  if constexpr (E4M3) {
    const float xs = *p.x_scale;
    g *= xs * p.g_scale[f];
    u *= xs * p.u_scale[f];
  }
  h[f] = static_cast<uint16_t>(pack2<BF16>(act_value(g, p.act) * u, 0.f) & 0xffffu);
}

// ------------------------------------------------------------ tile orders ---

// Row blocks in groups of GT_GROUP, column blocks across, row blocks of the group fastest: the
// CTAs at work at one time cover a patch of the output, so each operand panel that L2 holds serves
// several of them. Groups of 4, 8, 16 and 32, one B200, interleaved: 8192 x 4096 x 14336 backward
// 3290, 3200, 3150 and 3390 us; 16384 x 1536 x 8960 forward 714 (8), 668 (16), 690 us (32).
__device__ __forceinline__ void grouped_tile(int u, int num_m, int num_n, int& m, int& n) {
  const int per = GT_GROUP * num_n;
  const int grp = u / per, m0 = grp * GT_GROUP;
  const int gm = min(GT_GROUP, num_m - m0);
  const int r = u - grp * per;
  n = r / gm;
  m = m0 + (r - n * gm);
}

constexpr int GP_TOK = 256;  // pair tile: tokens
constexpr int GP_FT = 128;   // pair tile: features

// ---------------------------------------------------------------- forward ---

// BF16: the type of 16-bit operands and of h. The stage rows are 256 bytes whatever the type.
template <bool BF16, bool E4M3, bool SAVE>
__global__ void __launch_bounds__(P_THREADS, 1)
    gated_fwd_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_g,
                     const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_h,
                     const GatedParams p) {
  constexpr int KB = E4M3 ? 2 * P_KB : P_KB;  // K per stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + P_STAGES * P_STAGE_BYTES);
  uint64_t* empty_bar = full_bar + P_STAGES;
  uint64_t* tfull_bar = empty_bar + P_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int unit0 = static_cast<int>(cluster_id_x()), step = static_cast<int>(cluster_count_x());
  const int num_m = (p.N + GP_TOK - 1) / GP_TOK, num_n = (p.F + GP_FT - 1) / GP_FT;
  const int total = num_m * num_n;
  const int nkb = (p.H + KB - 1) / KB;

  if (threadIdx.x == 0) {
    for (int s = 0; s < P_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 2 * P_EPI);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_g);
    tma_prefetch_desc(&map_u);
    tma_prefetch_desc(&map_h);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const uint64_t tlimit = p.timeout_ns;

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer ---
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full_leader = mapa_shared(smem_u32(full_bar), 0);
      const CUtensorMap* map_b = rank == 0 ? &map_g : &map_u;
      for (int u = unit0; ok && u < total; u += step) {
        int m, n;
        grouped_tile(u, num_m, num_n, m, n);
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, tlimit)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * P_STAGE_BYTES;
          uint8_t* sb = sa + P_A_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * P_STAGE_BYTES);
          const uint32_t fb = full_leader + 8u * stage;
          tma_load_3d_pair(sa, &map_x, fb, 0, m * GP_TOK + BM * static_cast<int>(rank), 2 * kb);
          tma_load_3d_pair(sb, map_b, fb, 0, n * GP_FT, 2 * kb);
          ++issued;
          if (++stage == P_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        raise_error(p.err, ERR_TIMEOUT);
        *abort_flag = 1;
        if (rank == 0) {
          const int outstanding = issued < P_STAGES ? issued : P_STAGES;
          for (int i = 1; i <= outstanding; ++i) {
            int s = stage - i;
            uint32_t ph = phase;
            if (s < 0) {
              s += P_STAGES;
              ph ^= 1u;
            }
            volatile int no_abort = 0;
            mbar_wait(&full_bar[s], ph, &no_abort, tlimit);
          }
        }
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------- UMMA issuer ---
    if (lane == 0 && rank == 0) {
      // kind::f8f6f4's e4m3 has the format code that kind::f16 gives to f16
      constexpr uint32_t idesc = make_idesc_f16(BF16 && !E4M3, false, false, 2 * BM, 2 * GP_FT);
      const uint32_t peer_empty = mapa_shared(smem_u32(empty_bar), 1);
      const uint32_t peer_tfull = mapa_shared(smem_u32(tfull_bar), 1);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int u = unit0; ok && u < total; u += step) {
        if (!mbar_wait_cluster(&tempty_bar[acc], acc_phase ^ 1u, abort_flag, tlimit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag, tlimit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * P_STAGE_BYTES);
          const uint32_t sb = sa + P_A_BYTES;
          // eight K steps of 32 bytes
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t accumulate = (kb | k) != 0 ? 1u : 0u;
            if constexpr (E4M3)
              umma_f8_ss_pair(d_tmem, pair_operand_desc(sa, false, k), pair_operand_desc(sb, false, k), idesc,
                              accumulate);
            else
              umma_f16_ss_pair(d_tmem, pair_operand_desc(sa, false, k), pair_operand_desc(sb, false, k), idesc,
                               accumulate);
          }
          umma_commit_pair(smem_u32(&empty_bar[stage]));
          umma_commit_pair(peer_empty + 8u * stage);
          if (++stage == P_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair(smem_u32(&tfull_bar[acc]));
        umma_commit_pair(peer_tfull + 8u * acc);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) {
        raise_error(p.err, ERR_TIMEOUT);
        *abort_flag = 1;
      }
      umma_commit_pair(smem_u32(drain_bar));
      volatile int no_abort = 0;
      mbar_wait(drain_bar, 0, &no_abort, tlimit);
    }
  } else {
    // ---------------------------------------------------------- epilogue ---
    const int q = warp & 3;          // TMEM lane quadrant
    const int ch = (warp - 2) >> 2;  // half of the tile's features this warp handles
    uint8_t* xstage = smem + P_STAGES * P_STAGE_BYTES + 1024 + (warp - 2) * P_SLICE_BYTES;
    const uint32_t lane_base = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t leader_tempty = mapa_shared(smem_u32(tempty_bar), 0);
    const int fblocks = p.F / 32;
    int acc = 0, half = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int u = unit0; u < total; u += step) {
      int m, n;
      grouped_tile(u, num_m, num_n, m, n);
      const int row0 = m * GP_TOK + BM * static_cast<int>(rank) + q * 32;  // this warp's first token
      float xs = 0.f;
      if constexpr (E4M3) xs = row0 + lane < p.N ? p.x_scale[row0 + lane] : 0.f;
      if (!mbar_wait(&tfull_bar[acc], acc_phase, abort_flag, tlimit)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + lane_base + static_cast<uint32_t>(acc * BN);
#pragma unroll 1
      for (int c = ch * (GP_FT / 64); c < (ch + 1) * (GP_FT / 64); ++c) {
        const int f0 = n * GP_FT + c * 32;
        uint32_t rg[32], ru[32];
        __syncwarp();
        tmem_ld_32x32b_x32(taddr + c * 32, rg);
        tmem_ld_32x32b_x32(taddr + 128 + c * 32, ru);
        tmem_ld_wait(rg);
        tmem_ld_wait(ru);
        if (f0 >= p.F || row0 >= p.N) continue;  // F is a multiple of 64: a chunk lies wholly inside or past it
        if constexpr (E4M3) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p.g_scale + f0) + j);
            const float4 b = __ldg(reinterpret_cast<const float4*>(p.u_scale + f0) + j);
            const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              rg[4 * j + i] = __float_as_uint(__uint_as_float(rg[4 * j + i]) * xs * av[i]);
              ru[4 * j + i] = __float_as_uint(__uint_as_float(ru[4 * j + i]) * xs * bv[i]);
            }
          }
        }
        // What leaves goes through two 2 KB halves of the warp's slice in turn, each written once the
        // store of two before has read it.
        const auto next_half = [&]() {
          uint8_t* box = xstage + half * 2048;
          half ^= 1;
          if (lane == 0) bulk_wait_read_1();
          __syncwarp();
          return box;
        };
        const auto written = [&]() {
          fence_async_shared();
          __syncwarp();
          return lane == 0;
        };
        float v[32];
        if constexpr (SAVE) {
          // g's 3 KB, then u's, through the slice (two 2 KB halves in turn, which waits less at each
          // step, is as fast for few stages and 1-4% slower for many)
          uint8_t* blk = p.saved + (static_cast<size_t>(row0 / 32) * fblocks + f0 / 32) * GATED_SAVE_BLOCK;
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
          save_part(xstage + lane * 16, rg);
          if (written()) {
            bulk_store(blk, xstage, GATED_SAVE_PART);
            bulk_commit_group();
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = act_value(__uint_as_float(rg[j]), p.act) * __uint_as_float(ru[j]);
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
          save_part(xstage + lane * 16, ru);
          if (written()) {
            bulk_store(blk + GATED_SAVE_PART, xstage, GATED_SAVE_PART);
            bulk_commit_group();
            bulk_wait_read_all();
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = act_value(__uint_as_float(rg[j]), p.act) * __uint_as_float(ru[j]);
        }
        // the warp's 32 tokens x 32 features of h, a 64-byte-swizzled box; tokens past N are clipped
        uint8_t* box = next_half();
        uint4* row = reinterpret_cast<uint4*>(box + lane * 64);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          row[i ^ ((lane >> 1) & 3)] =
              make_uint4(pack2<BF16>(v[8 * i], v[8 * i + 1]), pack2<BF16>(v[8 * i + 2], v[8 * i + 3]),
                         pack2<BF16>(v[8 * i + 4], v[8 * i + 5]), pack2<BF16>(v[8 * i + 6], v[8 * i + 7]));
        if (written()) {
          tma_store_2d(&map_h, box, f0, row0);
          bulk_commit_group();
        }
      }
      tc_fence_before();
      mbar_arrive_cluster(leader_tempty + 8u * acc);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (lane == 0) bulk_wait_all();
    if (!ok) {
      raise_error(p.err, ERR_TIMEOUT);
      *abort_flag = 1;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------ forward, up to 128 tokens ---

// One CTA per 64 features and all tokens: here the weights' read is all that counts, so they are
// the A operand (64 gate rows and 64 up rows, M = 128) and the tokens the narrow B operand
// (N = b_rows, the tokens rounded up to 16). With the tokens as A (M = 128 whatever their
// number, one UMMA of N = 64 per projection) the UMMAs themselves read 6 KB of shared memory per
// 4 KB of weights and held every SM to 21 bytes of weights per clock (one B200: 3584 x 18944 in
// 16 bits 47 us, 4096 x 14336, whose 224 tiles leave 72 SMs idle in the second round, 53 us).
// Boxes end with the tokens there are: one whose rows lie mostly outside its tensor arrives
// later than one that is read (72 us for 1 token in 128-row boxes against 50 us for 64).
// A stage is K = 128 (256 for e4m3): per 128-byte column block the gate rows and the up rows
// follow one another, four 8 KB boxes. Lanes 0-63 of the accumulator are gate features, 64-127
// the same features of up: the up warps hand their values over through shared memory.
// Against the pairs at the border (bf16): 128 tokens here 15.4 us at 1536 x 8960 and 50.4 us at
// 4096 x 14336, 129 tokens there 16.4 and 64.4 us.
constexpr int GF_FT = 64;
constexpr int GF_W_BYTES = 2 * GF_FT * 2 * 128;          // 32 KB of weights per stage
constexpr int GF_MAX_STAGES = 5;
constexpr int GF_STAGE_AREA = P_STAGES * P_STAGE_BYTES;  // shared memory for stages
constexpr int GF_XCH_PITCH = 17;                         // floats per feature of a handed-over block

template <bool BF16, bool E4M3, bool SAVE>
__global__ void __launch_bounds__(P_THREADS, 1)
    gated_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_g,
                     const __grid_constant__ CUtensorMap map_u, uint16_t* __restrict__ h, const GatedParams p) {
  constexpr int KB = E4M3 ? 2 * P_KB : P_KB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = GF_W_BYTES + p.b_rows * 256;
  const int stages = min(GF_MAX_STAGES, GF_STAGE_AREA / stage_bytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + GF_STAGE_AREA);
  uint64_t* empty_bar = full_bar + GF_MAX_STAGES;
  uint64_t* tfull_bar = empty_bar + GF_MAX_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x & 31;
  const int total = p.F / GF_FT;
  const int nkb = (p.H + KB - 1) / KB;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], P_EPI);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_g);
    tma_prefetch_desc(&map_u);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const uint64_t tlimit = p.timeout_ns;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int n = blockIdx.x; ok && n < total; n += gridDim.x) {
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, tlimit)) {
            ok = false;
            break;
          }
          uint8_t* sw = smem + stage * stage_bytes;
          mbar_arrive_expect_tx(&full_bar[stage], stage_bytes);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            tma_load_3d(sw + z * (GF_W_BYTES / 2), &map_g, &full_bar[stage], 0, n * GF_FT, 2 * kb + z);
            tma_load_3d(sw + z * (GF_W_BYTES / 2) + GF_W_BYTES / 4, &map_u, &full_bar[stage], 0, n * GF_FT,
                        2 * kb + z);
          }
          tma_load_3d(sw + GF_W_BYTES, &map_x, &full_bar[stage], 0, 0, 2 * kb);
          ++issued;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        raise_error(p.err, ERR_TIMEOUT);
        *abort_flag = 1;
        const int outstanding = issued < stages ? issued : stages;
        for (int i = 1; i <= outstanding; ++i) {
          int s = stage - i;
          uint32_t ph = phase;
          if (s < 0) {
            s += stages;
            ph ^= 1u;
          }
          volatile int no_abort = 0;
          mbar_wait(&full_bar[s], ph, &no_abort, tlimit);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // N of the instruction is the launch's: uniform for all threads, computed once
      const uint32_t idesc = make_idesc_f16(BF16 && !E4M3, false, false, BM, p.b_rows);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int n = blockIdx.x; ok && n < total; n += gridDim.x) {
        if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, abort_flag, tlimit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * 128);
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag, tlimit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sw = smem_u32(smem + stage * stage_bytes), sx = sw + GF_W_BYTES;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t step = (k & 3) * (UMMA_K * 2);
            const uint64_t a = smem_desc_sw128(sw + (k >> 2) * (GF_W_BYTES / 2) + step, 16, 1024);
            const uint64_t b = smem_desc_sw128(sx + (k >> 2) * (p.b_rows * 128) + step, 16, 1024);
            if constexpr (E4M3)
              umma_f8_ss(d_tmem, a, b, idesc, (kb | k) != 0 ? 1u : 0u);
            else
              umma_f16_ss(d_tmem, a, b, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          umma_commit(&empty_bar[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(&tfull_bar[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) {
        raise_error(p.err, ERR_TIMEOUT);
        *abort_flag = 1;
      }
      umma_commit(drain_bar);
      volatile int no_abort = 0;
      mbar_wait(drain_bar, 0, &no_abort, tlimit);
    }
  } else {
    // Two groups of four warps take the 32-token column chunks in turn; in each, warps of lane
    // quadrants 0 and 1 hold gate, 2 and 3 up.
    const int q = warp & 3, grp = (warp - 2) >> 2;
    const bool is_gate = q < 2;
    float* blocks = reinterpret_cast<float*>(smem + GF_STAGE_AREA + 1024) + grp * (2 * GF_FT * GF_XCH_PITCH) +
                    ((q & 1) * 32 + lane) * GF_XCH_PITCH;
    float* give = blocks + (is_gate ? 0 : GF_FT * GF_XCH_PITCH);
    const float* take = blocks + (is_gate ? GF_FT * GF_XCH_PITCH : 0);
    const uint32_t lane_base = static_cast<uint32_t>(q * 32) << 16;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int n = blockIdx.x; n < total; n += gridDim.x) {
      const int f = n * GF_FT + (q & 1) * 32 + lane;
      float scale = 1.f;
      if constexpr (E4M3) scale = is_gate ? p.g_scale[f] : p.u_scale[f];
      if (!mbar_wait(&tfull_bar[acc], acc_phase, abort_flag, tlimit)) ok = false;
      // the four warps of a group leave the loop together: the barriers below count all of them
      if (!(grp == 0 ? named_bar_all<1, 128>(ok) : named_bar_all<2, 128>(ok))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + lane_base + static_cast<uint32_t>(acc * 128);
      for (int t0 = grp * 32; t0 < p.N; t0 += 64) {
        uint32_t raw[32];
        __syncwarp();
        tmem_ld_32x32b_x32(taddr + t0, raw);
        tmem_ld_wait(raw);
        float own[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          own[j] = __uint_as_float(is_gate ? raw[j] : raw[16 + j]) * scale;
          give[j] = __uint_as_float(is_gate ? raw[16 + j] : raw[j]) * scale;
        }
        grp == 0 ? named_bar<1, 128>() : named_bar<2, 128>();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = t0 + j + (is_gate ? 0 : 16);
          if (t < p.N) {
            const float other = take[j];
            float g = is_gate ? own[j] : other, u = is_gate ? other : own[j];
            if constexpr (E4M3) {
              const float xs = __ldg(p.x_scale + t);
              g *= xs;
              u *= xs;
            }
            if constexpr (SAVE) {
              uint8_t* blk = p.saved + (static_cast<size_t>(t / 32) * (p.F / 32) + f / 32) * GATED_SAVE_BLOCK;
              const int fl = f % 32, tl = t % 32;
              const int hi = fl / 8 * 512 + tl * 16 + fl % 8 * 2;
              const int lo = GATED_SAVE_HI + fl / 16 * 512 + tl * 16 + fl % 16;
              const uint32_t gb = __float_as_uint(g), ub = __float_as_uint(u);
              *reinterpret_cast<uint16_t*>(blk + hi) = static_cast<uint16_t>(gb >> 16);
              *reinterpret_cast<uint16_t*>(blk + GATED_SAVE_PART + hi) = static_cast<uint16_t>(ub >> 16);
              blk[lo] = static_cast<uint8_t>(gb >> 8);
              blk[GATED_SAVE_PART + lo] = static_cast<uint8_t>(ub >> 8);
            }
            h[static_cast<size_t>(t) * p.F + f] =
                static_cast<uint16_t>(pack2<BF16>(act_value(g, p.act) * u, 0.f) & 0xffffu);
          }
        }
        grp == 0 ? named_bar<1, 128>() : named_bar<2, 128>();
      }
      tc_fence_before();
      mbar_arrive(&tempty_bar[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (!ok) {
      raise_error(p.err, ERR_TIMEOUT);
      *abort_flag = 1;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, BN);
  }
}

// --------------------------------------------------- backward: dg and du ---

// A block of four warps per 32 tokens x 64 features (two of the saved blocks), 16 features per
// warp and one token per lane: g and u arrive as they were stored (512 contiguous bytes per
// load); dh and the results pass through shared memory, 128 contiguous bytes per token in global
// memory and a 144-byte pitch here (conflict-free by row and by column). Memory-bound, 12 bytes
// per element. The next tile's loads are in flight while one is computed and written.
constexpr int GATED_DACT_THREADS = 128;
template <bool BF16, int ACT>
__global__ void __launch_bounds__(GATED_DACT_THREADS, 5)
    gated_dact_kernel(const uint8_t* __restrict__ saved, const uint4* __restrict__ dh, int n, int f,
                      uint4* __restrict__ dg, uint4* __restrict__ du) {
  __shared__ uint4 st[2][32][9];  // dh, then dg; du
  constexpr int PART = GATED_SAVE_PART / 16;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int tf = f / 64, vec = f / 8;
  const long long tiles = static_cast<long long>((n + 31) / 32) * tf;
  const int r0 = threadIdx.x >> 3, c = threadIdx.x & 7;  // global accesses: rows r0 and r0 + 16
  uint4 gh[2], uh[2], gl, ul, d0, d1;
  const auto load = [&](long long b) {
    const int rb = static_cast<int>(b / tf), cb = static_cast<int>(b - static_cast<long long>(rb) * tf);
    const uint8_t* blk = saved + (static_cast<long long>(rb) * (f / 32) + cb * 2 + (warp >> 1)) * GATED_SAVE_BLOCK;
    const uint4* hi = reinterpret_cast<const uint4*>(blk) + (warp & 1) * 64 + lane;
    const uint4* lo = reinterpret_cast<const uint4*>(blk + GATED_SAVE_HI) + (warp & 1) * 32 + lane;
    const long long at = (static_cast<long long>(rb) * 32 + r0) * vec + cb * 8 + c;
    d0 = d1 = make_uint4(0u, 0u, 0u, 0u);
    if (rb * 32 + r0 < n) d0 = __ldcs(dh + at);
    if (rb * 32 + r0 + 16 < n) d1 = __ldcs(dh + at + 16ll * vec);
    gh[0] = __ldcs(hi);
    gh[1] = __ldcs(hi + 32);
    gl = __ldcs(lo);
    uh[0] = __ldcs(hi + PART);
    uh[1] = __ldcs(hi + PART + 32);
    ul = __ldcs(lo + PART);
  };
  long long b = blockIdx.x;
  if (b < tiles) load(b);
  for (; b < tiles; b += gridDim.x) {
    const int rb = static_cast<int>(b / tf), cb = static_cast<int>(b - static_cast<long long>(rb) * tf);
    const long long at = (static_cast<long long>(rb) * 32 + r0) * vec + cb * 8 + c;
    const bool live0 = rb * 32 + r0 < n, live1 = rb * 32 + r0 + 16 < n;
    st[0][r0][c] = d0;
    st[0][r0 + 16][c] = d1;
    __syncthreads();
    float d[16], e[16], g[16], u[16];
    uint4* own0 = &st[0][lane][warp * 2];
    uint4* own1 = &st[1][lane][warp * 2];
    unpack8<BF16>(own0[0], d);
    unpack8<BF16>(own0[1], d + 8);
    load_part(gh, gl, g);
    load_part(uh, ul, u);
    if (b + gridDim.x < tiles) load(b + gridDim.x);  // in flight while this tile is computed and written
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float a, da;
      act_both(g[j], ACT, a, da);
      e[j] = d[j] * a;
      d[j] = d[j] * u[j] * da;
    }
    own0[0] = pack8<BF16>(d);
    own0[1] = pack8<BF16>(d + 8);
    own1[0] = pack8<BF16>(e);
    own1[1] = pack8<BF16>(e + 8);
    __syncthreads();
    if (live0) {
      dg[at] = st[0][r0][c];
      du[at] = st[1][r0][c];
    }
    if (live1) {
      dg[at + 16ll * vec] = st[0][r0 + 16][c];
      du[at + 16ll * vec] = st[1][r0 + 16][c];
    }
    __syncthreads();
  }
}

// ------------------------------------------------ backward: the products ---

// One launch for dx, dWg and dWu on CTA pairs. A unit is a 256 x 256 output tile with a range
// of K stages:
//   DX  256 tokens x 256 hidden, K over the gate features and then the up features (A = dg or
//       du, K-major; B = the weight, MN-major); `splits` units share a tile when there are few
//       tiles, each leaving an fp32 partial that gated_dx_sum_kernel adds in order
//   DW  256 features x 256 hidden of one weight, K over the tokens (both operands MN-major)
// DX units are the longer ones and come first; the pairs that get one DX unit less than the
// others take that many stages' worth of DW units before the rest is dealt out in turn. The
// assignment is a function of the sizes alone: no counters, the same sums every time.
constexpr int GATED_UNIT_STAGES = 5;  // a unit's epilogue takes about as long as five stages

struct GatedBwdParams {
  int N, H, F;
  int n_dx, splits, dx_stages;   // DX units (tiles x splits), splits per tile, K stages of a whole tile
  int n_dw, dw_first;            // DW units; first weight wanted (0 gate, 1 up)
  int rows_pad;                  // rows of one split's partial
  int* err;
  unsigned long long timeout_ns;
};

struct GatedUnits {
  int pair, pairs, n_dx, n_dw;
  int extra, extra_step, extra_at;   // DW units this pair takes ahead of the rest
  int common;                        // first DW unit of the common part
  int phase, next;

  __device__ __forceinline__ void init(const GatedBwdParams& p, int pair_, int pairs_) {
    pair = pair_;
    pairs = pairs_;
    n_dx = p.n_dx;
    n_dw = p.n_dw;
    const int heavy = n_dx % pairs;
    const int light = heavy ? pairs - heavy : 0;
    const int lx = max(GATED_UNIT_STAGES, (p.dx_stages + p.splits - 1) / p.splits);
    const int ld = max(GATED_UNIT_STAGES, (p.N + P_KB - 1) / P_KB);
    const int ahead = light ? lx / ld : 0;
    common = static_cast<int>(min(static_cast<long long>(n_dw), static_cast<long long>(light) * ahead));
    extra = pair >= heavy && light ? ahead : 0;
    extra_step = light;
    extra_at = pair - heavy;
    phase = 0;
    next = pair;
  }

  // The next unit: a DX unit's index, or n_dx + a DW unit's index; -1 at the end.
  __device__ __forceinline__ int get() {
    if (phase == 0) {
      if (next < n_dx) {
        const int u = next;
        next += pairs;
        return u;
      }
      phase = 1;
    }
    if (phase == 1) {
      if (extra > 0 && extra_at < common) {
        const int u = extra_at;
        extra_at += extra_step;
        --extra;
        return n_dx + u;
      }
      phase = 2;
      next = common + pair;
    }
    if (next >= n_dw) return -1;
    const int u = next;
    next += pairs;
    return n_dx + u;
  }
};

struct GatedTile {
  bool dx;
  int which;        // DW: 0 gate, 1 up
  int m, n;         // row block, column block
  int split;
  int k0, k1;       // stages

  __device__ __forceinline__ void decode(const GatedBwdParams& p, int u) {
    const int nh = (p.H + 255) / 256;
    dx = u < p.n_dx;
    which = 0;
    split = 0;
    k0 = 0;
    if (dx) {
      const int tiles = p.n_dx / p.splits;
      split = u / tiles;
      grouped_tile(u - split * tiles, (p.N + 255) / 256, nh, m, n);
      k0 = static_cast<int>(static_cast<long long>(split) * p.dx_stages / p.splits);
      k1 = static_cast<int>(static_cast<long long>(split + 1) * p.dx_stages / p.splits);
    } else {
      const int per = nh * ((p.F + 255) / 256);
      int i = u - p.n_dx;
      which = p.dw_first + i / per;
      i %= per;
      m = i / nh;
      n = i - m * nh;
      k1 = (p.N + P_KB - 1) / P_KB;
    }
  }
};

template <bool BF16>
__global__ void __launch_bounds__(P_THREADS, 1)
    gated_bwd_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_wg,
                     const __grid_constant__ CUtensorMap map_wu, const __grid_constant__ CUtensorMap map_dg,
                     const __grid_constant__ CUtensorMap map_du, const __grid_constant__ CUtensorMap map_dx,
                     const __grid_constant__ CUtensorMap map_dwg, const __grid_constant__ CUtensorMap map_dwu,
                     const GatedBwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + P_STAGES * P_STAGE_BYTES);
  uint64_t* empty_bar = full_bar + P_STAGES;
  uint64_t* tfull_bar = empty_bar + P_STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = static_cast<int>(cluster_id_x()), pairs = static_cast<int>(cluster_count_x());
  const int fstages = (p.F + P_KB - 1) / P_KB;  // stages of one weight's features

  if (threadIdx.x == 0) {
    for (int s = 0; s < P_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 2 * P_EPI);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const uint64_t tlimit = p.timeout_ns;
  GatedUnits units;
  units.init(p, pair, pairs);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full_leader = mapa_shared(smem_u32(full_bar), 0);
      const int r = static_cast<int>(rank);
      for (int u = units.get(); ok && u >= 0; u = units.get()) {
        GatedTile t;
        t.decode(p, u);
        const CUtensorMap* dw_a = t.which ? &map_du : &map_dg;
        for (int kb = t.k0; kb < t.k1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, tlimit)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * P_STAGE_BYTES;
          uint8_t* sb = sa + P_A_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * P_STAGE_BYTES);
          const uint32_t fb = full_leader + 8u * stage;
          const int nblk = (t.n * 256 + BM * r) / 64;
          if (t.dx) {
            const bool up = kb >= fstages;
            const int k = up ? kb - fstages : kb;
            tma_load_3d_pair(sa, up ? &map_du : &map_dg, fb, 0, t.m * 256 + BM * r, 2 * k);
            tma_load_3d_pair(sb, up ? &map_wu : &map_wg, fb, 0, k * P_KB, nblk);
          } else {
            tma_load_3d_pair(sa, dw_a, fb, 0, kb * P_KB, (t.m * 256 + BM * r) / 64);
            tma_load_3d_pair(sb, &map_x, fb, 0, kb * P_KB, nblk);
          }
          ++issued;
          if (++stage == P_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        raise_error(p.err, ERR_TIMEOUT);
        *abort_flag = 1;
        if (rank == 0) {
          const int outstanding = issued < P_STAGES ? issued : P_STAGES;
          for (int i = 1; i <= outstanding; ++i) {
            int s = stage - i;
            uint32_t ph = phase;
            if (s < 0) {
              s += P_STAGES;
              ph ^= 1u;
            }
            volatile int no_abort = 0;
            mbar_wait(&full_bar[s], ph, &no_abort, tlimit);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t peer_empty = mapa_shared(smem_u32(empty_bar), 1);
      const uint32_t peer_tfull = mapa_shared(smem_u32(tfull_bar), 1);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      long long waited = 0;
      for (int u = units.get(); u >= 0; u = units.get()) {
        GatedTile t;
        t.decode(p, u);
        if (!mbar_wait_cluster(&tempty_bar[acc], acc_phase ^ 1u, abort_flag, tlimit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        ok = t.dx ? mma_tile_pair<BF16, false, true, BN>(smem, full_bar, empty_bar, peer_empty, t.k1 - t.k0, d_tmem,
                                                         stage, phase, abort_flag, tlimit, waited)
                  : mma_tile_pair<BF16, true, true, BN>(smem, full_bar, empty_bar, peer_empty, t.k1 - t.k0, d_tmem,
                                                        stage, phase, abort_flag, tlimit, waited);
        if (!ok) break;
        umma_commit_pair(smem_u32(&tfull_bar[acc]));
        umma_commit_pair(peer_tfull + 8u * acc);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) {
        raise_error(p.err, ERR_TIMEOUT);
        *abort_flag = 1;
      }
      umma_commit_pair(smem_u32(drain_bar));
      volatile int no_abort = 0;
      mbar_wait(drain_bar, 0, &no_abort, tlimit);
    }
  } else {
    const int q = warp & 3;
    const int ch = (warp - 2) >> 2;
    uint8_t* xstage = smem + P_STAGES * P_STAGE_BYTES + 1024 + (warp - 2) * P_SLICE_BYTES;
    const uint32_t lane_base = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t leader_tempty = mapa_shared(smem_u32(tempty_bar), 0);
    int acc = 0, half = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int u = units.get(); u >= 0; u = units.get()) {
      GatedTile t;
      t.decode(p, u);
      const int row0 = t.m * 256 + BM * static_cast<int>(rank) + q * 32;
      const int rows = t.dx ? p.N : p.F;
      const CUtensorMap* map_o = t.dx ? &map_dx : t.which ? &map_dwu : &map_dwg;
      const bool partial = t.dx && p.splits > 1;
      if (!mbar_wait(&tfull_bar[acc], acc_phase, abort_flag, tlimit)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + lane_base + static_cast<uint32_t>(acc * BN);
#pragma unroll 1
      for (int c = ch * 4; c < ch * 4 + 4; ++c) {
        const int h0 = t.n * 256 + c * 32;
        uint32_t raw[32];
        __syncwarp();
        tmem_ld_32x32b_x32(taddr + c * 32, raw);
        tmem_ld_wait(raw);
        if (h0 >= p.H || row0 >= rows) continue;  // H is a multiple of 64
        if (partial) {
          // 32 x 32 fp32 in the 128-byte swizzled box layout, the whole slice
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
          uint4* sl = reinterpret_cast<uint4*>(xstage);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            sl[lane * 8 + (i ^ (lane & 7))] =
                make_uint4(raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]);
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(map_o, xstage, h0, t.split * p.rows_pad + row0);
            bulk_commit_group();
          }
          half = 0;
        } else {
          uint8_t* box = xstage + half * 2048;
          half ^= 1;
          if (lane == 0) bulk_wait_read_1();  // the box of two stores ago has left it
          __syncwarp();
          uint4* row = reinterpret_cast<uint4*>(box + lane * 64);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            row[i ^ ((lane >> 1) & 3)] = make_uint4(
                pack2<BF16>(__uint_as_float(raw[8 * i]), __uint_as_float(raw[8 * i + 1])),
                pack2<BF16>(__uint_as_float(raw[8 * i + 2]), __uint_as_float(raw[8 * i + 3])),
                pack2<BF16>(__uint_as_float(raw[8 * i + 4]), __uint_as_float(raw[8 * i + 5])),
                pack2<BF16>(__uint_as_float(raw[8 * i + 6]), __uint_as_float(raw[8 * i + 7])));
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(map_o, box, h0, row0);
            bulk_commit_group();
          }
        }
      }
      if (partial && lane == 0) bulk_wait_read_all();  // the next unit may use the slice as two boxes
      tc_fence_before();
      mbar_arrive_cluster(leader_tempty + 8u * acc);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (lane == 0) bulk_wait_all();
    if (!ok) {
      raise_error(p.err, ERR_TIMEOUT);
      *abort_flag = 1;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// dx = dtype(sum over splits of the fp32 partials, in order); rows of `vec` 4-value units.
template <bool BF16>
__global__ void gated_dx_sum_kernel(const float4* __restrict__ part, int splits, long long split_stride,
                                    long long total, uint2* __restrict__ dx) {
  for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    float4 v = __ldcs(part + i);
    for (int s = 1; s < splits; ++s) {
      const float4 w = __ldcs(part + s * split_stride + i);
      v.x += w.x;
      v.y += w.y;
      v.z += w.z;
      v.w += w.w;
    }
    dx[i] = make_uint2(pack2<BF16>(v.x, v.y), pack2<BF16>(v.z, v.w));
  }
}

}  // namespace lmce
