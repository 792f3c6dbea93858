// Residual addition with its RMSNorm, forward (16-bit or e4m3 output) and backward: what a
// decoder block runs in front of each of its projections (the reference fuses the same
// pair in rms_norm_fwd / rms_norm_bwd, solution/kernels.py:124-190).
//   s = dtype(x + residual)            the residual stream, kept in the inputs' type
//   rstd = 1 / sqrt(mean(s^2) + eps)   fp32
//   y = dtype(s * rstd * w)            one rounding
//   e4m3: scale = max|s * rstd * w| / 448 per row (1 for a row of zeros), q = e4m3(y / scale)
// Backward, with p = dy * w and n = s * rstd (both gradients of the sum are the same):
//   dx = dtype(ds + rstd * (p - n * mean(p * n))),  dw = sum over rows of dy * n
// All sums are fp32. The norm reads the rounded s, so the backward, which only has s, sees
// the forward's values exactly.
//
// Memory-bound: a row is read once into registers (VPT 16-byte vectors per thread, T
// threads per row) and leaves as s and y from there. The T threads of a row are whole warps
// (T = 32 ceil(vec / (32 VPT))), so common widths fill them (1536: 96 x 2 vectors, 3584: 224
// x 2), and a block holds R rows' groups.
#pragma once

#include <cuda_fp8.h>

#include "lmce_rmsnorm.cuh"

namespace lmce {

constexpr int AN_MAX_WARPS = 16;

struct AddNormParams {
  const uint4* x;
  const uint4* residual;  // null: s = x, not written
  const uint4* w;
  uint4* s_out;           // null without residual
  uint4* y;               // 16-bit output
  uint2* q;               // e4m3 output (8 bytes per 8 values)
  float* scale;           // e4m3: [n]
  float* rstd;            // null: not kept
  long long n;
  int vec;                // 16-byte vectors per row
  int threads;            // threads per row, a multiple of 32
  int rows;               // rows per block
  float inv_cols, eps;
};

struct AddNormBwdParams {
  const uint4* dy;        // null: zero
  const uint4* ds;        // null: zero
  const uint4* s;
  const uint4* w;
  const float* rstd;
  uint4* dx;              // null: not wanted
  float* dw_part;         // [gridDim.x][8 * vec] (null: not wanted)
  long long n;
  int vec, threads, rows;
  float inv_cols;
};

// Sum over the threads of a row, and with MAX the maximum of a second value in the same pass.
// `red` holds one pair per warp of the block. Every thread of the block calls it (the row groups
// run in step); the first __syncthreads keeps the last call's readers ahead of this one's writes.
template <bool MAX>
__device__ __forceinline__ float2 row_reduce(float sum, float top, float2* red, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if constexpr (MAX) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (warps == 1) return make_float2(sum, top);
  const int w = threadIdx.x / 32;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[w] = make_float2(sum, top);
  __syncthreads();
  const int w0 = w / warps * warps;
  float2 t = red[w0];
  for (int i = 1; i < warps; ++i) {
    t.x += red[w0 + i].x;
    if constexpr (MAX) t.y = fmaxf(t.y, red[w0 + i].y);
  }
  return t;
}

__device__ __forceinline__ uint2 pack8_e4m3(const float* f) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
}

// A bf16 row whose s w passes fp32 (1e19 and more on both sides) where s rstd w does not: its e4m3
// output once more, from s rstd w in this order. Each warp goes over the whole row, as it is held, for
// the largest magnitude: no barrier, which the block's other rows would have to join.
__device__ __forceinline__ void norm_first(const AddNormParams& p, long long row, int t, float rstd) {
  const uint4* held = (p.residual ? p.s_out : p.x) + row * p.vec;
  const auto products = [&](int c, float* v) {
    float w[8];
    unpack8<true>(held[c], v);
    unpack8<true>(__ldg(p.w + c), w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * rstd * w[j];
  };
  __syncwarp();  // a row of one warp: the other lanes' part of the sum (of more, row_reduce had a barrier)
  float top = 0.f, v[8];
#pragma unroll 1
  for (int c = threadIdx.x & 31; c < p.vec; c += 32) {
    products(c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float k = 448.0f / top;
  if (t == 0) p.scale[row] = top / 448.0f;
#pragma unroll 1
  for (int c = t; c < p.vec; c += p.threads) {
    products(c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= k;
    p.q[row * p.vec + c] = pack8_e4m3(v);
  }
}

template <bool BF16, int VPT, bool E4M3>
__global__ void __launch_bounds__(512) add_norm_kernel(const AddNormParams p) {
  __shared__ float2 red[AN_MAX_WARPS];
  const int g = threadIdx.x / p.threads, t = threadIdx.x - g * p.threads;
  const int warps = p.threads / 32;
  for (long long row0 = static_cast<long long>(blockIdx.x) * p.rows; row0 < p.n;
       row0 += static_cast<long long>(gridDim.x) * p.rows) {
    const long long row = row0 + g;
    const bool live = row < p.n;
    float f[VPT][8];
    uint4 a[VPT], b[VPT];
    float ss = 0.f, top = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * p.threads;
      if (live && c < p.vec) {
        a[i] = __ldcs(p.x + row * p.vec + c);
        if (p.residual) b[i] = __ldcs(p.residual + row * p.vec + c);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * p.threads;
      if (live && c < p.vec) {
        unpack8<BF16>(a[i], f[i]);
        if (p.residual) {
          float r[8];
          unpack8<BF16>(b[i], r);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i][j] += r[j];
          const uint4 s = pack8<BF16>(f[i]);
          p.s_out[row * p.vec + c] = s;
          unpack8<BF16>(s, f[i]);  // the norm reads the stream as it is held
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(f[i][j], f[i][j], ss);
        if constexpr (E4M3) {
          float w[8];
          unpack8<BF16>(__ldg(p.w + c), w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            f[i][j] *= w[j];
            top = fmaxf(top, fabsf(f[i][j]));
          }
        }
      }
    }
    const float2 both = row_reduce<E4M3>(ss, top, red, warps);
    const float rstd = rsqrtf(both.x * p.inv_cols + p.eps);
    if constexpr (!E4M3) {
      if (p.rstd && live && t == 0) p.rstd[row] = rstd;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = t + i * p.threads;
        if (live && c < p.vec) {
          float w[8];
          unpack8<BF16>(__ldg(p.w + c), w);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i][j] = f[i][j] * rstd * w[j];
          p.y[row * p.vec + c] = pack8<BF16>(f[i]);
        }
      }
    } else {
      // rstd scales the whole row, so it cancels in q: with m = max|s w|, q = s w (448 / m), and
      // only the scale, m rstd / 448, carries it. A row of zeros keeps scale 1, and so does one
      // whose sum of squares is infinite (rstd = 0: its finite values become 0, as in y); a row
      // with a NaN has rstd and scale NaN.
      const float m = both.y;
      const bool null = m == 0.f || rstd == 0.f;
      float k = null ? 0.f : 448.0f / m;
      if (!null && m < 1e-30f) {  // 448 / m may be infinite
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i][j] *= 0x1p100f;
        k = 448.0f / (m * 0x1p100f);
      }
      if (live && t == 0) p.scale[row] = null ? 1.0f : m * rstd / 448.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = t + i * p.threads;
        if (live && c < p.vec) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i][j] *= k;
          p.q[row * p.vec + c] = pack8_e4m3(f[i]);
        }
      }
      if constexpr (BF16) {
        if (m == INFINITY && rstd > 0.f) norm_first(p, row, t, rstd);
      }
    }
  }
}

// Each block walks over rows and keeps its share of dw in registers (a thread's columns stay
// the same for every row); at the end the block's row groups add up in shared memory in a
// fixed order and one partial row per block goes to dw_part, summed by add_norm_dw_kernel:
// no atomics, so dw does not depend on the order in which blocks run.
template <bool BF16, int VPT>
__global__ void __launch_bounds__(512) add_norm_bwd_kernel(const AddNormBwdParams p) {
  extern __shared__ float dw_smem[];  // [rows][8 * vec] when rows > 1 and dw is wanted
  __shared__ float2 red[AN_MAX_WARPS];
  const int g = threadIdx.x / p.threads, t = threadIdx.x - g * p.threads;
  const int warps = p.threads / 32;
  float acc[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
  const long long stride = static_cast<long long>(gridDim.x) * p.rows;
  uint4 na[VPT], nb[VPT], ne[VPT];
  float nrstd = 0.f;
  const auto load = [&](long long row) {
    const bool live = row < p.n;
    nrstd = live ? p.rstd[row] : 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * p.threads;
      na[i] = nb[i] = ne[i] = make_uint4(0u, 0u, 0u, 0u);
      if (live && c < p.vec) {
        na[i] = __ldcs(p.s + row * p.vec + c);
        if (p.dy) nb[i] = __ldcs(p.dy + row * p.vec + c);
        if (p.ds) ne[i] = __ldcs(p.ds + row * p.vec + c);
      }
    }
  };
  load(static_cast<long long>(blockIdx.x) * p.rows + g);
  for (long long row0 = static_cast<long long>(blockIdx.x) * p.rows; row0 < p.n; row0 += stride) {
    const long long row = row0 + g;
    const bool live = row < p.n;
    uint4 a[VPT], b[VPT], e[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      a[i] = na[i];
      b[i] = nb[i];
      e[i] = ne[i];
    }
    const float rstd = nrstd;
    load(row + stride);  // in flight while this row is reduced
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * p.threads;
      if (c < p.vec) {
        float s[8], d[8], w[8];
        unpack8<BF16>(a[i], s);
        unpack8<BF16>(b[i], d);
        unpack8<BF16>(__ldg(p.w + c), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float dn = d[j] * (s[j] * rstd);
          acc[i][j] += dn;
          dot = fmaf(dn, w[j], dot);
        }
      }
    }
    if (p.dx == nullptr) continue;
    const float mean = row_reduce<false>(dot, 0.f, red, warps).x * p.inv_cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * p.threads;
      if (live && c < p.vec) {
        float s[8], d[8], w[8], o[8];
        unpack8<BF16>(a[i], s);
        unpack8<BF16>(b[i], d);
        unpack8<BF16>(e[i], o);
        unpack8<BF16>(__ldg(p.w + c), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = fmaf(rstd, fmaf(d[j], w[j], -(s[j] * rstd) * mean), o[j]);
        p.dx[row * p.vec + c] = pack8<BF16>(o);
      }
    }
  }
  if (p.dw_part == nullptr) return;
  float4* out = reinterpret_cast<float4*>(p.dw_part + static_cast<size_t>(blockIdx.x) * p.vec * 8);
  if (p.rows > 1) {
    float4* mine = reinterpret_cast<float4*>(dw_smem) + static_cast<size_t>(g) * p.vec * 2;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * p.threads;
      if (c < p.vec) {
        mine[2 * c] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
        mine[2 * c + 1] = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
      }
    }
    __syncthreads();
    const float4* all = reinterpret_cast<const float4*>(dw_smem);
    for (int c = threadIdx.x; c < 2 * p.vec; c += blockDim.x) {
      float4 v = all[c];
      for (int r = 1; r < p.rows; ++r) {
        const float4 u = all[static_cast<size_t>(r) * p.vec * 2 + c];
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
      out[c] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * p.threads;
      if (c < p.vec) {
        out[2 * c] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
        out[2 * c + 1] = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
      }
    }
  }
}

// dw[c] = dtype(sum over parts of dw_part[.][c]): 8 columns per block (one 32-byte sector of a
// part), 32 slices of threads that each sum every 32nd part, then a fixed-order sum of the 32.
template <bool BF16>
__global__ void __launch_bounds__(256) add_norm_dw_kernel(const float* __restrict__ part, int parts, int cols,
                                                          uint16_t* __restrict__ dw) {
  __shared__ float sm[8][33];
  const int cx = threadIdx.x & 7, ry = threadIdx.x >> 3;
  const float* col = part + blockIdx.x * 8 + cx;  // cols is a multiple of 8
  float v = 0.f;
#pragma unroll 4
  for (int r = ry; r < parts; r += 32) v += col[static_cast<size_t>(r) * cols];
  sm[cx][ry] = v;
  __syncthreads();
  const int w = threadIdx.x / 32;
  v = warp_sum(sm[w][threadIdx.x & 31]);
  if ((threadIdx.x & 31) == 0) dw[blockIdx.x * 8 + w] = static_cast<uint16_t>(pack2<BF16>(v, 0.f) & 0xffffu);
}

}  // namespace lmce
