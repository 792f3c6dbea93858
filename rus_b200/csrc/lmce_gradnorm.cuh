// Global 2-norm of many gradient tensors and their scaling to a largest norm, in place:
//   total = sqrt(sum over all tensors of sum g^2),  k = max_norm / (total + 1e-6)
//   g = dtype(g * k) where k < 1 (or is not a number); else the gradients stay as they are
// (what the training loop around the reference's head calls after backward: TRL logs
// grad_norm and clips at max_grad_norm).
//
// Two launches per 1024 tensors: the tensors' addresses and sizes travel in the kernel's
// parameters (no table to copy, nothing kept between calls, safe in a captured graph), and
// blocks walk over fixed-size pieces of all tensors, so a small tensor costs a piece and not
// a launch. Memory-bound: the gradients are read once for the norm and, when clipped, read and
// written once more; the second pass runs backwards, so that it starts with what the first
// left in the L2 cache.
//
// Sums: eight (fp16 / bf16) or four (fp32) squares in fp32, then fp64. A vector whose largest
// magnitude lies outside [2^-40, 2^40] is squared in fp64, so neither large nor tiny gradients
// overflow or vanish (infinities and NaN reach the total through the same path).
#pragma once

#include <cstdint>

#include "lmce_rmsnorm.cuh"

namespace lmce {

constexpr int GN_THREADS = 256;
constexpr int GN_VECS = 8;                            // 16-byte vectors per thread and piece
constexpr int GN_PIECE = GN_THREADS * GN_VECS;        // vectors per piece: 32 KB
constexpr int GN_MAX_TENSORS = 1024;                  // per launch

enum : int { GN_F16 = 0, GN_BF16 = 1, GN_F32 = 2 };

// Tensors of one launch. first[i] is the number of pieces before tensor i. A tensor's pieces
// start at its address rounded down to 16 bytes; `lead` elements of that vector are not its own.
template <int MAXT>
struct GradBatch {
  int count;
  int first[MAXT + 1];
  void* ptr[MAXT];
  long long numel[MAXT];
  uint8_t dtype[MAXT];
};

template <int MAXT>
__device__ __forceinline__ int grad_tensor_of(const GradBatch<MAXT>& b, int piece) {
  int lo = 0, hi = b.count;  // first[lo] <= piece < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.first[mid] <= piece)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Geometry of a tensor seen as 16-byte vectors from its rounded-down address.
struct GradSpan {
  uint4* base;
  long long lead, end;  // its elements are [lead, end) of the vectors' elements
  int per;              // elements per vector
  int dt;
};

template <int MAXT>
__device__ __forceinline__ GradSpan grad_span(const GradBatch<MAXT>& b, int i) {
  GradSpan s;
  s.dt = b.dtype[i];
  const int size = s.dt == GN_F32 ? 4 : 2;
  const uintptr_t a = reinterpret_cast<uintptr_t>(b.ptr[i]);
  s.base = reinterpret_cast<uint4*>(a & ~uintptr_t(15));
  s.per = 16 / size;
  s.lead = static_cast<long long>((a & 15) / size);
  s.end = s.lead + b.numel[i];
  return s;
}

// The eight values of a vector; of fp32 the four it holds and four zeros.
__device__ __forceinline__ void grad_unpack(const uint4& u, int dt, float* f) {
  if (dt == GN_F32) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
    f[4] = f[5] = f[6] = f[7] = 0.f;
  } else if (dt == GN_BF16) {
    unpack8<true>(u, f);
  } else {
    unpack8<false>(u, f);
  }
}

__device__ __forceinline__ uint4 grad_pack(const float* f, int dt) {
  if (dt == GN_F32)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  return dt == GN_BF16 ? pack8<true>(f) : pack8<false>(f);
}

// One element at a time: the first and last vector of a tensor may share their 16 bytes with
// other data, which is neither read nor written.
__device__ __forceinline__ uint4 grad_load_part(const GradSpan& s, long long v) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  for (int j = 0; j < s.per; ++j) {
    const long long e = v * s.per + j;
    if (e < s.lead || e >= s.end) continue;
    if (s.per == 4)
      w[j] = reinterpret_cast<const uint32_t*>(s.base)[e];
    else
      w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(s.base)[e]) << (16 * (j & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void grad_store_part(const GradSpan& s, long long v, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  for (int j = 0; j < s.per; ++j) {
    const long long e = v * s.per + j;
    if (e < s.lead || e >= s.end) continue;
    if (s.per == 4)
      reinterpret_cast<uint32_t*>(s.base)[e] = w[j];
    else
      reinterpret_cast<uint16_t*>(s.base)[e] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
  }
}

__device__ __forceinline__ double sum_squares(const float* f) {
  float top = 0.f, low = 0.f, ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    top = fmaxf(top, fabsf(f[j]));
    ss = fmaf(f[j], f[j], ss);
    low += f[j];  // not a number where any value is (fmaxf drops them)
  }
  if (top == 0.f && low == 0.f) return 0.0;
  if (top >= 0x1p-40f && top <= 0x1p40f && low == low) return static_cast<double>(ss);
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) d += static_cast<double>(f[j]) * static_cast<double>(f[j]);
  return d;
}

__device__ __forceinline__ double block_sum(double v, double* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < GN_THREADS / 32; ++i) t += sm[i];
  return t;
}

// The run of pieces of this block.
__device__ __forceinline__ int grad_run(int pieces, int block) {
  return static_cast<int>(static_cast<long long>(pieces) * block / gridDim.x);
}

// partial[blockIdx.x] = this block's share of the sum of squares (the same gradients give the
// same bits).
template <int MAXT>
__global__ void __launch_bounds__(GN_THREADS, 4) grad_norm_kernel(const __grid_constant__ GradBatch<MAXT> b,
                                                               double* __restrict__ partial) {
  __shared__ double sm[GN_THREADS / 32];
  double sum = 0.0;
  const int pieces = b.first[b.count];
  const int p0 = grad_run(pieces, blockIdx.x), p1 = grad_run(pieces, blockIdx.x + 1);
  int i = p0 < p1 ? grad_tensor_of(b, p0) : 0;
  for (int piece = p0; piece < p1; ++piece) {
    while (b.first[i + 1] <= piece) ++i;
    const GradSpan s = grad_span(b, i);
    const long long v0 = static_cast<long long>(piece - b.first[i]) * GN_PIECE + threadIdx.x;
    const long long full_lo = s.lead > 0 ? 1 : 0, full_hi = s.end / s.per, all = (s.end + s.per - 1) / s.per;
    uint4 u[GN_VECS];
#pragma unroll
    for (int k = 0; k < GN_VECS; ++k) {
      const long long v = v0 + k * GN_THREADS;
      u[k] = make_uint4(0u, 0u, 0u, 0u);
      if (v >= full_lo && v < full_hi)
        u[k] = s.base[v];
      else if (v < all)
        u[k] = grad_load_part(s, v);
    }
#pragma unroll
    for (int k = 0; k < GN_VECS; ++k) {
      float f[8];
      grad_unpack(u[k], s.dt, f);
      sum += sum_squares(f);
    }
  }
  sum = block_sum(sum, sm);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// Adds the partial sums (every block the same way), and scales this launch's tensors when the
// norm exceeds max_norm. Two blocks per SM with 32 KB of loads each in flight: four (64
// registers) write 10% slower (one B200, 988 MB: 315 against 350 us). `total`, if not null,
// receives the norm (block 0).
template <int MAXT>
__global__ void __launch_bounds__(GN_THREADS, 2) grad_scale_kernel(const __grid_constant__ GradBatch<MAXT> b,
                                                                const double* __restrict__ partial, int parts,
                                                                float max_norm, float* __restrict__ total) {
  __shared__ double sm[GN_THREADS / 32];
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += GN_THREADS) sum += partial[i];
  const float norm = static_cast<float>(sqrt(block_sum(sum, sm)));
  if (total != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *total = norm;
  const float k = max_norm / (norm + 1e-6f);
  if (k >= 1.0f || max_norm == INFINITY) return;  // not a number: scale, so that it shows
  const int pieces = b.first[b.count];
  const int p0 = grad_run(pieces, blockIdx.x), p1 = grad_run(pieces, blockIdx.x + 1);
  int i = p0 < p1 ? grad_tensor_of(b, p1 - 1) : 0;
  for (int piece = p1 - 1; piece >= p0; --piece) {
    while (b.first[i] > piece) --i;
    const GradSpan s = grad_span(b, i);
    const long long v0 = static_cast<long long>(piece - b.first[i]) * GN_PIECE + threadIdx.x;
    const long long full_lo = s.lead > 0 ? 1 : 0, full_hi = s.end / s.per, all = (s.end + s.per - 1) / s.per;
    uint4 u[GN_VECS];
#pragma unroll
    for (int q = 0; q < GN_VECS; ++q) {
      const long long v = v0 + q * GN_THREADS;
      if (v >= full_lo && v < full_hi)
        u[q] = s.base[v];
      else if (v < all)
        u[q] = grad_load_part(s, v);
    }
#pragma unroll
    for (int q = 0; q < GN_VECS; ++q) {
      const long long v = v0 + q * GN_THREADS;
      if (v >= all) continue;
      float f[8];
      grad_unpack(u[q], s.dt, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= k;
      const uint4 o = grad_pack(f, s.dt);
      if (v >= full_lo && v < full_hi)
        s.base[v] = o;
      else
        grad_store_part(s, v, o);
    }
  }
}

}  // namespace lmce
