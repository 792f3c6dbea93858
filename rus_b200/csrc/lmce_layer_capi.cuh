// C entries of the operators around the head: residual add + RMSNorm and gradient clipping.
// Part of lmce_capi.cu (it uses that file's error, device and launch helpers).
#pragma once

#include <algorithm>
#include <new>

#include "lmce_addnorm.cuh"
#include "lmce_gradnorm.cuh"

namespace {

// ------------------------------------------------------ residual add + norm ---

constexpr int kAnThreads = 512;      // most threads of a row
constexpr int kAnBlock = 256;        // threads a block is filled up to with rows
constexpr int kAnBwdBlocks = 592;    // partial rows of dw: four blocks on each of 148 SMs
constexpr int64_t kAnMaxHidden = 32768;

struct RowShape {
  int vpt, threads, rows;
};

// Threads and vectors per thread for a row of `vec` 16-byte vectors: one vector per thread
// while rows are few (latency), two when there are enough rows to fill the SMs (more loads in
// flight per thread), more where a row would need over 512 threads.
RowShape row_shape(int64_t n, int vec, int sms) {
  RowShape s;
  s.vpt = n > 4ll * sms && vec > 32 ? 2 : 1;
  const auto threads = [&] { return (vec + 32 * s.vpt - 1) / (32 * s.vpt) * 32; };
  while (threads() > kAnThreads) s.vpt *= 2;
  s.threads = threads();
  s.rows = s.threads >= kAnBlock ? 1 : kAnBlock / s.threads;
  return s;
}

template <bool BF16, bool E4M3>
void launch_add_norm(const AddNormParams& p, int vpt, int grid, cudaStream_t st) {
  const int threads = p.threads * p.rows;
  switch (vpt) {
    case 1: add_norm_kernel<BF16, 1, E4M3><<<grid, threads, 0, st>>>(p); break;
    case 2: add_norm_kernel<BF16, 2, E4M3><<<grid, threads, 0, st>>>(p); break;
    case 4: add_norm_kernel<BF16, 4, E4M3><<<grid, threads, 0, st>>>(p); break;
    default: add_norm_kernel<BF16, 8, E4M3><<<grid, threads, 0, st>>>(p); break;
  }
}

template <bool BF16>
void launch_add_norm_bwd(const AddNormBwdParams& p, int vpt, int grid, size_t smem, cudaStream_t st) {
  const int threads = p.threads * p.rows;
  switch (vpt) {
    case 1: add_norm_bwd_kernel<BF16, 1><<<grid, threads, smem, st>>>(p); break;
    case 2: add_norm_bwd_kernel<BF16, 2><<<grid, threads, smem, st>>>(p); break;
    case 4: add_norm_bwd_kernel<BF16, 4><<<grid, threads, smem, st>>>(p); break;
    default: add_norm_bwd_kernel<BF16, 8><<<grid, threads, smem, st>>>(p); break;
  }
}

int check_rows(int64_t n, int64_t h, int dtype) {
  if (n <= 0 || n > (1ll << 30)) return fail(LMCE_ERR_INVALID_ARGUMENT, "bad n_rows");
  if (h <= 0 || h % 8 != 0 || h > kAnMaxHidden)
    return fail(LMCE_ERR_UNSUPPORTED, "hidden_dim must be a multiple of 8, at most %lld", (long long)kAnMaxHidden);
  if (dtype != LMCE_DTYPE_F16 && dtype != LMCE_DTYPE_BF16) return fail(LMCE_ERR_UNSUPPORTED, "dtype %d", dtype);
  return LMCE_OK;
}

// Both output forms of the forward (q null: 16-bit y).
int add_norm(const void* x, const void* residual, const void* weight, float eps, int64_t n, int64_t h, int dtype,
             void* s_out, void* y, void* q, float* scale, float* rstd, void* stream) {
  if (!x || !weight || (residual && !s_out) || !(q ? static_cast<void*>(scale) : y))
    return fail(LMCE_ERR_INVALID_ARGUMENT, "null pointer");
  if (int rc = check_rows(n, h, dtype)) return rc;
  if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || !aligned16(s_out) || !aligned16(y) ||
      !aligned16(q))
    return fail(LMCE_ERR_INVALID_ARGUMENT, "misaligned buffers");
  DevInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  const int vec = static_cast<int>(h / 8);
  const RowShape s = row_shape(n, vec, d->sms);
  AddNormParams p = {};
  p.x = static_cast<const uint4*>(x);
  p.residual = static_cast<const uint4*>(residual);
  p.w = static_cast<const uint4*>(weight);
  p.s_out = static_cast<uint4*>(s_out);
  p.y = static_cast<uint4*>(y);
  p.q = static_cast<uint2*>(q);
  p.scale = scale;
  p.rstd = rstd;
  p.n = n;
  p.vec = vec;
  p.threads = s.threads;
  p.rows = s.rows;
  p.inv_cols = 1.0f / static_cast<float>(h);
  p.eps = eps;
  const int64_t blocks = std::min<int64_t>((n + s.rows - 1) / s.rows, d->sms * 16ll);
  const int grid = static_cast<int>(blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LMCE_DTYPE_BF16)
    q ? launch_add_norm<true, true>(p, s.vpt, grid, st) : launch_add_norm<true, false>(p, s.vpt, grid, st);
  else
    q ? launch_add_norm<false, true>(p, s.vpt, grid, st) : launch_add_norm<false, false>(p, s.vpt, grid, st);
  return launched();
}

// -------------------------------------------------------- gradient clipping ---

constexpr int kGnBlocks = 1184;  // eight blocks on each of 148 SMs; partial sums per launch

template <int MAXT>
int64_t fill_batch(GradBatch<MAXT>* b, void* const* grads, const int64_t* numels, const int32_t* dtypes,
                   int64_t count) {
  int64_t pieces = 0;
  b->count = static_cast<int>(count);
  for (int64_t i = 0; i < count; ++i) {
    b->first[i] = static_cast<int>(pieces);
    b->ptr[i] = grads[i];
    b->numel[i] = numels[i];
    b->dtype[i] = static_cast<uint8_t>(dtypes[i]);
    const int64_t size = dtypes[i] == LMCE_DTYPE_F32 ? 4 : 2;
    const int64_t bytes = (reinterpret_cast<uintptr_t>(grads[i]) & 15) + numels[i] * size;
    pieces += (bytes + 16ll * GN_PIECE - 1) / (16ll * GN_PIECE);
  }
  b->first[count] = static_cast<int>(pieces);
  return pieces;
}

template <int MAXT>
int launch_clip(bool scale, void* const* grads, const int64_t* numels, const int32_t* dtypes, int64_t count,
                double* partial, int parts, float max_norm, float* total, cudaStream_t st) {
  GradBatch<MAXT> b;
  const int64_t pieces = fill_batch(&b, grads, numels, dtypes, count);
  if (scale) {
    const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(pieces, 1), kGnBlocks));
    grad_scale_kernel<MAXT><<<grid, GN_THREADS, 0, st>>>(b, partial, parts, max_norm, total);
  } else {
    grad_norm_kernel<MAXT><<<kGnBlocks, GN_THREADS, 0, st>>>(b, partial);
  }
  return launched();
}

}  // namespace

extern "C" {

int lmce_add_rmsnorm(const void* x, const void* residual, const void* weight, float eps, int64_t n_rows,
                     int64_t hidden_dim, int dtype, void* s_out, void* y_out, float* rstd_out, void* stream) {
  return add_norm(x, residual, weight, eps, n_rows, hidden_dim, dtype, s_out, y_out, nullptr, nullptr, rstd_out,
                  stream);
}

int lmce_add_rmsnorm_e4m3(const void* x, const void* residual, const void* weight, float eps, int64_t n_rows,
                          int64_t hidden_dim, int dtype, void* s_out, void* q_out, float* scale_out, void* stream) {
  if (!q_out) return fail(LMCE_ERR_INVALID_ARGUMENT, "null pointer");
  return add_norm(x, residual, weight, eps, n_rows, hidden_dim, dtype, s_out, nullptr, q_out, scale_out, nullptr,
                  stream);
}

size_t lmce_add_rmsnorm_bwd_workspace_bytes(int64_t n_rows, int64_t hidden_dim) {
  if (n_rows <= 0 || hidden_dim <= 0) return 0;
  return static_cast<size_t>(std::min<int64_t>(n_rows, kAnBwdBlocks)) * hidden_dim * 4;
}

int lmce_add_rmsnorm_backward(const void* d_y, const void* d_s, const void* s, const void* weight, const float* rstd,
                              int64_t n_rows, int64_t hidden_dim, int dtype, void* d_x, void* d_weight,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (!s || !weight || !rstd || (!d_x && !d_weight)) return fail(LMCE_ERR_INVALID_ARGUMENT, "null pointer");
  if (int rc = check_rows(n_rows, hidden_dim, dtype)) return rc;
  if (!aligned16(d_y) || !aligned16(d_s) || !aligned16(s) || !aligned16(weight) || !aligned16(d_x) ||
      !aligned16(workspace))
    return fail(LMCE_ERR_INVALID_ARGUMENT, "misaligned buffers");
  if (d_weight && (!workspace || workspace_bytes < lmce_add_rmsnorm_bwd_workspace_bytes(n_rows, hidden_dim)))
    return fail(LMCE_ERR_WORKSPACE, "workspace too small");
  DevInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  const int vec = static_cast<int>(hidden_dim / 8);
  const RowShape sh = row_shape(n_rows, vec, d->sms);
  AddNormBwdParams p = {};
  p.dy = static_cast<const uint4*>(d_y);
  p.ds = static_cast<const uint4*>(d_s);
  p.s = static_cast<const uint4*>(s);
  p.w = static_cast<const uint4*>(weight);
  p.rstd = rstd;
  p.dx = static_cast<uint4*>(d_x);
  p.dw_part = d_weight ? static_cast<float*>(workspace) : nullptr;
  p.n = n_rows;
  p.vec = vec;
  p.threads = sh.threads;
  p.rows = sh.rows;
  p.inv_cols = 1.0f / static_cast<float>(hidden_dim);
  const int grid = static_cast<int>(std::min<int64_t>((n_rows + sh.rows - 1) / sh.rows, kAnBwdBlocks));
  const size_t smem = d_weight && sh.rows > 1 ? static_cast<size_t>(sh.rows) * hidden_dim * 4 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LMCE_DTYPE_BF16)
    launch_add_norm_bwd<true>(p, sh.vpt, grid, smem, st);
  else
    launch_add_norm_bwd<false>(p, sh.vpt, grid, smem, st);
  if (int rc = launched()) return rc;
  if (!d_weight) return LMCE_OK;
  const int cols = static_cast<int>(hidden_dim);
  if (dtype == LMCE_DTYPE_BF16)
    add_norm_dw_kernel<true><<<(cols + 31) / 32, 1024, 0, st>>>(p.dw_part, grid, cols,
                                                                static_cast<uint16_t*>(d_weight));
  else
    add_norm_dw_kernel<false><<<(cols + 31) / 32, 1024, 0, st>>>(p.dw_part, grid, cols,
                                                                 static_cast<uint16_t*>(d_weight));
  return launched();
}

size_t lmce_clip_grad_workspace_bytes(int64_t count) {
  if (count <= 0) return 0;
  return static_cast<size_t>((count + GN_MAX_TENSORS - 1) / GN_MAX_TENSORS) * kGnBlocks * sizeof(double);
}

int lmce_clip_grad_norm(void* const* grads, const int64_t* numels, const int32_t* dtypes, int64_t count,
                        float max_norm, float* total_norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (!grads || !numels || !dtypes || !total_norm || !workspace)
    return fail(LMCE_ERR_INVALID_ARGUMENT, "null pointer");
  if (count <= 0 || count > (1 << 20)) return fail(LMCE_ERR_INVALID_ARGUMENT, "bad count");
  if (!(max_norm >= 0.0f)) return fail(LMCE_ERR_INVALID_ARGUMENT, "max_norm must not be negative");
  if (workspace_bytes < lmce_clip_grad_workspace_bytes(count) || reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
    return fail(LMCE_ERR_WORKSPACE, "workspace too small or misaligned");
  struct Range {
    uintptr_t lo, hi;
  };
  Range* r = new (std::nothrow) Range[count];
  if (!r) return fail(LMCE_ERR_INVALID_ARGUMENT, "out of host memory");
  int rc = LMCE_OK;
  int64_t used = 0;
  for (int64_t i = 0; i < count && rc == LMCE_OK; ++i) {
    if (dtypes[i] != LMCE_DTYPE_F16 && dtypes[i] != LMCE_DTYPE_BF16 && dtypes[i] != LMCE_DTYPE_F32)
      rc = fail(LMCE_ERR_UNSUPPORTED, "gradient %lld: dtype %d", (long long)i, dtypes[i]);
    const uintptr_t size = dtypes[i] == LMCE_DTYPE_F32 ? 4 : 2;
    const uintptr_t a = reinterpret_cast<uintptr_t>(grads[i]);
    if (numels[i] < 0 || numels[i] > (1ll << 42) || (numels[i] > 0 && (a == 0 || a % size != 0)))
      rc = fail(LMCE_ERR_INVALID_ARGUMENT, "gradient %lld: null, misaligned or bad size", (long long)i);
    if (numels[i] > 0) r[used++] = {a, a + static_cast<uintptr_t>(numels[i]) * size};
  }
  if (rc == LMCE_OK) {
    // a gradient listed twice would be scaled by two blocks at once
    std::sort(r, r + used, [](const Range& x, const Range& y) { return x.lo < y.lo; });
    for (int64_t i = 1; i < used && rc == LMCE_OK; ++i)
      if (r[i].lo < r[i - 1].hi) rc = fail(LMCE_ERR_INVALID_ARGUMENT, "gradients overlap in memory");
  }
  delete[] r;
  if (rc) return rc;
  DevInfo* d = nullptr;
  if ((rc = device_info(&d))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  const int64_t batches = (count + GN_MAX_TENSORS - 1) / GN_MAX_TENSORS;
  const int parts = static_cast<int>(batches) * kGnBlocks;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t k = 0; k < batches; ++k) {
      const int64_t b = pass == 0 ? k : batches - 1 - k;  // the scaling pass runs backwards
      const int64_t i0 = b * GN_MAX_TENSORS, m = std::min<int64_t>(count - i0, GN_MAX_TENSORS);
      double* part = pass == 0 ? partial + b * kGnBlocks : partial;
      float* total = b == 0 ? total_norm : nullptr;
      // the parameters of a launch with few tensors stay small
      rc = m <= 64 ? launch_clip<64>(pass == 1, grads + i0, numels + i0, dtypes + i0, m, part, parts, max_norm, total,
                                     st)
                   : launch_clip<GN_MAX_TENSORS>(pass == 1, grads + i0, numels + i0, dtypes + i0, m, part, parts,
                                                 max_norm, total, st);
      if (rc) return rc;
    }
  }
  return LMCE_OK;
}

}  // extern "C"
