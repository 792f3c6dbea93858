// C entries of the operators around the head: residual add + RMSNorm, the gated projection of a
// feed-forward block, and gradient clipping.
// Part of lmce_capi.cu (it uses that file's error, device and launch helpers).
#pragma once

#include <algorithm>
#include <new>

#include "lmce_addnorm.cuh"
#include "lmce_gated.cuh"
#include "lmce_gradnorm.cuh"

namespace {

// ------------------------------------------------------ residual add + norm ---

constexpr int kAnThreads = 512;      // most threads of a row
constexpr int kAnBlock = 256;        // threads a block is filled up to with rows
constexpr int kAnBwdBlocks = 296;    // partial rows of dw: the two blocks that 148 SMs hold at once
constexpr int64_t kAnMaxHidden = 16384;

struct RowShape {
  int vpt, threads, rows;
};

// Threads and vectors per thread for a row of `vec` 16-byte vectors: one vector per thread while
// that is under 700 threads per SM (latency), two beyond (more loads in flight per thread), four
// where a row would need over 512 threads. One B200, forward, one and two vectors: 1 x 896 1.77
// and 2.02 us, 512 x 896 3.04 and 3.36, 300 x 4096 4.56 and 4.40 (e4m3 5.55 and 4.31), 32768 x
// 4096 200 and 169 (four: 178).
RowShape row_shape(int64_t n, int vec, int sms) {
  RowShape s;
  s.vpt = n * vec > 700ll * sms && vec > 32 ? 2 : 1;
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
    default: add_norm_kernel<BF16, 4, E4M3><<<grid, threads, 0, st>>>(p); break;
  }
}

template <bool BF16>
void launch_add_norm_bwd(const AddNormBwdParams& p, int vpt, int grid, size_t smem, cudaStream_t st) {
  const int threads = p.threads * p.rows;
  switch (vpt) {
    case 1: add_norm_bwd_kernel<BF16, 1><<<grid, threads, smem, st>>>(p); break;
    case 2: add_norm_bwd_kernel<BF16, 2><<<grid, threads, smem, st>>>(p); break;
    default: add_norm_bwd_kernel<BF16, 4><<<grid, threads, smem, st>>>(p); break;
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
  if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || (residual && !aligned16(s_out)) ||
      !aligned16(y) || !aligned16(q))
    return fail(LMCE_ERR_INVALID_ARGUMENT, "misaligned buffers");
  DevInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  const int vec = static_cast<int>(h / 8);
  const RowShape s = row_shape(n, vec, d->sms);
  AddNormParams p = {};
  p.x = static_cast<const uint4*>(x);
  p.residual = static_cast<const uint4*>(residual);
  p.w = static_cast<const uint4*>(weight);
  p.s_out = residual ? static_cast<uint4*>(s_out) : nullptr;
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

constexpr int kGnBlocks = 592;  // the four blocks that 148 SMs hold at once; partial sums per launch

int64_t grad_pieces(const void* grad, int64_t numel, int32_t dtype) {
  const int64_t size = dtype == LMCE_DTYPE_F32 ? 4 : 2;
  const int64_t bytes = static_cast<int64_t>(reinterpret_cast<uintptr_t>(grad) & 15) + numel * size;
  return numel > 0 ? (bytes + 16ll * GN_PIECE - 1) / (16ll * GN_PIECE) : 0;
}

// One launch of either pass over `count` tensors.
template <int MAXT>
int launch_clip(bool scale, void* const* grads, const int64_t* numels, const int32_t* dtypes, int64_t count, int grid,
                double* partial, int parts, float max_norm, float* total, cudaStream_t st) {
  GradBatch<MAXT> b;
  int64_t pieces = 0;
  b.count = static_cast<int>(count);
  for (int64_t i = 0; i < count; ++i) {
    b.first[i] = static_cast<int>(pieces);
    b.ptr[i] = grads[i];
    b.numel[i] = numels[i];
    b.dtype[i] = static_cast<uint8_t>(dtypes[i]);
    pieces += grad_pieces(grads[i], numels[i], dtypes[i]);
  }
  b.first[count] = static_cast<int>(pieces);
  if (scale)
    grad_scale_kernel<MAXT><<<(grid + 1) / 2, GN_THREADS, 0, st>>>(b, partial, parts, max_norm, total);
  else
    grad_norm_kernel<MAXT><<<grid, GN_THREADS, 0, st>>>(b, partial);
  return launched();
}

// ------------------------------------------------------- gated projection ---

constexpr int64_t kGatedMaxRows = 1ll << 26;   // tiles and token indices stay within 32 bits
constexpr int64_t kGatedMaxDim = 1ll << 20;
constexpr int kGatedPairs = 74;                // CTA pairs the backward's K splits are sized for
constexpr int kGatedMaxSplits = 16;

// [outer][inner] bytes (e4m3) as a 3-D view {128, outer, inner / 128 blocks}, 128-byte swizzle:
// the boxes hold the same bytes as those of 64 16-bit values (make_map_3d).
int make_map_3d_bytes(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint32_t box_y,
                      uint32_t box_z) {
  cuuint64_t dims[3] = {128, outer, inner / 128};
  cuuint64_t strides[2] = {inner, 128};
  cuuint32_t box[3] = {128, box_y, box_z};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(LMCE_ERR_CUDA, "cuTensorMapEncodeTiled (bytes) failed (%d)", static_cast<int>(r));
  return LMCE_OK;
}

// maps: x, gate, up, h
template <bool BF16, bool E4M3, bool SAVE>
int launch_gated_pairs(const CUtensorMap* maps, const GatedParams& p, int sms, cudaStream_t st) {
  auto kern = gated_fwd_kernel<BF16, E4M3, SAVE>;
  static bool done[kMaxDevices] = {};
  if (int rc = ensure_smem_attr(kern, PBWD_SMEM_BYTES, done)) return rc;
  static int cache[kMaxDevices] = {};
  const int slots = max_pairs(kern, PBWD_SMEM_BYTES, sms, cache, P_THREADS);
  const int64_t units = static_cast<int64_t>((p.N + GP_TOK - 1) / GP_TOK) * ((p.F + GP_FT - 1) / GP_FT);
  const int grid = 2 * static_cast<int>(std::min<int64_t>(units, slots));
  return launch_ex(kern, grid, P_THREADS, PBWD_SMEM_BYTES, 2, st, maps[0], maps[1], maps[2], maps[3], p);
}

template <bool BF16, bool E4M3, bool SAVE>
int launch_gated_few(const CUtensorMap* maps, const GatedParams& p, void* h, int sms, cudaStream_t st) {
  auto kern = gated_few_kernel<BF16, E4M3, SAVE>;
  static bool done[kMaxDevices] = {};
  if (int rc = ensure_smem_attr(kern, PBWD_SMEM_BYTES, done)) return rc;
  const int grid = std::min(p.F / GF_FT, sms);
  return launch_ex(kern, grid, P_THREADS, PBWD_SMEM_BYTES, 1, st, maps[0], maps[1], maps[2], static_cast<uint16_t*>(h),
                   p);
}

template <bool BF16, bool E4M3>
int launch_gated(const CUtensorMap* maps, const GatedParams& p, void* h, int sms, cudaStream_t st) {
  const bool pairs = p.N > BM;
  if constexpr (!E4M3) {
    if (p.saved != nullptr)
      return pairs ? launch_gated_pairs<BF16, E4M3, true>(maps, p, sms, st)
                   : launch_gated_few<BF16, E4M3, true>(maps, p, h, sms, st);
  }
  return pairs ? launch_gated_pairs<BF16, E4M3, false>(maps, p, sms, st)
               : launch_gated_few<BF16, E4M3, false>(maps, p, h, sms, st);
}

template <bool BF16, bool E4M3>
int launch_gated_token(const void* x, const void* wg, const void* wu, const GatedParams& p, void* h,
                       cudaStream_t st) {
  const int vec = p.H / (E4M3 ? 16 : 8), grid = (p.F + GT_WARPS - 1) / GT_WARPS;
  gated_token_kernel<BF16, E4M3><<<grid, 32 * GT_WARPS, 0, st>>>(
      static_cast<const uint4*>(x), static_cast<const uint4*>(wg), static_cast<const uint4*>(wu), vec, p,
      static_cast<uint16_t*>(h));
  return launched();
}

int check_gated(int64_t n, int64_t h, int64_t f, int dtype, int act, int64_t h_step) {
  if (n <= 0 || n > kGatedMaxRows) return fail(LMCE_ERR_INVALID_ARGUMENT, "bad n_rows");
  if (h <= 0 || h % h_step != 0 || h > kGatedMaxDim)
    return fail(LMCE_ERR_UNSUPPORTED, "hidden_dim must be a multiple of %lld, at most 2^20", (long long)h_step);
  if (f <= 0 || f % 64 != 0 || f > kGatedMaxDim)
    return fail(LMCE_ERR_UNSUPPORTED, "ffn_dim must be a multiple of 64, at most 2^20");
  if (((n + 127) / 128) * ((f + 63) / 64) > 0x7fffffffll || ((n + 255) / 256) * ((h + 255) / 256) > 0x3ffffffll)
    return fail(LMCE_ERR_UNSUPPORTED, "too many tiles");
  if (dtype != LMCE_DTYPE_F16 && dtype != LMCE_DTYPE_BF16) return fail(LMCE_ERR_UNSUPPORTED, "dtype %d", dtype);
  if (act != LMCE_ACT_SILU && act != LMCE_ACT_GELU_TANH) return fail(LMCE_ERR_UNSUPPORTED, "activation %d", act);
  return LMCE_OK;
}

struct GatedBwdLayout {
  size_t dg, du, part, total;
  int splits, stages, rows_pad;
};

// K splits of a dx tile, so that a few tiles with a long K (few tokens) do not hold up the rest:
// the number with the least expected time, in stages of a pair. That is the longest pair's work
// (the assignment of GatedUnits) plus, for the partials, a launch and their bytes written and
// read, N * H * 8 per split at 6.4 TB/s and 0.55 us per stage. Within 4% of the best number at
// 18 shapes from 64 to 3000 tokens on one B200 (693 x 1536 x 8960: 2 splits 79.7 us, 3 81.1, 1
// 109, 16 99; the weights frozen: 4 splits 50.4 us, 1 103).
int gated_splits(int64_t n, int64_t h, int64_t tiles, int64_t stages, int64_t n_dw) {
  const int64_t P = kGatedPairs;
  const double cd = static_cast<double>(std::max<int64_t>((n + 127) / 128, GATED_UNIT_STAGES));
  int best = 1;
  double least = 0;
  for (int s = 1; s <= kGatedMaxSplits && s <= stages; ++s) {
    const int64_t n_dx = tiles * s, heavy = n_dx % P, light = heavy ? P - heavy : 0;
    const double cx = static_cast<double>(std::max<int64_t>((stages + s - 1) / s, GATED_UNIT_STAGES));
    const int64_t ahead = light ? static_cast<int64_t>(cx / cd) : 0;
    const int64_t common = std::min(n_dw, light * ahead), rest = n_dw - common;
    // the fullest of the pairs with one DX unit more (the first pair), and of the others
    const int64_t dw_first = (rest + P - 1) / P;
    const int64_t dw_other = (light ? (common + light - 1) / light : 0) +
                             std::max<int64_t>(0, (rest - heavy + P - 1) / P);
    const double first = static_cast<double>(n_dx / P + (heavy ? 1 : 0)) * cx + static_cast<double>(dw_first) * cd;
    const double other = static_cast<double>(n_dx / P) * cx + static_cast<double>(dw_other) * cd;
    const double t = std::max(first, other) + (s > 1 ? 5.0 + 2.3e-6 * static_cast<double>(s) * n * h : 0.0);
    if (s == 1 || t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

GatedBwdLayout gated_bwd_layout(int64_t n, int64_t h, int64_t f, bool want_dx, int n_weights) {
  GatedBwdLayout L = {};
  const int64_t nh = (h + 255) / 256;
  L.stages = static_cast<int>(2 * ((f + 127) / 128));
  L.splits = want_dx ? gated_splits(n, h, (n + 255) / 256 * nh, L.stages, n_weights * ((f + 255) / 256) * nh) : 1;
  L.rows_pad = static_cast<int>((n + 255) / 256 * 256);
  size_t off = 0;
  L.dg = off;
  off = align_up(off + static_cast<size_t>(n) * f * 2, 256);
  L.du = off;
  off = align_up(off + static_cast<size_t>(n) * f * 2, 256);
  L.part = off;
  if (want_dx && L.splits > 1) off = align_up(off + static_cast<size_t>(L.splits) * L.rows_pad * h * 4, 256);
  L.total = off;
  return L;
}

template <bool BF16>
int launch_gated_bwd(const CUtensorMap* maps, const GatedBwdParams& p, int sms, cudaStream_t st) {
  auto kern = gated_bwd_kernel<BF16>;
  static bool done[kMaxDevices] = {};
  if (int rc = ensure_smem_attr(kern, PBWD_SMEM_BYTES, done)) return rc;
  static int cache[kMaxDevices] = {};
  const int slots = max_pairs(kern, PBWD_SMEM_BYTES, sms, cache, P_THREADS);
  const int grid = 2 * static_cast<int>(std::min<int64_t>(static_cast<int64_t>(p.n_dx) + p.n_dw, slots));
  return launch_ex(kern, grid, P_THREADS, PBWD_SMEM_BYTES, 2, st, maps[0], maps[1], maps[2], maps[3], maps[4], maps[5],
                   maps[6], maps[7], p);
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
    add_norm_dw_kernel<true><<<cols / 8, 256, 0, st>>>(p.dw_part, grid, cols,
                                                                static_cast<uint16_t*>(d_weight));
  else
    add_norm_dw_kernel<false><<<cols / 8, 256, 0, st>>>(p.dw_part, grid, cols,
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
  if (count <= 0 || count > (1 << 20))
    return fail(LMCE_ERR_INVALID_ARGUMENT, "%lld gradients (need 1 to 2^20)", (long long)count);
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
    if (numels[i] < 0 || numels[i] > (1ll << 34) || (numels[i] > 0 && (a == 0 || a % size != 0)))
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
  const auto grid_of = [&](int64_t i0, int64_t m) {
    int64_t pieces = 0;
    for (int64_t i = i0; i < i0 + m; ++i) pieces += grad_pieces(grads[i], numels[i], dtypes[i]);
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>(pieces, 1), kGnBlocks));
  };
  int parts = 0;  // blocks of the first pass so far
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t k = 0; k < batches; ++k) {
      const int64_t b = pass == 0 ? k : batches - 1 - k;  // the scaling pass runs backwards
      const int64_t i0 = b * GN_MAX_TENSORS, m = std::min<int64_t>(count - i0, GN_MAX_TENSORS);
      const int grid = grid_of(i0, m);
      double* part = pass == 0 ? partial + parts : partial;
      if (pass == 0) parts += grid;
      float* total = b == 0 ? total_norm : nullptr;
      // the parameters of a launch with few tensors stay small
      rc = m <= 64 ? launch_clip<64>(pass == 1, grads + i0, numels + i0, dtypes + i0, m, grid, part, parts, max_norm,
                                     total, st)
                   : launch_clip<GN_MAX_TENSORS>(pass == 1, grads + i0, numels + i0, dtypes + i0, m, grid, part, parts,
                                                 max_norm, total, st);
      if (rc) return rc;
    }
  }
  return LMCE_OK;
}

size_t lmce_gated_saved_bytes(int64_t n_rows, int64_t ffn_dim) {
  if (n_rows <= 0 || ffn_dim <= 0) return 0;
  return static_cast<size_t>((n_rows + 31) / 32 * 32) * ffn_dim * 6;
}

int lmce_gated_linear(const void* x, const void* w_gate, const void* w_up, int64_t n_rows, int64_t hidden_dim,
                      int64_t ffn_dim, int dtype, int act, void* h_out, void* saved, void* stream) {
  if (!x || !w_gate || !w_up || !h_out) return fail(LMCE_ERR_INVALID_ARGUMENT, "null pointer");
  if (int rc = check_gated(n_rows, hidden_dim, ffn_dim, dtype, act, 64)) return rc;
  if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(h_out) || !aligned16(saved))
    return fail(LMCE_ERR_INVALID_ARGUMENT, "misaligned buffers");
  DevInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  if (int rc = get_encoder()) return rc;
  const bool bf16 = dtype == LMCE_DTYPE_BF16, pair = n_rows > BM;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  GatedParams p = {};
  p.N = static_cast<int>(n_rows);
  p.H = static_cast<int>(hidden_dim);
  p.F = static_cast<int>(ffn_dim);
  p.act = act;
  p.saved = static_cast<uint8_t*>(saved);
  p.err = d->err_ptr;
  p.timeout_ns = wait_timeout_ns();
  if (n_rows == 1 && !saved)
    return bf16 ? launch_gated_token<true, false>(x, w_gate, w_up, p, h_out, st)
                : launch_gated_token<false, false>(x, w_gate, w_up, p, h_out, st);
  const uint32_t x_rows = pair ? 128 : static_cast<uint32_t>((n_rows + 15) / 16 * 16);
  const uint32_t w_rows = pair ? 128 : 64, w_blocks = pair ? 2 : 1;
  p.b_rows = static_cast<int>(x_rows);
  CUtensorMap maps[4];
  if (int rc = make_map_3d(&maps[0], x, bf16, hidden_dim, n_rows, hidden_dim, x_rows, 2)) return rc;
  if (int rc = make_map_3d(&maps[1], w_gate, bf16, hidden_dim, ffn_dim, hidden_dim, w_rows, w_blocks)) return rc;
  if (int rc = make_map_3d(&maps[2], w_up, bf16, hidden_dim, ffn_dim, hidden_dim, w_rows, w_blocks)) return rc;
  if (int rc = make_map_store16(&maps[3], h_out, bf16, ffn_dim, n_rows, ffn_dim)) return rc;
  return bf16 ? launch_gated<true, false>(maps, p, h_out, d->sms, st)
              : launch_gated<false, false>(maps, p, h_out, d->sms, st);
}

int lmce_gated_linear_e4m3(const void* x, const float* x_scale, const void* w_gate, const float* gate_scale,
                           const void* w_up, const float* up_scale, int64_t n_rows, int64_t hidden_dim,
                           int64_t ffn_dim, int out_dtype, int act, void* h_out, void* stream) {
  if (!x || !x_scale || !w_gate || !gate_scale || !w_up || !up_scale || !h_out)
    return fail(LMCE_ERR_INVALID_ARGUMENT, "null pointer");
  if (int rc = check_gated(n_rows, hidden_dim, ffn_dim, out_dtype, act, 128)) return rc;
  if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(h_out) || !aligned16(gate_scale) ||
      !aligned16(up_scale) || reinterpret_cast<uintptr_t>(x_scale) % 4 != 0)
    return fail(LMCE_ERR_INVALID_ARGUMENT, "misaligned buffers");
  DevInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  if (int rc = get_encoder()) return rc;
  const bool bf16 = out_dtype == LMCE_DTYPE_BF16, pair = n_rows > BM;
  GatedParams p = {};
  p.N = static_cast<int>(n_rows);
  p.H = static_cast<int>(hidden_dim);
  p.F = static_cast<int>(ffn_dim);
  p.act = act;
  p.x_scale = x_scale;
  p.g_scale = gate_scale;
  p.u_scale = up_scale;
  p.err = d->err_ptr;
  p.timeout_ns = wait_timeout_ns();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n_rows == 1)
    return bf16 ? launch_gated_token<true, true>(x, w_gate, w_up, p, h_out, st)
                : launch_gated_token<false, true>(x, w_gate, w_up, p, h_out, st);
  const uint32_t x_rows = pair ? 128 : static_cast<uint32_t>((n_rows + 15) / 16 * 16);
  const uint32_t w_rows = pair ? 128 : 64, w_blocks = pair ? 2 : 1;
  p.b_rows = static_cast<int>(x_rows);
  CUtensorMap maps[4];
  if (int rc = make_map_3d_bytes(&maps[0], x, hidden_dim, n_rows, x_rows, 2)) return rc;
  if (int rc = make_map_3d_bytes(&maps[1], w_gate, hidden_dim, ffn_dim, w_rows, w_blocks)) return rc;
  if (int rc = make_map_3d_bytes(&maps[2], w_up, hidden_dim, ffn_dim, w_rows, w_blocks)) return rc;
  if (int rc = make_map_store16(&maps[3], h_out, bf16, ffn_dim, n_rows, ffn_dim)) return rc;
  return bf16 ? launch_gated<true, true>(maps, p, h_out, d->sms, st)
              : launch_gated<false, true>(maps, p, h_out, d->sms, st);
}

size_t lmce_gated_bwd_workspace_bytes(int64_t n_rows, int64_t hidden_dim, int64_t ffn_dim, int want_dx,
                                      int n_weights) {
  if (n_rows <= 0 || hidden_dim <= 0 || ffn_dim <= 0) return 0;
  return gated_bwd_layout(n_rows, hidden_dim, ffn_dim, want_dx != 0, n_weights).total;
}

int lmce_gated_backward(const void* d_h, const void* saved, const void* x, const void* w_gate, const void* w_up,
                        int64_t n_rows, int64_t hidden_dim, int64_t ffn_dim, int dtype, int act, void* d_x,
                        void* d_gate, void* d_up, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d_h || !saved || !x || !w_gate || !w_up || !workspace || (!d_x && !d_gate && !d_up))
    return fail(LMCE_ERR_INVALID_ARGUMENT, "null pointer");
  if (int rc = check_gated(n_rows, hidden_dim, ffn_dim, dtype, act, 64)) return rc;
  if (!aligned16(d_h) || !aligned16(saved) || !aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) ||
      !aligned16(d_x) || !aligned16(d_gate) || !aligned16(d_up) || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(LMCE_ERR_INVALID_ARGUMENT, "misaligned buffers");
  const int n_weights = (d_gate ? 1 : 0) + (d_up ? 1 : 0);
  const GatedBwdLayout L = gated_bwd_layout(n_rows, hidden_dim, ffn_dim, d_x != nullptr, n_weights);
  if (workspace_bytes < L.total) return fail(LMCE_ERR_WORKSPACE, "workspace too small");
  DevInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  if (int rc = get_encoder()) return rc;
  const bool bf16 = dtype == LMCE_DTYPE_BF16;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  void *dg = ws + L.dg, *du = ws + L.du;
  float* part = reinterpret_cast<float*>(ws + L.part);
  const int64_t n = n_rows, h = hidden_dim, f = ffn_dim;
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  const int dgrid = static_cast<int>(std::min<int64_t>((n + 31) / 32 * (f / 64), d->sms * 5ll));
  const bool silu = act == LMCE_ACT_SILU;
  const auto dact = bf16 ? (silu ? gated_dact_kernel<true, ACT_SILU> : gated_dact_kernel<true, ACT_GELU_TANH>)
                         : (silu ? gated_dact_kernel<false, ACT_SILU> : gated_dact_kernel<false, ACT_GELU_TANH>);
  dact<<<dgrid, GATED_DACT_THREADS, 0, st>>>(static_cast<const uint8_t*>(saved), static_cast<const uint4*>(d_h),
                                             static_cast<int>(n), static_cast<int>(f), static_cast<uint4*>(dg),
                                             static_cast<uint4*>(du));
  if (int rc = launched()) return rc;

  CUtensorMap maps[8];
  if (int rc = make_map_3d(&maps[0], x, bf16, h, n, h, 128, 2)) return rc;
  if (int rc = make_map_3d(&maps[1], w_gate, bf16, h, f, h, 128, 2)) return rc;
  if (int rc = make_map_3d(&maps[2], w_up, bf16, h, f, h, 128, 2)) return rc;
  if (int rc = make_map_3d(&maps[3], dg, bf16, f, n, f, 128, 2)) return rc;
  if (int rc = make_map_3d(&maps[4], du, bf16, f, n, f, 128, 2)) return rc;
  // outputs that are not wanted keep a valid map that no unit uses
  if (d_x && L.splits > 1) {
    if (int rc = make_map_f32(&maps[5], part, h, static_cast<uint64_t>(L.splits) * L.rows_pad, h, 32, 32)) return rc;
  } else if (int rc = make_map_store16(&maps[5], d_x ? d_x : dg, bf16, d_x ? h : f, n, d_x ? h : f)) {
    return rc;
  }
  if (int rc = make_map_store16(&maps[6], d_gate ? d_gate : dg, bf16, d_gate ? h : f, d_gate ? f : n, d_gate ? h : f))
    return rc;
  if (int rc = make_map_store16(&maps[7], d_up ? d_up : dg, bf16, d_up ? h : f, d_up ? f : n, d_up ? h : f)) return rc;

  const int64_t nh = (h + 255) / 256;
  GatedBwdParams p = {};
  p.N = static_cast<int>(n);
  p.H = static_cast<int>(h);
  p.F = static_cast<int>(f);
  p.splits = d_x ? L.splits : 1;
  p.n_dx = d_x ? static_cast<int>((n + 255) / 256 * nh) * L.splits : 0;
  p.dx_stages = L.stages;
  p.n_dw = n_weights * static_cast<int>((f + 255) / 256 * nh);
  p.dw_first = d_gate ? 0 : 1;
  p.rows_pad = L.rows_pad;
  p.err = d->err_ptr;
  p.timeout_ns = wait_timeout_ns();
  if (int rc = bf16 ? launch_gated_bwd<true>(maps, p, d->sms, st) : launch_gated_bwd<false>(maps, p, d->sms, st))
    return rc;
  if (!d_x || L.splits == 1) return LMCE_OK;
  const long long total = n * h / 4, stride = static_cast<long long>(L.rows_pad) * h / 4;
  const int sgrid = static_cast<int>(std::min<long long>((total + 255) / 256, d->sms * 8ll));
  if (bf16)
    gated_dx_sum_kernel<true><<<sgrid, 256, 0, st>>>(reinterpret_cast<const float4*>(part), L.splits, stride, total,
                                                     static_cast<uint2*>(d_x));
  else
    gated_dx_sum_kernel<false><<<sgrid, 256, 0, st>>>(reinterpret_cast<const float4*>(part), L.splits, stride, total,
                                                      static_cast<uint2*>(d_x));
  return launched();
}

}  // extern "C"
