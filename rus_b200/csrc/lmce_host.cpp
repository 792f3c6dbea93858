// Host side of the operators around the head: argument checks, allocation and the autograd
// nodes of lmce_add_rmsnorm, lmce_gated_linear and their e4m3 forms, and the walk over the
// gradients of lmce_clip_grad_norm, calling the C ABI of liblmce.so. In C++ because these
// operators are short: a Python autograd function that does nothing takes 73-91 us a step on the
// hosts of a B200, where the kernels of a small batch take 17 (one B200, residual norm with
// backward, 2048 x 1536: 118 us a call through Python, 80-82 us here; 392 gradients to clip: 157 us
// of host work in Python, 28 us here).
//
// Every function returns nothing where an argument is not one it takes: the Python module
// then says what is wrong with it (norm.py, gated.py, clip.py). Errors of the library
// become the package's LmceError, in a backward as well.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <dlfcn.h>

#include <cmath>
#include <cstdlib>
#include <functional>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "lmce.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

#define LMCE_HOST_ENTRIES(X)                                                                        \
  X(lmce_last_error) X(lmce_device_error) X(lmce_add_rmsnorm) X(lmce_add_rmsnorm_e4m3)               \
  X(lmce_add_rmsnorm_bwd_workspace_bytes) X(lmce_add_rmsnorm_backward) X(lmce_gated_saved_bytes)     \
  X(lmce_gated_linear) X(lmce_gated_linear_e4m3) X(lmce_gated_bwd_workspace_bytes)                   \
  X(lmce_gated_backward) X(lmce_clip_grad_workspace_bytes) X(lmce_clip_grad_norm)

struct Lib {
#define X(name) decltype(&::name) name = nullptr;
  LMCE_HOST_ENTRIES(X)
#undef X
} lib;

// An LMCE_ERR_* status with the library's message.
struct Status : std::runtime_error {
  int code;
  Status(int code_, const std::string& text) : std::runtime_error(text), code(code_) {}
};

py::object& error_type() {
  static py::object* type = new py::object();  // outlives the interpreter's teardown
  return *type;
}

void check(int rc) {
  if (rc != LMCE_OK) throw Status(rc, lib.lmce_last_error());
}

// With LMCE_DEBUG set: wait for the current stream, which the library's own read of the error word
// does not when the stream is not the default one, and raise what a kernel recorded. Not while a
// graph is captured: nothing has run then.
void check_device() {
  const char* s = std::getenv("LMCE_DEBUG");
  if (s == nullptr || s[0] == '\0' || (s[0] == '0' && s[1] == '\0')) return;
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return;
  c10::cuda::getCurrentCUDAStream().synchronize();
  const int rc = lib.lmce_device_error(1);
  if (rc != LMCE_OK) throw Status(rc, "reported by a kernel");
}

// What a backward raises: autograd hands a Python exception on as it is, so the caller sees the
// package's error there too.
[[noreturn]] void raise_in_backward(const Status& e) {
  const py::gil_scoped_acquire gil;
  PyErr_SetObject(error_type().ptr(), error_type()(e.code, e.what()).ptr());
  python_error raised;
  raised.persist();
  throw raised;
}

void no_second_order(const char* who) {
  // autograd runs a backward in grad mode only to differentiate it again
  if (at::GradMode::is_enabled())
    throw Status(LMCE_ERR_UNSUPPORTED, std::string(who) + ": no second derivative (create_graph=True)");
}

// None of these operators has a forward-mode derivative, and the plain path would drop a tangent.
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

void no_tangents(const char* who, std::initializer_list<std::reference_wrapper<const Tensor>> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : tensors)
    if (dual(t)) throw Status(LMCE_ERR_UNSUPPORTED, std::string(who) + ": no forward-mode derivative");
}

// A tracer sees the allocation of an output, not the kernel that fills it: what it records would
// return memory as it was found.
void no_trace(const char* who) {
  using Key = c10::impl::TorchDispatchModeKey;
  bool traced = at::tracer::impl::is_dispatch_enabled() ||
                c10::impl::tls_is_dispatch_key_included(at::DispatchKey::PreDispatch);
  if (!traced && c10::impl::TorchDispatchModeTLS::any_modes_set())
    traced = c10::impl::TorchDispatchModeTLS::get_mode(Key::PROXY).has_value() ||
             c10::impl::TorchDispatchModeTLS::get_mode(Key::FAKE).has_value();
  if (traced)
    throw Status(LMCE_ERR_UNSUPPORTED,
                 std::string(who) + ": cannot be traced (torch.jit.trace, make_fx, torch.export, fake tensors)");
}

bool is16(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int dtype_code(at::ScalarType t) { return t == at::kHalf ? LMCE_DTYPE_F16 : LMCE_DTYPE_BF16; }

// `t` contiguous and on a 16-byte boundary (a copy where it is not).
Tensor rows(const Tensor& t) {
  const Tensor c = t.is_contiguous() ? t : t.contiguous();
  const void* p = c.data_ptr();
  // the library would take the null pointer for an argument left out
  if (p == nullptr && c.numel() > 0)
    throw Status(LMCE_ERR_UNSUPPORTED, "a tensor that holds no memory (a wrapper of another, or zeros without storage)");
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 ? c : c.clone(at::MemoryFormat::Contiguous);
}

// A saved tensor as a hook of torch.autograd.graph.saved_tensors_hooks gives it back: its strides may
// be others than those that were saved; with another device, type or size it is refused, since the
// kernels go by those of the gradient.
Tensor unpacked(const Tensor& t, const Tensor& grad, at::ScalarType type, at::IntArrayRef sizes) {
  if (!t.defined() || t.layout() != at::kStrided || t.device() != grad.device() || t.scalar_type() != type ||
      t.sizes() != sizes)
    throw Status(LMCE_ERR_INVALID_ARGUMENT, "a saved tensor came back with another device, type or size");
  return rows(t);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
bool usable(const Tensor& t) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided; }

Tensor bytes(const Tensor& like, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte).requires_grad(false));
}

// ------------------------------------------------------ residual add + norm ---

bool norm_args(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& w) {
  if (!usable(x) || !usable(w) || !is16(x.scalar_type()) || x.dim() == 0 || w.dim() != 1) return false;
  const int64_t h = x.size(-1);
  if (w.scalar_type() != x.scalar_type() || w.device() != x.device() || w.size(0) != h) return false;
  if (h % 8 != 0 || h <= 0 || h > 16384) return false;
  return !residual || (usable(*residual) && residual->scalar_type() == x.scalar_type() &&
                       residual->device() == x.device() && residual->sizes() == x.sizes());
}

struct NormOut {
  Tensor y, s, w, rstd;
};

NormOut norm_forward(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double eps,
                     bool keep_rstd) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t h = x.size(-1);
  const Tensor xc = rows(x), rc = residual ? rows(*residual) : Tensor();
  const int64_t n = xc.numel() / h;
  NormOut o;
  o.w = rows(weight);
  o.y = at::empty_like(xc);
  o.s = residual ? at::empty_like(xc) : xc;
  if (keep_rstd) o.rstd = at::empty({n}, xc.options().dtype(at::kFloat));
  if (n > 0)
    check(lib.lmce_add_rmsnorm(xc.data_ptr(), ptr(rc), o.w.data_ptr(), static_cast<float>(eps), n, h,
                               dtype_code(x.scalar_type()), residual ? o.s.data_ptr() : nullptr, o.y.data_ptr(),
                               static_cast<float*>(ptr(o.rstd)), stream(x)));
  return o;
}

// Inputs x, residual (optional), weight, eps; outputs y and, with a residual, s.
struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual,
                               const Tensor& weight, double eps) {
    NormOut o = norm_forward(x, residual, weight, eps, true);
    ctx->save_for_backward({o.s, o.w, o.rstd});
    ctx->set_materialize_grads(false);
    ctx->saved_data["residual"] = residual.has_value();
    if (residual) return {o.y, o.s};
    return {o.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    try {
      return gradients(ctx, grads);
    } catch (const Status& e) {
      raise_in_backward(e);
    }
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    no_trace("add_rms_norm");
    no_second_order("add_rms_norm");
    const auto saved = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    // edges are counted over the tensors there are
    const bool want_x = ctx->needs_input_grad(0), want_r = residual && ctx->needs_input_grad(1);
    const bool want_w = ctx->needs_input_grad(residual ? 2 : 1);
    const Tensor dy = grads[0], ds = residual ? grads[1] : Tensor();
    if (!dy.defined() && !ds.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor& d = dy.defined() ? dy : ds;  // both have the shape and type of s
    const int64_t h = d.size(-1), n = d.numel() / h;
    const c10::cuda::CUDAGuard guard(d.device());
    const Tensor s = unpacked(saved[0], d, d.scalar_type(), d.sizes());
    const Tensor w = unpacked(saved[1], d, d.scalar_type(), {h});
    const Tensor rstd = unpacked(saved[2], d, at::kFloat, {n});
    Tensor dx, dw, ws;
    if (want_x || want_r) dx = at::empty_like(s);
    const bool run_w = want_w && dy.defined() && n > 0;
    if (want_w) dw = run_w ? at::empty_like(w) : at::zeros_like(w);
    if (n > 0 && (dx.defined() || run_w)) {
      const Tensor g = dy.defined() ? rows(dy) : Tensor(), gs = ds.defined() ? rows(ds) : Tensor();
      const size_t need = run_w ? lib.lmce_add_rmsnorm_bwd_workspace_bytes(n, h) : 0;
      if (run_w) ws = bytes(s, need);
      check(lib.lmce_add_rmsnorm_backward(ptr(g), ptr(gs), s.data_ptr(), w.data_ptr(),
                                          static_cast<const float*>(rstd.data_ptr()), n, h,
                                          dtype_code(s.scalar_type()), ptr(dx), run_w ? dw.data_ptr() : nullptr,
                                          ptr(ws), need, stream(s)));
    }
    return {want_x ? dx : Tensor(), want_r ? dx : Tensor(), dw, Tensor()};
  }
};

bool records(const Tensor& a, const Tensor& b, const std::optional<Tensor>& c) {
  return at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad() || (c && c->requires_grad()));
}

std::optional<std::tuple<Tensor, Tensor>> add_rms_norm(const Tensor& x, const std::optional<Tensor>& residual,
                                                       const Tensor& weight, double eps) {
  no_trace("add_rms_norm");
  no_tangents("add_rms_norm", {x, residual ? *residual : x, weight});
  if (!norm_args(x, residual, weight)) return std::nullopt;
  if (records(x, weight, residual)) {
    variable_list out = NormNode::apply(x, residual, weight, eps);
    return std::make_tuple(out[0], residual ? out[1] : x);
  }
  NormOut o = norm_forward(x, residual, weight, eps, false);
  return std::make_tuple(o.y, residual ? o.s : x);
}

std::optional<std::tuple<Tensor, Tensor, Tensor>> add_rms_norm_e4m3(const Tensor& x,
                                                                    const std::optional<Tensor>& residual,
                                                                    const Tensor& weight, double eps) {
  no_trace("add_rms_norm_e4m3");
  no_tangents("add_rms_norm_e4m3", {x, residual ? *residual : x, weight});
  if (!norm_args(x, residual, weight) || records(x, weight, residual)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t h = x.size(-1);
  const Tensor xc = rows(x), rc = residual ? rows(*residual) : Tensor(), w = rows(weight);
  const int64_t n = xc.numel() / h;
  const auto plain = xc.options().requires_grad(false);
  Tensor q = at::empty(x.sizes(), plain.dtype(at::kFloat8_e4m3fn));
  Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), plain.dtype(at::kFloat));
  Tensor s = residual ? at::empty_like(xc) : x;
  if (n > 0)
    check(lib.lmce_add_rmsnorm_e4m3(xc.data_ptr(), ptr(rc), w.data_ptr(), static_cast<float>(eps), n, h,
                                    dtype_code(x.scalar_type()), residual ? s.data_ptr() : nullptr, q.data_ptr(),
                                    static_cast<float*>(scale.data_ptr()), stream(x)));
  return std::make_tuple(q, scale, s);
}

// -------------------------------------------------------- gated projection ---

bool gated_args(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t step) {
  if (!usable(x) || !usable(wg) || !usable(wu) || x.dim() == 0 || wg.dim() != 2 || wu.sizes() != wg.sizes())
    return false;
  const int64_t f = wg.size(0), h = wg.size(1);
  return wg.scalar_type() == x.scalar_type() && wu.scalar_type() == x.scalar_type() && wg.device() == x.device() &&
         wu.device() == x.device() && x.size(-1) == h && f > 0 && f % 64 == 0 && h > 0 && h % step == 0;
}

std::vector<int64_t> out_sizes(const Tensor& x, int64_t f) {
  std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = f;
  return sizes;
}

struct GatedOut {
  Tensor h, x, wg, wu, saved;
};

GatedOut gated_forward(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, int64_t act, bool save) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t f = w_gate.size(0), h = w_gate.size(1);
  GatedOut o;
  o.x = rows(x);
  o.wg = rows(w_gate);
  o.wu = rows(w_up);
  const int64_t n = o.x.numel() / h;
  o.h = at::empty(out_sizes(x, f), o.x.options().requires_grad(false));
  if (n > 0) {
    if (save) o.saved = bytes(o.x, lib.lmce_gated_saved_bytes(n, f));
    check(lib.lmce_gated_linear(o.x.data_ptr(), o.wg.data_ptr(), o.wu.data_ptr(), n, h, f,
                                dtype_code(x.scalar_type()), static_cast<int>(act), o.h.data_ptr(), ptr(o.saved),
                                stream(x)));
    check_device();
  }
  return o;
}

struct GatedNode : torch::autograd::Function<GatedNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                        int64_t act) {
    GatedOut o = gated_forward(x, w_gate, w_up, act, true);
    ctx->save_for_backward({o.x, o.wg, o.wu, o.saved});
    ctx->saved_data["act"] = act;
    return o.h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    try {
      return gradients(ctx, grads);
    } catch (const Status& e) {
      raise_in_backward(e);
    }
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    no_trace("gated_linear");
    no_second_order("gated_linear");
    const auto saved = ctx->get_saved_variables();
    const Tensor& d = grads[0];
    const c10::cuda::CUDAGuard guard(d.device());
    const at::ScalarType type = d.scalar_type();
    const int64_t f = d.size(-1), n = d.numel() / f, h = saved[1].size(-1);
    const Tensor x = unpacked(saved[0], d, type, out_sizes(d, h));
    const Tensor wg = unpacked(saved[1], d, type, {f, h}), wu = unpacked(saved[2], d, type, {f, h});
    const bool want_x = ctx->needs_input_grad(0), want_g = ctx->needs_input_grad(1),
               want_u = ctx->needs_input_grad(2);
    const auto make = [&](bool want, const Tensor& like) {
      return !want ? Tensor() : n > 0 ? at::empty_like(like) : at::zeros_like(like);
    };
    Tensor dx = make(want_x, x), dg = make(want_g, wg), du = make(want_u, wu);
    if (n > 0 && (want_x || want_g || want_u)) {
      const Tensor kept =
          unpacked(saved[3], d, at::kByte, {static_cast<int64_t>(lib.lmce_gated_saved_bytes(n, f))});
      const Tensor g = rows(d);
      const size_t need = lib.lmce_gated_bwd_workspace_bytes(n, h, f, want_x, want_g + want_u);
      const Tensor ws = bytes(x, need);
      check(lib.lmce_gated_backward(g.data_ptr(), kept.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(),
                                    n, h, f, dtype_code(x.scalar_type()),
                                    static_cast<int>(ctx->saved_data["act"].toInt()), ptr(dx), ptr(dg), ptr(du),
                                    ws.data_ptr(), need, stream(x)));
      check_device();
    }
    return {dx, dg, du, Tensor()};
  }
};

std::optional<Tensor> gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, int64_t act) {
  no_trace("gated_linear");
  no_tangents("gated_linear", {x, w_gate, w_up});
  if (!gated_args(x, w_gate, w_up, 64) || !is16(x.scalar_type())) return std::nullopt;
  if (records(x, w_gate, w_up)) return GatedNode::apply(x, w_gate, w_up, act);
  return gated_forward(x, w_gate, w_up, act, false).h;
}

std::optional<Tensor> gated_linear_e4m3(const Tensor& x, const Tensor& x_scale, const Tensor& w_gate,
                                        const Tensor& gate_scale, const Tensor& w_up, const Tensor& up_scale,
                                        int64_t act, at::ScalarType out_dtype) {
  no_trace("gated_linear_e4m3");
  no_tangents("gated_linear_e4m3", {x, x_scale, w_gate, gate_scale, w_up, up_scale});
  if (!gated_args(x, w_gate, w_up, 128) || x.scalar_type() != at::kFloat8_e4m3fn || !is16(out_dtype))
    return std::nullopt;
  const int64_t f = w_gate.size(0), h = w_gate.size(1);
  const auto scale_ok = [&](const Tensor& t, at::IntArrayRef sizes) {
    return usable(t) && t.scalar_type() == at::kFloat && t.sizes() == sizes && t.device() == x.device();
  };
  if (!scale_ok(x_scale, x.sizes().slice(0, x.dim() - 1)) || !scale_ok(gate_scale, {f}) || !scale_ok(up_scale, {f}) ||
      records(x_scale, gate_scale, up_scale) || records(x, w_gate, w_up))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor xc = rows(x), wg = rows(w_gate), wu = rows(w_up);
  const Tensor sx = rows(x_scale), sg = rows(gate_scale), su = rows(up_scale);
  const int64_t n = xc.numel() / h;
  Tensor out = at::empty(out_sizes(x, f), x.options().dtype(out_dtype).requires_grad(false));
  if (n > 0) {
    check(lib.lmce_gated_linear_e4m3(xc.data_ptr(), static_cast<const float*>(sx.data_ptr()), wg.data_ptr(),
                                     static_cast<const float*>(sg.data_ptr()), wu.data_ptr(),
                                     static_cast<const float*>(su.data_ptr()), n, h, f, dtype_code(out_dtype),
                                     static_cast<int>(act), out.data_ptr(), stream(x)));
    check_device();
  }
  return out;
}

// ------------------------------------------------------- gradient clipping ---

// The gradients of a list of parameters, or a list of gradients. The common case: dense contiguous
// fp16, bf16 or fp32 gradients on one device, at least one and none shared. Nothing for any other,
// and nothing is launched then; what the library says against a list of gradients is raised.
std::optional<Tensor> clip_grad_norm(const py::list& tensors, double max_norm, bool of_parameters) {
  no_trace("clip_grad_norm_");
  std::vector<void*> ptrs;
  std::vector<int64_t> numels;
  std::vector<int32_t> dtypes;
  std::vector<at::TensorImpl*> impls;
  Tensor first;
  const size_t count = tensors.size();
  ptrs.reserve(count);
  numels.reserve(count);
  dtypes.reserve(count);
  impls.reserve(count);
  for (size_t i = 0; i < count; ++i) {
    PyObject* o = PyList_GET_ITEM(tensors.ptr(), static_cast<Py_ssize_t>(i));
    if (!THPVariable_Check(o)) return std::nullopt;
    const Tensor& t0 = THPVariable_Unpack(o);
    const Tensor& g = of_parameters ? t0.grad() : t0;
    if (!g.defined()) continue;
    no_tangents("clip_grad_norm_", {g});
    const at::ScalarType t = g.scalar_type();
    if (!usable(g) || !(is16(t) || t == at::kFloat) || !g.is_contiguous()) return std::nullopt;
    if (!first.defined())
      first = g;
    else if (g.device() != first.device())
      return std::nullopt;
    ptrs.push_back(g.data_ptr());
    numels.push_back(g.numel());
    dtypes.push_back(t == at::kFloat ? LMCE_DTYPE_F32 : dtype_code(t));
    impls.push_back(g.unsafeGetTensorImpl());
  }
  if (!first.defined()) return std::nullopt;
  const c10::cuda::CUDAGuard guard(first.device());
  Tensor total = at::empty({}, first.options().dtype(at::kFloat).requires_grad(false));
  const int64_t n = static_cast<int64_t>(ptrs.size());
  const size_t need = lib.lmce_clip_grad_workspace_bytes(n);
  const Tensor ws = bytes(first, need);
  const int rc = lib.lmce_clip_grad_norm(ptrs.data(), numels.data(), dtypes.data(), n, static_cast<float>(max_norm),
                                         static_cast<float*>(total.data_ptr()), ws.data_ptr(), need, stream(first));
  // refused before any launch: a parameter listed twice, say, which the Python module sorts out
  if (rc == LMCE_ERR_INVALID_ARGUMENT && of_parameters) return std::nullopt;
  check(rc);
  // an in-place change that autograd has to see: a graph that saved a gradient must not use it scaled
  if (static_cast<float>(max_norm) != INFINITY)
    for (at::TensorImpl* g : impls)
      if (!g->is_inference()) g->bump_version();
  return total;
}

void init(const std::string& library, const py::object& error) {
  void* handle = dlopen(library.c_str(), RTLD_NOW);
  if (handle == nullptr) throw std::runtime_error(dlerror());
#define X(name)                                                                \
  lib.name = reinterpret_cast<decltype(&::name)>(dlsym(handle, #name));        \
  if (lib.name == nullptr) throw std::runtime_error("liblmce.so has no " #name);
  LMCE_HOST_ENTRIES(X)
#undef X
  error_type() = error;
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.attr("torch_version") = TORCH_VERSION;
  m.def("init", &init);
  using Release = py::call_guard<py::gil_scoped_release>;
  m.def("add_rms_norm", &add_rms_norm, Release());
  m.def("add_rms_norm_e4m3", &add_rms_norm_e4m3, Release());
  m.def("gated_linear", &gated_linear, Release());
  m.def("gated_linear_e4m3", &gated_linear_e4m3, Release());
  m.def("clip_grad_norm", &clip_grad_norm);
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Status& e) {
      const py::object value = error_type()(e.code, e.what());
      PyErr_SetObject(error_type().ptr(), value.ptr());
    }
  });
}
