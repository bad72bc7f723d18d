// Torch binding of the selective-mixer operators: argument checks, allocation,
// autograd and the calls through the C ABI of libspikegpt_wkv.so (include/
// spikegpt_wkv.h), registered in the spikegpt_b200 namespace.
//
// These operators run every few microseconds in a generation loop and four times a
// block in training, where a Python autograd function costs more than their kernels
// (a layer norm of 8192 x 512 forward and backward: 125 us of host time in Python, 74
// here, 50 of them the autograd engine's own). Each has a forward and a backward
// operator with CUDA and Meta kernels, and one that differentiates, so eager calls,
// CUDA graphs and torch.compile take the same path. The library's functions are looked
// up in the file that bind_library names, the one the ctypes binding uses.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <atomic>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "spikegpt_wkv.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------ the C ABI

struct Library {
  decltype(&wkv_last_error) last_error;
  decltype(&causal_conv_forward) conv_forward;
  decltype(&causal_conv_workspace_size) conv_workspace;
  decltype(&causal_conv_backward) conv_backward;
  decltype(&causal_conv_step) conv_step;
  decltype(&selective_scan_state_size) scan_state;
  decltype(&selective_scan_forward_workspace_size) scan_forward_workspace;
  decltype(&selective_scan_forward) scan_forward;
  decltype(&selective_scan_backward_workspace_size) scan_backward_workspace;
  decltype(&selective_scan_backward) scan_backward;
  decltype(&selective_scan_step) scan_step;
  decltype(&layer_norm_forward) norm_forward;
  decltype(&layer_norm_workspace_size) norm_workspace;
  decltype(&layer_norm_backward) norm_backward;
  decltype(&q4_matvec) q4;
};
Library g_lib;
std::atomic<bool> g_bound{false};

bool bind_library(std::string path) {
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (g_bound.load()) return true;
  void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(handle != nullptr, "spikegpt_b200: cannot load ", path, ": ", dlerror());
  auto find = [&](auto& f, const char* name) {
    void* p = dlsym(handle, name);
    TORCH_CHECK(p != nullptr, "spikegpt_b200: ", path, " lacks ", name);
    f = reinterpret_cast<std::decay_t<decltype(f)>>(p);
  };
  find(g_lib.last_error, "wkv_last_error");
  find(g_lib.conv_forward, "causal_conv_forward");
  find(g_lib.conv_workspace, "causal_conv_workspace_size");
  find(g_lib.conv_backward, "causal_conv_backward");
  find(g_lib.conv_step, "causal_conv_step");
  find(g_lib.scan_state, "selective_scan_state_size");
  find(g_lib.scan_forward_workspace, "selective_scan_forward_workspace_size");
  find(g_lib.scan_forward, "selective_scan_forward");
  find(g_lib.scan_backward_workspace, "selective_scan_backward_workspace_size");
  find(g_lib.scan_backward, "selective_scan_backward");
  find(g_lib.scan_step, "selective_scan_step");
  find(g_lib.norm_forward, "layer_norm_forward");
  find(g_lib.norm_workspace, "layer_norm_workspace_size");
  find(g_lib.norm_backward, "layer_norm_backward");
  find(g_lib.q4, "q4_matvec");
  g_bound.store(true);
  return true;
}

const Library& lib() {
  TORCH_CHECK(g_bound.load(std::memory_order_acquire), "spikegpt_b200: bind_library has not been called");
  return g_lib;
}

void check(int status, const char* where) {
  TORCH_CHECK(status == WKV_OK, where, " (status ", status, "): ", lib().last_error());
}

// -------------------------------------------------------------- helpers

int code_of(const char* name, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return WKV_DTYPE_F32;
    case at::kBFloat16: return WKV_DTYPE_BF16;
    case at::kHalf: return WKV_DTYPE_F16;
    default:
      TORCH_CHECK_VALUE(false, "unsupported dtype ", t.scalar_type(), " of ", name,
                        "; expected float32, bfloat16 or float16");
  }
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
const void* ptr(const OptTensor& t) { return has(t) ? t->const_data_ptr() : nullptr; }
const float* fptr(const OptTensor& t) { return static_cast<const float*>(ptr(t)); }
const float* fptr(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }
float* fout(Tensor& t) { return t.numel() ? static_cast<float*>(t.mutable_data_ptr()) : nullptr; }
void* out_ptr(Tensor& t, bool on) { return on ? t.mutable_data_ptr() : nullptr; }
Tensor opt(const OptTensor& t) { return has(t) ? *t : Tensor(); }
OptTensor some(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// Sizes and strides as numbers, also while a graph is traced with symbolic ones.
int64_t size_of(const Tensor& t, int64_t d) { return t.sym_size(d).guard_int(__FILE__, __LINE__); }
int64_t stride_of(const Tensor& t, int64_t d) { return t.sym_stride(d).guard_int(__FILE__, __LINE__); }
std::vector<int64_t> shape_of(const Tensor& t) {
  std::vector<int64_t> r;
  for (int64_t d = 0; d < t.dim(); ++d) r.push_back(size_of(t, d));
  return r;
}
void need_shape(const char* name, const OptTensor& t, at::IntArrayRef shape) {
  if (!has(t)) return;
  bool same = t->dim() == (int64_t)shape.size();
  for (int64_t d = 0; same && d < t->dim(); ++d) same = size_of(*t, d) == shape[d];
  TORCH_CHECK_VALUE(same, name, " must have shape ", shape, "; got ", shape_of(*t));
}
void need_dtype(const char* name, const OptTensor& t, at::ScalarType type, const char* of) {
  if (has(t))
    TORCH_CHECK_VALUE(t->scalar_type() == type, name, " must have the dtype of ", of, " (", type, "); got ",
                      t->scalar_type());
}
void need_cuda(const char* op, const Tensor& first, std::initializer_list<const OptTensor*> others) {
  TORCH_CHECK_NOT_IMPLEMENTED(first.is_cuda() || first.is_meta(), "spikegpt_b200.", op, " runs on CUDA tensors only");
  for (const OptTensor* t : others)
    if (has(*t))
      TORCH_CHECK_VALUE((*t)->device() == first.device(), "all tensors of ", op, " must be on ", first.device(),
                        "; got one on ", (*t)->device());
}
// A parameter as the kernels read it: float32 and contiguous.
Tensor parameter(const Tensor& t) {
  if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
  return t.to(at::kFloat).contiguous();
}
OptTensor parameter(const OptTensor& t) { return has(t) ? OptTensor(parameter(*t)) : OptTensor(); }
// Unit stride of the last index (a copy only where it lacks that).
Tensor rows(const Tensor& t) {
  return !t.defined() || stride_of(t, -1) == 1 || size_of(t, -1) == 1 ? t : t.contiguous();
}
OptTensor rows(const OptTensor& t) { return has(t) ? OptTensor(rows(*t)) : OptTensor(); }
OptTensor lengths_of(const OptTensor& t, int64_t b) {
  if (!has(t)) return OptTensor();
  TORCH_CHECK_VALUE(t->dim() == 1 && size_of(*t, 0) == b && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong),
                    "lengths must be int32 or int64 of shape [", b, "]; got ", t->scalar_type(), " ", shape_of(*t));
  return t->scalar_type() == at::kLong ? t->clamp(0, INT_MAX).to(at::kInt).contiguous() : t->contiguous();
}
int64_t stride0(const OptTensor& t, int d) { return has(t) ? t->stride(d) : 0; }
Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, like.options().dtype(type));
}
Tensor empty(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options()); }
bool requires_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool requires_grad(const OptTensor& t) { return t.has_value() && requires_grad(*t); }
template <class... Ts>
bool wants_grad(const Ts&... ts) {
  return at::GradMode::is_enabled() && (requires_grad(ts) || ...);
}
template <class... Ts>
void no_grad_only(const char* op, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad(ts...), "spikegpt_b200.", op,
                              " has no gradient; call it under torch.no_grad()");
}
// Forward-mode derivatives (dual tensors, torch.func.jvp) are not there; without this a
// tangent would be lost below autograd without a word.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <class... Ts>
void no_tangents(const char* op, const Ts&... ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(ts) || ...), "spikegpt_b200.", op, " has no forward-mode derivative");
}
// A call of a backward operator. While a graph of the gradients is recorded
// (create_graph) it goes through their Autograd kernel, which gives them a node that
// raises: there are no second derivatives.
template <class F>
auto backward_call(const char* op, const Tensor& g, const OptTensor& other, F&& call) {
  no_tangents(op, g, other);
  if (at::GradMode::is_enabled()) return call();
  at::AutoDispatchBelowADInplaceOrView below;
  return call();
}
template <class F>
auto typed(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// ----------------------------------------------------------- layer norm

using Tensor3 = std::tuple<Tensor, Tensor, Tensor>;

Tensor3 norm_fwd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t n = x.size(0), c = x.size(1);
  Tensor y = empty(x, {n, c}), mean = empty(x, {n}, at::kFloat), rstd = empty(x, {n}, at::kFloat);
  check(lib().norm_forward(code_of("x", x), x.const_data_ptr(), fptr(weight), fptr(bias), y.mutable_data_ptr(),
                           fout(mean), fout(rstd), n, c, x.stride(0), (float)eps, stream_of(x)),
        "layer_norm_forward");
  return {y, mean, rstd};
}
Tensor3 norm_fwd_meta(const Tensor& x, const OptTensor&, const OptTensor&, double) {
  const c10::SymInt n = x.sym_size(0);
  const auto f32 = x.options().dtype(at::kFloat);
  return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint({n}, f32), at::empty_symint({n}, f32)};
}
Tensor3 norm_bwd(const Tensor& g_, const Tensor& x, const OptTensor& weight, const Tensor& mean, const Tensor& rstd,
                 bool want_w, bool want_b) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor g = rows(g_);
  const int64_t n = x.size(0), c = x.size(1);
  const int code = code_of("x", x);
  Tensor gx = empty(x, {n, c}), gw = empty(x, {want_w ? c : 0}, at::kFloat), gb = empty(x, {want_b ? c : 0}, at::kFloat);
  const int64_t nws = (int64_t)lib().norm_workspace(code, n, c);
  Tensor ws = empty(x, {nws}, at::kByte);
  check(lib().norm_backward(code, g.const_data_ptr(), x.const_data_ptr(), fptr(weight), fptr(mean), fptr(rstd),
                            gx.mutable_data_ptr(), fout(gw), fout(gb), ws.mutable_data_ptr(), nws, n, c, g.stride(0),
                            x.stride(0), stream_of(x)),
        "layer_norm_backward");
  return {gx, gw, gb};
}
Tensor3 norm_bwd_meta(const Tensor&, const Tensor& x, const OptTensor&, const Tensor&, const Tensor&, bool want_w,
                      bool want_b) {
  const auto f32 = x.options().dtype(at::kFloat);
  const c10::SymInt c = x.sym_size(1), none = 0;
  return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint({want_w ? c : none}, f32),
          at::empty_symint({want_b ? c : none}, f32)};
}

const auto& norm_fwd_op() {
  static const auto op = typed<decltype(norm_fwd)>("spikegpt_b200::layer_norm_fwd");
  return op;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, mean, rstd] = norm_fwd_op().call(x, w, b, eps);
    ctx->save_for_backward({x, opt(w), mean, rstd});
    ctx->saved_data["w"] = has(w) && w->requires_grad();
    ctx->saved_data["b"] = has(b) && b->requires_grad();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = typed<decltype(norm_bwd)>("spikegpt_b200::layer_norm_bwd");
    const auto saved = ctx->get_saved_variables();
    const bool want_w = ctx->saved_data["w"].toBool(), want_b = ctx->saved_data["b"].toBool();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor g = grads[0].to(saved[0].scalar_type());
    auto [gx, gw, gb] = backward_call("layer_norm", g, {}, [&] {
      return op.call(g, saved[0], some(saved[1]), saved[2], saved[3], want_w, want_b);
    });
    return {gx, want_w ? gw : Tensor(), want_b ? gb : Tensor(), Tensor()};
  }
};

Tensor norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  const int64_t c = size_of(x, -1);
  TORCH_CHECK_VALUE(c >= 1 && c <= 16384, "layer_norm takes rows of 1 to 16384 values; got ", c);
  code_of("x", x);
  need_shape("weight", weight, {c});
  need_shape("bias", bias, {c});
  need_cuda("layer_norm", x, {&weight, &bias});
  no_tangents("layer_norm", x, weight, bias);
  const OptTensor w = parameter(weight), b = parameter(bias);
  const Tensor flat = rows(x.dim() == 2 ? x : x.reshape({-1, c}));
  Tensor y;
  if (wants_grad(flat, w, b)) {
    y = LayerNorm::apply(flat, w, b, eps);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    y = std::get<0>(norm_fwd_op().call(flat, w, b, eps));
  }
  return x.dim() == 2 ? y : y.view_symint(x.sym_sizes());
}

// --------------------------------------------------- causal convolution

using Tensor2 = std::tuple<Tensor, Tensor>;
using Tensor4 = std::tuple<Tensor, Tensor, Tensor, Tensor>;

Tensor2 conv_fwd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& window,
                 const OptTensor& lengths, bool silu, bool want_window) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t b = x.size(0), t = x.size(1), c = x.size(2), w = weight.size(1);
  Tensor y = empty(x, {b, t, c}), next = want_window ? empty(x, {b, w - 1, c}) : empty(x, {0});
  check(lib().conv_forward(code_of("x", x), x.const_data_ptr(), fptr(weight), fptr(bias), ptr(window),
                           static_cast<const int*>(ptr(lengths)), y.mutable_data_ptr(), out_ptr(next, want_window), b,
                           t, c, (int)w, x.stride(0), x.stride(1), silu, stream_of(x)),
        "causal_conv_forward");
  return {y, next};
}
Tensor2 conv_fwd_meta(const Tensor& x, const Tensor& weight, const OptTensor&, const OptTensor&, const OptTensor&,
                      bool, bool want_window) {
  const c10::SymInt w1 = weight.sym_size(1) - 1;
  return {at::empty_symint(x.sym_sizes(), x.options()),
          want_window ? at::empty_symint({x.sym_size(0), w1, x.sym_size(2)}, x.options()) : empty(x, {0})};
}
Tensor4 conv_bwd(const Tensor& g_, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                 const OptTensor& window, const OptTensor& lengths, bool silu, bool want_window) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor g = rows(g_);
  const int64_t b = x.size(0), t = x.size(1), c = x.size(2), w = weight.size(1);
  Tensor gx = empty(x, {b, t, c}), gw = empty(x, {c, w}, at::kFloat), gb = empty(x, {has(bias) ? c : 0}, at::kFloat);
  Tensor gwin = want_window ? empty(x, {b, w - 1, c}) : empty(x, {0});
  const int64_t nws = (int64_t)lib().conv_workspace(b, t, c, (int)w);
  Tensor ws = empty(x, {nws}, at::kByte);
  check(lib().conv_backward(code_of("x", x), g.const_data_ptr(), x.const_data_ptr(), fptr(weight), fptr(bias),
                            ptr(window), static_cast<const int*>(ptr(lengths)), gx.mutable_data_ptr(),
                            static_cast<float*>(gw.mutable_data_ptr()), fout(gb), out_ptr(gwin, want_window),
                            ws.mutable_data_ptr(), nws, b, t, c, (int)w, g.stride(0), g.stride(1), x.stride(0),
                            x.stride(1), silu, stream_of(x)),
        "causal_conv_backward");
  return {gx, gw, gb, gwin};
}
Tensor4 conv_bwd_meta(const Tensor&, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor&,
                      const OptTensor&, bool, bool want_window) {
  const c10::SymInt w1 = weight.sym_size(1) - 1, none = 0;
  const auto f32 = x.options().dtype(at::kFloat);
  return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint(weight.sym_sizes(), f32),
          at::empty_symint({has(bias) ? x.sym_size(2) : none}, f32),
          want_window ? at::empty_symint({x.sym_size(0), w1, x.sym_size(2)}, x.options()) : empty(x, {0})};
}

const auto& conv_fwd_op() {
  static const auto op = typed<decltype(conv_fwd)>("spikegpt_b200::causal_conv_fwd");
  return op;
}

struct CausalConv : torch::autograd::Function<CausalConv> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                        const OptTensor& window, const OptTensor& lengths, bool silu) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({x, weight, opt(bias), opt(window), opt(lengths)});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["window"] = has(window) && window->requires_grad();
    return std::get<0>(conv_fwd_op().call(x, weight, bias, window, lengths, silu, false));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = typed<decltype(conv_bwd)>("spikegpt_b200::causal_conv_bwd");
    const auto s = ctx->get_saved_variables();
    const bool want = ctx->saved_data["window"].toBool();
    if (!grads[0].defined()) return variable_list(6);
    const Tensor g = grads[0].to(s[0].scalar_type());
    auto [gx, gw, gb, gwin] = backward_call("causal_conv", g, {}, [&] {
      return op.call(g, s[0], s[1], some(s[2]), some(s[3]), some(s[4]), ctx->saved_data["silu"].toBool(), want);
    });
    return {gx, gw, s[2].defined() ? gb : Tensor(), want ? gwin : Tensor(), Tensor(), Tensor()};
  }
};

int64_t conv_weight(const Tensor& weight, int64_t c) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && size_of(weight, 0) == c && size_of(weight, 1) >= 1 && size_of(weight, 1) <= 4,
                    "weight must have shape [C=", c, ", W] with W from 1 to 4; got ", shape_of(weight));
  return size_of(weight, 1);
}

Tensor2 conv(const Tensor& x_, const Tensor& weight, const OptTensor& bias, const OptTensor& state,
             const OptTensor& lengths, bool silu, bool return_state) {
  TORCH_CHECK_VALUE(x_.dim() == 3, "x must have shape [B, T, C]; got ", shape_of(x_));
  const int64_t b = size_of(x_, 0), t = size_of(x_, 1), c = size_of(x_, 2), w = conv_weight(weight, c);
  code_of("x", x_);
  need_shape("bias", bias, {c});
  need_shape("initial_state", state, {b, w - 1, c});
  need_dtype("initial_state", state, x_.scalar_type(), "x");
  const OptTensor weight_ = weight;
  need_cuda("causal_conv", x_, {&weight_, &bias, &state, &lengths});
  no_tangents("causal_conv", x_, weight, bias, state);
  const Tensor wt = parameter(weight), x = rows(x_);
  const OptTensor bi = parameter(bias), lens = lengths_of(lengths, b);
  const OptTensor window = has(state) ? OptTensor(state->contiguous()) : OptTensor();
  if (!wants_grad(x, wt, bi, window)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return conv_fwd_op().call(x, wt, bi, window, lens, silu, return_state);
  }
  Tensor y = CausalConv::apply(x, wt, bi, window, lens, silu), next;
  if (return_state) {  // a copy of rows, with autograd's gradient
    const Tensor full = at::cat({has(window) ? *window : at::zeros({b, w - 1, c}, x.options()), x}, 1);
    if (has(lens)) {
      const Tensor at_ = lens->to(at::kLong).clamp(0, t).unsqueeze(1) + at::arange(w - 1, lens->options().dtype(at::kLong));
      next = at::gather(full, 1, at_.unsqueeze(2).expand({b, w - 1, c}));
    } else {
      next = full.slice(1, t).contiguous();
    }
  } else {
    next = empty(x, {0});
  }
  return {y, next};
}

Tensor conv_step(const Tensor& x_, const Tensor& state, const Tensor& weight, const OptTensor& bias, bool silu) {
  TORCH_CHECK_VALUE(x_.dim() == 2, "x must have shape [B, C]; got ", shape_of(x_));
  const int64_t b = size_of(x_, 0), c = size_of(x_, 1), w = conv_weight(weight, c);
  const int code = code_of("x", x_);
  const OptTensor os = state, ow = weight;
  need_shape("state", os, {b, w - 1, c});
  need_dtype("state", os, x_.scalar_type(), "x");
  need_shape("bias", bias, {c});
  need_cuda("causal_conv_step_", x_, {&os, &ow, &bias});
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous");
  if (x_.is_meta()) return at::empty_like(x_, {}, at::MemoryFormat::Contiguous);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows(x_), wt = parameter(weight);
  const OptTensor bi = parameter(bias);
  Tensor y = empty(x, {b, c});
  check(lib().conv_step(code, x.const_data_ptr(), fptr(wt), fptr(bi), state.mutable_data_ptr(), y.mutable_data_ptr(), b,
                        c, (int)w, x.stride(0), silu, stream_of(x)),
        "causal_conv_step");
  return y;
}

// ------------------------------------------------------------------ scan

Tensor3 scan_fwd(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                 const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, const OptTensor& h0,
                 const OptTensor& lengths, bool softplus, bool want_last, bool want_kept) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t b = x.size(0), t = x.size(1), c = x.size(2), n = A.size(1);
  const int code = code_of("x", x);
  Tensor out = empty(x, {b, t, c}), last = want_last ? empty(x, {b, c, n}, at::kFloat) : empty(x, {0}, at::kFloat);
  const int64_t nkept = want_kept ? (int64_t)lib().scan_state(b, t, c, n) : 0;
  const int64_t nws = (int64_t)lib().scan_forward_workspace(code, b, t, c, n);
  Tensor kept = empty(x, {nkept}, at::kByte), ws = empty(x, {nws}, at::kByte);
  check(lib().scan_forward(code, x.const_data_ptr(), dt.const_data_ptr(), fptr(A), B.const_data_ptr(),
                           C.const_data_ptr(), fptr(D), ptr(z), fptr(dt_bias), fptr(h0),
                           static_cast<const int*>(ptr(lengths)), out.mutable_data_ptr(),
                           static_cast<float*>(out_ptr(last, want_last)), static_cast<float*>(out_ptr(kept, want_kept)),
                           nkept, ws.mutable_data_ptr(), nws, b, t, c, n, x.stride(0), x.stride(1), dt.stride(0),
                           dt.stride(1), B.stride(0), B.stride(1), C.stride(0), C.stride(1), stride0(z, 0),
                           stride0(z, 1), softplus, stream_of(x)),
        "selective_scan_forward");
  return {out, last, kept};
}
Tensor3 scan_fwd_meta(const Tensor& x, const Tensor&, const Tensor& A, const Tensor&, const Tensor&, const OptTensor&,
                      const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, bool, bool want_last,
                      bool want_kept) {
  const c10::SymInt b = x.sym_size(0), t = x.sym_size(1), c = x.sym_size(2), n = A.sym_size(1), none = 0;
  const auto f32 = x.options().dtype(at::kFloat);
  const c10::SymInt kept = b * ((t + 7) / 8) * c * n * 4;  // selective_scan_state_size
  return {at::empty_symint(x.sym_sizes(), x.options()),
          want_last ? at::empty_symint({b, c, n}, f32) : empty(x, {0}, at::kFloat),
          at::empty_symint({want_kept ? kept : none}, x.options().dtype(at::kByte))};
}

// Gradients of x, dt, A, B, C, D, z, dt_bias and the initial state; empty tensors for
// the inputs that are absent (and for a state that is not asked for).
std::vector<Tensor> scan_bwd(const Tensor& g_, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                             const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                             const OptTensor& lengths, const Tensor& kept, const OptTensor& glast_, bool softplus,
                             bool want_h0) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor g = rows(g_);
  const OptTensor glast = has(glast_) ? OptTensor(glast_->contiguous()) : OptTensor();
  const int64_t b = x.size(0), t = x.size(1), c = x.size(2), n = A.size(1);
  const int code = code_of("x", x);
  Tensor gx = empty(x, {b, t, c}), gdt = empty(x, {b, t, c}), gB = empty(x, {b, t, n}), gC = empty(x, {b, t, n});
  Tensor gA = empty(x, {c, n}, at::kFloat), gD = empty(x, {has(D) ? c : 0}, at::kFloat);
  Tensor gz = has(z) ? empty(x, {b, t, c}) : empty(x, {0}), gbias = empty(x, {has(dt_bias) ? c : 0}, at::kFloat);
  Tensor gh0 = want_h0 ? empty(x, {b, c, n}, at::kFloat) : empty(x, {0}, at::kFloat);
  const int64_t nws = (int64_t)lib().scan_backward_workspace(code, b, t, c, n);
  Tensor ws = empty(x, {nws}, at::kByte);
  check(lib().scan_backward(code, g.const_data_ptr(), x.const_data_ptr(), dt.const_data_ptr(), fptr(A),
                            B.const_data_ptr(), C.const_data_ptr(), fptr(D), ptr(z), fptr(dt_bias), 
                            static_cast<const float*>(kept.const_data_ptr()), static_cast<const int*>(ptr(lengths)),
                            fptr(glast), gx.mutable_data_ptr(), gdt.mutable_data_ptr(),
                            static_cast<float*>(gA.mutable_data_ptr()), gB.mutable_data_ptr(), gC.mutable_data_ptr(),
                            fout(gD), out_ptr(gz, has(z)), fout(gbias), static_cast<float*>(out_ptr(gh0, want_h0)),
                            ws.mutable_data_ptr(), nws, b, t, c, n, g.stride(0), g.stride(1), x.stride(0), x.stride(1),
                            dt.stride(0), dt.stride(1), B.stride(0), B.stride(1), C.stride(0), C.stride(1),
                            stride0(z, 0), stride0(z, 1), softplus, stream_of(x)),
        "selective_scan_backward");
  return {gx, gdt, gA, gB, gC, gD, gz, gbias, gh0};
}
std::vector<Tensor> scan_bwd_meta(const Tensor&, const Tensor& x, const Tensor&, const Tensor& A, const Tensor& B,
                                  const Tensor&, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                                  const OptTensor&, const Tensor&, const OptTensor&, bool, bool want_h0) {
  const c10::SymInt b = x.sym_size(0), c = x.sym_size(2), n = A.sym_size(1), none = 0;
  const auto f32 = x.options().dtype(at::kFloat);
  auto wide = [&] { return at::empty_symint(x.sym_sizes(), x.options()); };
  auto thin = [&] { return at::empty_symint(B.sym_sizes(), x.options()); };
  return {wide(),
          wide(),
          at::empty_symint(A.sym_sizes(), f32),
          thin(),
          thin(),
          at::empty_symint({has(D) ? c : none}, f32),
          has(z) ? wide() : empty(x, {0}),
          at::empty_symint({has(dt_bias) ? c : none}, f32),
          want_h0 ? at::empty_symint({b, c, n}, f32) : empty(x, {0}, at::kFloat)};
}

const auto& scan_fwd_op() {
  static const auto op = typed<decltype(scan_fwd)>("spikegpt_b200::selective_scan_fwd");
  return op;
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A,
                               const Tensor& B, const Tensor& C, const OptTensor& D, const OptTensor& z,
                               const OptTensor& dt_bias, const OptTensor& h0, const OptTensor& lengths, bool softplus,
                               bool want_last) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, last, kept] = scan_fwd_op().call(x, dt, A, B, C, D, z, dt_bias, h0, lengths, softplus, want_last, true);
    ctx->save_for_backward({x, dt, A, B, C, opt(D), opt(z), opt(dt_bias), opt(lengths), kept});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["h0"] = has(h0) && h0->requires_grad();
    ctx->set_materialize_grads(false);
    if (!want_last) ctx->mark_non_differentiable({last});
    return {out, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = typed<decltype(scan_bwd)>("spikegpt_b200::selective_scan_bwd");
    const auto s = ctx->get_saved_variables();
    const bool want_h0 = ctx->saved_data["h0"].toBool();
    variable_list r(12);
    if (!grads[0].defined() && !grads[1].defined()) return r;
    const Tensor g = grads[0].defined() ? grads[0].to(s[0].scalar_type()) : at::zeros_like(s[0]);
    const auto got = backward_call("selective_scan", g, some(grads[1]), [&] {
      return op.call(g, s[0], s[1], s[2], s[3], s[4], some(s[5]), some(s[6]), some(s[7]), some(s[8]), s[9],
                     some(grads[1]), ctx->saved_data["softplus"].toBool(), want_h0);
    });
    const bool on[9] = {true, true, true, true, true, s[5].defined(), s[6].defined(), s[7].defined(), want_h0};
    for (int i = 0; i < 9; ++i)
      if (on[i]) r[i] = got[i];
    return r;
  }
};

int64_t scan_parameters(const Tensor& A, const OptTensor& D, const OptTensor& dt_bias, int64_t c) {
  TORCH_CHECK_VALUE(A.dim() == 2 && size_of(A, 0) == c && size_of(A, 1) >= 1 && size_of(A, 1) <= 64,
                    "A must have shape [C=", c, ", N] with N from 1 to 64; got ", shape_of(A));
  need_shape("D", D, {c});
  need_shape("dt_bias", dt_bias, {c});
  return size_of(A, 1);
}

Tensor2 scan(const Tensor& x_, const Tensor& dt_, const Tensor& A_, const Tensor& B_, const Tensor& C_,
             const OptTensor& D_, const OptTensor& z_, const OptTensor& dt_bias_, const OptTensor& state,
             const OptTensor& lengths, bool softplus, bool return_state) {
  TORCH_CHECK_VALUE(x_.dim() == 3, "x must have shape [B, T, C]; got ", shape_of(x_));
  const int64_t b = size_of(x_, 0), t = size_of(x_, 1), c = size_of(x_, 2), n = scan_parameters(A_, D_, dt_bias_, c);
  code_of("x", x_);
  const OptTensor od = dt_, oA = A_, oB = B_, oC = C_;
  need_shape("dt", od, {b, t, c});
  need_shape("z", z_, {b, t, c});
  need_shape("B", oB, {b, t, n});
  need_shape("C", oC, {b, t, n});
  need_dtype("dt", od, x_.scalar_type(), "x");
  need_dtype("B", oB, x_.scalar_type(), "x");
  need_dtype("C", oC, x_.scalar_type(), "x");
  need_dtype("z", z_, x_.scalar_type(), "x");
  need_shape("initial_state", state, {b, c, n});
  TORCH_CHECK_VALUE(!has(state) || state->scalar_type() == at::kFloat, "initial_state must be float32");
  need_cuda("selective_scan", x_, {&od, &oA, &oB, &oC, &D_, &z_, &dt_bias_, &state, &lengths});
  no_tangents("selective_scan", x_, dt_, A_, B_, C_, D_, z_, dt_bias_, state);
  const Tensor x = rows(x_), dt = rows(dt_), A = parameter(A_), B = rows(B_), C = rows(C_);
  const OptTensor D = parameter(D_), z = rows(z_), dt_bias = parameter(dt_bias_), lens = lengths_of(lengths, b);
  const OptTensor h0 = has(state) ? OptTensor(state->contiguous()) : OptTensor();
  if (wants_grad(x_, dt_, A_, B_, C_, D, z, dt_bias, h0)) {
    const auto r = SelectiveScan::apply(x, dt, A, B, C, D, z, dt_bias, h0, lens, softplus, return_state);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const auto r = scan_fwd_op().call(x, dt, A, B, C, D, z, dt_bias, h0, lens, softplus, return_state, false);
  return {std::get<0>(r), std::get<1>(r)};
}

Tensor scan_step(const Tensor& x_, const Tensor& dt_, const Tensor& A_, const Tensor& B_, const Tensor& C_,
                 const Tensor& state, const OptTensor& D_, const OptTensor& z_, const OptTensor& dt_bias_,
                 bool softplus) {
  TORCH_CHECK_VALUE(x_.dim() == 2, "x must have shape [B, C]; got ", shape_of(x_));
  const int64_t b = size_of(x_, 0), c = size_of(x_, 1), n = scan_parameters(A_, D_, dt_bias_, c);
  const int code = code_of("x", x_);
  const OptTensor od = dt_, oA = A_, oB = B_, oC = C_, os = state;
  need_shape("dt", od, {b, c});
  need_shape("z", z_, {b, c});
  need_shape("B", oB, {b, n});
  need_shape("C", oC, {b, n});
  need_dtype("dt", od, x_.scalar_type(), "x");
  need_dtype("B", oB, x_.scalar_type(), "x");
  need_dtype("C", oC, x_.scalar_type(), "x");
  need_dtype("z", z_, x_.scalar_type(), "x");
  need_shape("state", os, {b, c, n});
  TORCH_CHECK_VALUE(state.scalar_type() == at::kFloat && state.is_contiguous(), "state must be contiguous float32");
  need_cuda("selective_scan_step_", x_, {&od, &oA, &oB, &oC, &os, &D_, &z_, &dt_bias_});
  if (x_.is_meta()) return at::empty_like(x_, {}, at::MemoryFormat::Contiguous);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows(x_), dt = rows(dt_), A = parameter(A_), B = rows(B_), C = rows(C_);
  const OptTensor D = parameter(D_), z = rows(z_), dt_bias = parameter(dt_bias_);
  Tensor out = empty(x, {b, c});
  check(lib().scan_step(code, x.const_data_ptr(), dt.const_data_ptr(), fptr(A), B.const_data_ptr(), C.const_data_ptr(),
                        static_cast<float*>(state.mutable_data_ptr()), fptr(D), ptr(z), fptr(dt_bias),
                        out.mutable_data_ptr(), b, c, n, x.stride(0), dt.stride(0), B.stride(0), C.stride(0),
                        stride0(z, 0), softplus, stream_of(x)),
        "selective_scan_step");
  return out;
}

// ----------------------------------------------------------- 4-bit weights

constexpr int64_t kFewTokens = 64;  // tokens of one call into the library

Tensor q4_linear(const Tensor& x_, const Tensor& packed, const Tensor& scales, const OptTensor& zeros,
                 const OptTensor& bias_, int64_t group) {
  TORCH_CHECK_VALUE(x_.dim() >= 1, "x must have at least one dimension");
  TORCH_CHECK_VALUE(group >= 32 && group % 32 == 0, "group_size must be a positive multiple of 32; got ", group);
  const int64_t k = size_of(x_, -1), pitch = (k + 31) / 32 * 16, groups = (k + group - 1) / group;
  TORCH_CHECK_VALUE(packed.dim() == 2 && packed.scalar_type() == at::kByte && size_of(packed, 1) == pitch,
                    "packed must be uint8 [N, ", pitch, "] for ", k, " inputs; got ", packed.scalar_type(), " ",
                    shape_of(packed));
  const int64_t n = size_of(packed, 0);
  const OptTensor op = packed, os = scales;
  need_shape("scales", os, {n, groups});
  need_shape("zeros", zeros, {n, groups});
  need_shape("bias", bias_, {n});
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kBFloat16 && (!has(zeros) || zeros->scalar_type() == at::kByte),
                    "scales must be bfloat16 and zeros uint8");
  const int code = code_of("x", x_);
  need_cuda("q4_linear", x_, {&op, &os, &zeros, &bias_});
  TORCH_CHECK_VALUE(packed.is_contiguous() && scales.is_contiguous() && (!has(zeros) || zeros->is_contiguous()),
                    "packed, scales and zeros must be contiguous");
  if (x_.is_meta()) {
    c10::SymDimVector shape(x_.sym_sizes().begin(), x_.sym_sizes().end());
    shape.back() = n;
    return at::empty_symint(shape, x_.options());
  }
  const c10::cuda::CUDAGuard guard(x_.device());
  const OptTensor bias = parameter(bias_);
  // the weights come by 16-byte copies: a view at another offset of a flat buffer is copied
  const Tensor weights = reinterpret_cast<uintptr_t>(packed.const_data_ptr()) % 16 == 0 ? packed : packed.clone();
  const Tensor x = rows(x_.dim() == 2 ? x_ : x_.reshape({-1, k}));
  const int64_t m = size_of(x, 0);
  Tensor y = empty(x, {m, n});
  for (int64_t at = 0; at < m; at += kFewTokens) {
    const int64_t few = std::min(kFewTokens, m - at);
    const char* from = static_cast<const char*>(x.const_data_ptr()) + at * x.stride(0) * x.element_size();
    char* to = static_cast<char*>(y.mutable_data_ptr()) + at * n * y.element_size();
    check(lib().q4(code, from, static_cast<const uint8_t*>(weights.const_data_ptr()), scales.const_data_ptr(),
                   static_cast<const uint8_t*>(ptr(zeros)), fptr(bias), to, few, n, k, group, x.stride(0),
                   stream_of(x)),
          "q4_matvec");
  }
  if (x_.dim() == 2) return y;
  auto shape = x_.sizes().vec();
  shape.back() = n;
  return y.view(shape);
}

// ------------------------------------- the operators without a gradient
//
// Autograd kernels that refuse inputs which want a derivative. They see what the kernels
// below them do not: the tensors of torch.func's transforms.

// Tells autograd that a tensor was written in place, so that a backward which saved it
// refuses to run. (An inference tensor cannot be saved and has no version.)
void written(const Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

Tensor conv_step_autograd(const Tensor& x, const Tensor& state, const Tensor& weight, const OptTensor& bias,
                          bool silu) {
  static const auto op = typed<decltype(conv_step)>("spikegpt_b200::causal_conv_step_");
  no_grad_only("causal_conv_step_", x, state, weight, bias);
  no_tangents("causal_conv_step_", x, state, weight, bias);
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    y = op.call(x, state, weight, bias, silu);
  }
  written(state);
  return y;
}
Tensor scan_step_autograd(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                          const Tensor& state, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                          bool softplus) {
  static const auto op = typed<decltype(scan_step)>("spikegpt_b200::selective_scan_step_");
  no_grad_only("selective_scan_step_", x, dt, A, B, C, state, D, z, dt_bias);
  no_tangents("selective_scan_step_", x, dt, A, B, C, state, D, z, dt_bias);
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    y = op.call(x, dt, A, B, C, state, D, z, dt_bias, softplus);
  }
  written(state);
  return y;
}
Tensor q4_linear_autograd(const Tensor& x, const Tensor& packed, const Tensor& scales, const OptTensor& zeros,
                          const OptTensor& bias, int64_t group) {
  static const auto op = typed<decltype(q4_linear)>("spikegpt_b200::q4_linear");
  no_grad_only("q4_linear", x, scales, bias);
  no_tangents("q4_linear", x, scales, bias);
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, packed, scales, zeros, bias, group);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(spikegpt_b200, m) {
  m.def("bind_library(str path) -> bool", &bind_library);
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_bwd(Tensor g, Tensor x, Tensor? weight, Tensor mean, Tensor rstd, bool want_weight, "
        "bool want_bias) -> (Tensor, Tensor, Tensor)");
  m.def("causal_conv(Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu, "
        "bool return_state) -> (Tensor, Tensor)");
  m.def("causal_conv_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? window, Tensor? lengths, bool silu, "
        "bool want_window) -> (Tensor, Tensor)");
  m.def("causal_conv_bwd(Tensor g, Tensor x, Tensor weight, Tensor? bias, Tensor? window, Tensor? lengths, bool silu, "
        "bool want_window) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("causal_conv_step_(Tensor x, Tensor(a!) state, Tensor weight, Tensor? bias, bool silu) -> Tensor");
  m.def("selective_scan(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, "
        "Tensor? state, Tensor? lengths, bool softplus, bool return_state) -> (Tensor, Tensor)");
  m.def("selective_scan_fwd(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, "
        "Tensor? h0, Tensor? lengths, bool softplus, bool want_last, bool want_kept) -> (Tensor, Tensor, Tensor)");
  m.def("selective_scan_bwd(Tensor g, Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, "
        "Tensor? dt_bias, Tensor? lengths, Tensor kept, Tensor? glast, bool softplus, bool want_h0) -> Tensor[]");
  m.def("selective_scan_step_(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor(a!) state, Tensor? D, "
        "Tensor? z, Tensor? dt_bias, bool softplus) -> Tensor");
  m.def("q4_linear(Tensor x, Tensor packed, Tensor scales, Tensor? zeros, Tensor? bias, int group_size) -> Tensor");
}

TORCH_LIBRARY_IMPL(spikegpt_b200, CompositeImplicitAutograd, m) {
  m.impl("layer_norm", &norm);
  m.impl("causal_conv", &conv);
  m.impl("selective_scan", &scan);
}

TORCH_LIBRARY_IMPL(spikegpt_b200, CUDA, m) {
  m.impl("layer_norm_fwd", &norm_fwd);
  m.impl("layer_norm_bwd", &norm_bwd);
  m.impl("causal_conv_fwd", &conv_fwd);
  m.impl("causal_conv_bwd", &conv_bwd);
  m.impl("selective_scan_fwd", &scan_fwd);
  m.impl("selective_scan_bwd", &scan_bwd);
}

TORCH_LIBRARY_IMPL(spikegpt_b200, Meta, m) {
  m.impl("layer_norm_fwd", &norm_fwd_meta);
  m.impl("layer_norm_bwd", &norm_bwd_meta);
  m.impl("causal_conv_fwd", &conv_fwd_meta);
  m.impl("causal_conv_bwd", &conv_bwd_meta);
  m.impl("selective_scan_fwd", &scan_fwd_meta);
  m.impl("selective_scan_bwd", &scan_bwd_meta);
}

// The steps and the 4-bit product have no gradient.
TORCH_LIBRARY_IMPL(spikegpt_b200, CompositeExplicitAutograd, m) {
  m.impl("causal_conv_step_", &conv_step);
  m.impl("selective_scan_step_", &scan_step);
  m.impl("q4_linear", &q4_linear);
}

TORCH_LIBRARY_IMPL(spikegpt_b200, Autograd, m) {
  m.impl("causal_conv_step_", &conv_step_autograd);
  m.impl("selective_scan_step_", &scan_step_autograd);
  m.impl("q4_linear", &q4_linear_autograd);
  m.impl("layer_norm_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("causal_conv_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("selective_scan_bwd", torch::autograd::autogradNotImplementedFallback());
}
