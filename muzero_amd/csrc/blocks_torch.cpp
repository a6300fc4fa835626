// The training-block operators (mz_layer_norm_*, mz_gated_ff_*, mz_dropout) as differentiable functions of torch tensors:
// the module muzero_amd._blocks behind muzero_amd/blocks.py, which documents them.
//
// Why not in Python like the learner's convolutions: those take tens of microseconds of GPU time and more a call, these
// a few.  A small training step is then all host time, most of it Python's on autograd's own thread, where it runs cold:
// a layer norm step of 18432 x 256 took 104 us as Python functions and needs 31 us of the GPU.
//
// Nothing here computes: arguments are checked (ValueError), memory comes from torch's allocator per call, and the C ABI
// is called on the tensors' device and its current stream.  The entry points are handed over as addresses by bind(), so
// that the module uses the library that muzero_amd._lib has loaded.
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <sstream>

#include "../../include/muzero_amd.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Api {
  decltype(&mz_last_error) last_error = nullptr;
  decltype(&mz_layer_norm_fwd) layer_norm_fwd = nullptr;
  decltype(&mz_layer_norm_workspace_bytes) layer_norm_workspace_bytes = nullptr;
  decltype(&mz_layer_norm_bwd) layer_norm_bwd = nullptr;
  decltype(&mz_gated_ff_workspace_bytes) gated_ff_workspace_bytes = nullptr;
  decltype(&mz_gated_ff_fwd) gated_ff_fwd = nullptr;
  decltype(&mz_gated_ff_bwd) gated_ff_bwd = nullptr;
  decltype(&mz_dropout) dropout = nullptr;
} api;

struct LibraryError : std::runtime_error {      // becomes muzero_amd.MuZeroAmdError
  using std::runtime_error::runtime_error;
};

void check(int rc, const char* name) {
  if (rc == 0) return;
  std::ostringstream s;
  s << name << " failed (" << rc << "): " << api.last_error();
  throw LibraryError(s.str());
}

template <typename... A> [[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw py::value_error(s.str());
}

constexpr int64_t kMaxCols = 1 << 24;          // columns of layer norm
constexpr int64_t kMaxWidth = 1 << 20;         // input and hidden width of the gated projection
constexpr int64_t kMaxStrideBytes = 1 << 22;   // between rows of its input

int type_code(at::ScalarType t) {
  return t == at::kFloat ? MZ_F32 : t == at::kBFloat16 ? MZ_BF16 : t == at::kHalf ? MZ_F16 : -1;
}
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor contiguous(const Tensor& t) { return t.defined() && !t.is_contiguous() ? t.contiguous() : t; }
Tensor like(const Tensor& x) { return at::empty_like(x, x.options(), at::MemoryFormat::Contiguous); }
Tensor bytes(int64_t n, const Tensor& x) { return n > 0 ? at::empty({n}, x.options().dtype(at::kByte)) : Tensor(); }
mz_stream_t stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.get_device()).stream(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
// values as they lie in memory (the imaginary part of a conjugate is a float tensor whose sign is to be read the other way)
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// the gradient of an output in the output's type, which is the input's, in memory
Tensor grad_as(const Tensor& g, at::ScalarType t) {
  if (g._is_zerotensor()) return at::zeros(g.sizes(), g.options().dtype(t));
  return g.scalar_type() == t ? plain(g) : g.to(t);
}

// ---- arguments
Tensor tensor(py::handle h, const char* name) {
  if (!THPVariable_Check(h.ptr())) refuse(name, ": tensor required");
  const Tensor t = THPVariable_Unpack(h.ptr());
  if (t._fw_grad(0).defined()) refuse(name, ": forward-mode derivatives are not offered");
  if (t._is_zerotensor()) refuse(name, ": a tensor without memory");
  if (torch::jit::tracer::isTracing()) refuse(name, ": cannot be traced (the trace would hold no trace of the kernels)");
  return plain(t);
}
Tensor optional_tensor(py::handle h, const char* name) {
  if (h.is_none()) return Tensor();
  return tensor(h, name);
}
void check_activation(const Tensor& x, const char* name) {
  if (!x.is_cuda()) refuse(name, ": must live on the GPU");
  if (type_code(x.scalar_type()) < 0) refuse(name, ": dtype ", x.scalar_type(), ", expected float32, bfloat16 or float16");
  if (x.layout() != at::kStrided) refuse(name, ": a dense tensor expected");
  if (x.dim() == 0 || x.size(-1) == 0) refuse(name, ": shape ", x.sizes(), ", expected a last dimension of at least 1");
}
void check_param(const Tensor& t, const char* name, at::IntArrayRef shape, const Tensor& like, at::ScalarType a,
                 at::ScalarType b) {
  if (t.device() != like.device()) refuse(name, ": on ", t.device(), ", expected ", like.device());
  if (t.scalar_type() != a && t.scalar_type() != b) {
    if (a == b) refuse(name, ": dtype ", t.scalar_type(), ", expected ", a);
    refuse(name, ": dtype ", t.scalar_type(), ", expected ", a, " or ", b);
  }
  if (t.layout() != at::kStrided) refuse(name, ": a dense tensor expected");
  if (t.sizes() != shape) refuse(name, ": shape ", t.sizes(), ", expected ", shape);
}

// x as rows of its last dimension, `ld` elements apart: a slice of wider rows stays in place, what a row stride cannot
// describe is copied
struct Rows {
  Tensor t;
  int64_t ld;
};
Rows rows_of(const Tensor& x) {
  const int64_t c = x.size(-1);
  if (x.is_contiguous()) return {x, c};
  Tensor r = x.reshape({-1, c});
  if ((c > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < c)) r = r.contiguous();
  return {r, r.size(0) > 1 ? r.stride(0) : c};
}
// for the matrix kernels: rows at most 4 MiB apart
Rows matrix_rows(const Tensor& x) {
  Rows r = rows_of(x);
  if (r.ld * x.element_size() > kMaxStrideBytes) r = {r.t.clone(at::MemoryFormat::Contiguous), x.size(-1)};
  return r;
}

// Gradients that a backward pass returns.  They are raw results: where somebody may ask for their own gradient, that has
// to fail and not to be taken for zero.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) {
      auto node = std::make_shared<torch::autograd::DelayedError>("this operator is differentiable once", 1);
      g = (*node)({g.detach().requires_grad_()})[0];
    }
  return grads;
}

// torch's Function counts the tensors it was given; an optional one that was not given is none of them
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor or_none(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
struct Wanted {
  AutogradContext* ctx;
  int next = 0;
  bool operator()(bool given) { return given && ctx->needs_input_grad(next++); }
};

// ------------------------------------------------------------------------------------------------------- layer norm
at::ScalarType affine_type(const Tensor& w, const Tensor& b) {
  return w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
}

Tensor layer_norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
  const int64_t c = x.size(-1), rows = x.numel() / c;
  const c10::DeviceGuard guard(x.device());
  Tensor y = like(x);
  if (stats) *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
  if (rows == 0) return y;
  const Rows r = rows_of(x);
  const Tensor wc = contiguous(w), bc = contiguous(b);
  float* mean = stats ? stats->data_ptr<float>() : nullptr;
  check(api.layer_norm_fwd(r.t.data_ptr(), r.ld, address(wc), address(bc), type_code(affine_type(w, b)), eps, rows, (int32_t)c,
                           type_code(x.scalar_type()), y.data_ptr(), mean, mean ? mean + rows : nullptr, stream_of(x)),
        "mz_layer_norm_fwd");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
    const Tensor w = or_none(weight), b = or_none(bias);
    Tensor stats;
    Tensor y = layer_norm_forward(x, w, b, eps, &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["affine"] = (int64_t)affine_type(w, b);
    ctx->saved_data["bias"] = b.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return once(compute(ctx, grads)); }
  static variable_list compute(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2], &g = grads[0];
    variable_list out(4);
    if (!g.defined()) return out;
    const at::AutoGradMode raw(false);
    const int64_t c = x.size(-1), rows = x.numel() / c;
    const c10::DeviceGuard guard(x.device());
    const auto affine = (at::ScalarType)ctx->saved_data["affine"].toInt();
    const auto options = x.options().dtype(affine);
    Wanted wanted{ctx};
    auto make = [&] { return rows ? at::empty({c}, options) : at::zeros({c}, options); };
    if (wanted(true)) out[0] = like(x);
    if (wanted(w.defined())) out[1] = make();
    if (wanted(ctx->saved_data["bias"].toBool())) out[2] = make();
    if (rows && (out[0].defined() || out[1].defined() || out[2].defined())) {
      const Rows xr = rows_of(x), gr = rows_of(grad_as(g, x.scalar_type()));
      const int64_t need = out[1].defined() || out[2].defined() ? api.layer_norm_workspace_bytes(rows, (int32_t)c) : 0;
      const Tensor ws = bytes(need, x), wc = contiguous(w);
      const float* mean = stats.data_ptr<float>();
      check(api.layer_norm_bwd(xr.t.data_ptr(), xr.ld, gr.t.data_ptr(), gr.ld, address(wc), type_code(affine), mean, mean + rows,
                               rows, (int32_t)c, type_code(x.scalar_type()), address(out[0]), address(out[1]),
                               address(out[2]), address(ws), need, stream_of(x)),
            "mz_layer_norm_bwd");
    }
    return out;
  }
};

Tensor layer_norm(py::handle hx, py::handle hw, py::handle hb, double eps) {
  const Tensor x = tensor(hx, "layer_norm: x"), w = optional_tensor(hw, "layer_norm: weight"),
               b = optional_tensor(hb, "layer_norm: bias");
  const py::gil_scoped_release others_run;
  check_activation(x, "layer_norm: x");
  const int64_t c = x.size(-1);
  if (c > kMaxCols) refuse("layer_norm: x: at most ", kMaxCols, " columns");
  if (w.defined()) check_param(w, "layer_norm: weight", {c}, x, at::kFloat, x.scalar_type());
  if (b.defined())
    check_param(b, "layer_norm: bias", {c}, x, w.defined() ? w.scalar_type() : at::kFloat,
                w.defined() ? w.scalar_type() : x.scalar_type());
  if (!(eps >= 0.0)) refuse("layer_norm: eps ", eps, ", expected at least 0");
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) return LayerNorm::apply(x, maybe(w), maybe(b), eps);
  return layer_norm_forward(x, w, b, eps, nullptr);
}

// ------------------------------------------------------------------------------------------- gated feed-forward
Tensor gated_ff_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int64_t act) {
  const int64_t hidden = wg.size(0), k = wg.size(1), rows = x.numel() / k;
  const c10::DeviceGuard guard(x.device());
  auto shape = x.sizes().vec();
  shape.back() = hidden;
  Tensor h = at::empty(shape, x.options());
  if (rows == 0) return h;
  const Rows r = matrix_rows(x);
  const Tensor wgc = contiguous(wg), wuc = contiguous(wu), bgc = contiguous(bg), buc = contiguous(bu);
  const int type = type_code(x.scalar_type());
  const int64_t need = api.gated_ff_workspace_bytes(rows, k, hidden, type, 0);
  const Tensor ws = bytes(need, x);
  check(api.gated_ff_fwd(r.t.data_ptr(), r.ld, wgc.data_ptr(), wuc.data_ptr(), address(bgc), address(buc), rows, k, hidden, type,
                         (int32_t)act, h.data_ptr(), address(ws), need, stream_of(x)),
        "mz_gated_ff_fwd");
  return h;
}

struct GatedFF : torch::autograd::Function<GatedFF> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Maybe& b_gate,
                        const Maybe& b_up, int64_t act) {
    const Tensor bg = or_none(b_gate), bu = or_none(b_up);
    ctx->save_for_backward({x, wg, wu, bg, bu});
    ctx->saved_data["activation"] = act;
    return gated_ff_forward(x, wg, wu, bg, bu, act);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return once(compute(ctx, grads)); }
  static variable_list compute(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &bg = saved[3], &bu = saved[4];
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const at::AutoGradMode raw(false);
    const int64_t hidden = wg.size(0), k = wg.size(1), rows = x.numel() / k;
    const c10::DeviceGuard guard(x.device());
    auto make = [&](at::IntArrayRef s) { return rows ? at::empty(s, x.options()) : at::zeros(s, x.options()); };
    Wanted wanted{ctx};
    bool want[5];
    for (int i = 0; i < 5; ++i) want[i] = wanted(saved[i].defined());
    const bool weights = want[1] || want[2];           // one kernel makes both
    if (want[0]) out[0] = like(x);
    for (int i = 1; i < 3; ++i)
      if (weights) out[i] = make({hidden, k});
    for (int i = 3; i < 5; ++i)
      if (want[i]) out[i] = make({hidden});
    if (rows && (out[0].defined() || weights || out[3].defined() || out[4].defined())) {
      const Rows r = matrix_rows(x);
      const Tensor wgc = contiguous(wg), wuc = contiguous(wu), bgc = contiguous(bg), buc = contiguous(bu);
      const Tensor dh = contiguous(grad_as(grads[0], x.scalar_type()));
      const int type = type_code(x.scalar_type());
      const int64_t need = api.gated_ff_workspace_bytes(rows, k, hidden, type, 1);
      const Tensor ws = bytes(need, x);
      check(api.gated_ff_bwd(r.t.data_ptr(), r.ld, wgc.data_ptr(), wuc.data_ptr(), address(bgc), address(buc), dh.data_ptr(),
                             rows, k, hidden, type, (int32_t)ctx->saved_data["activation"].toInt(), address(out[0]),
                             address(out[1]), address(out[2]), address(out[3]), address(out[4]), address(ws), need,
                             stream_of(x)),
            "mz_gated_ff_bwd");
    }
    for (int i = 1; i < 3; ++i)
      if (!want[i]) out[i] = Tensor();
    return out;
  }
};

Tensor gated_ff(py::handle hx, py::handle hwg, py::handle hwu, py::handle hbg, py::handle hbu, const std::string& activation) {
  static const char* const names[4] = {"silu", "gelu", "relu", "sigmoid"};
  int act = 0;
  while (act < 4 && activation != names[act]) ++act;
  if (act == 4) refuse("gated_ff: activation '", activation, "', expected one of silu, gelu, relu, sigmoid");
  Tensor x = tensor(hx, "gated_ff: x"), wg = tensor(hwg, "gated_ff: w_gate"), wu = tensor(hwu, "gated_ff: w_up"),
         bg = optional_tensor(hbg, "gated_ff: b_gate"), bu = optional_tensor(hbu, "gated_ff: b_up");
  const py::gil_scoped_release others_run;
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    const auto t = at::autocast::get_autocast_dtype(at::kCUDA);
    for (Tensor* v : {&x, &wg, &wu, &bg, &bu})
      if (v->defined()) *v = at::autocast::cached_cast(t, *v, at::kCUDA);
  }
  check_activation(x, "gated_ff: x");
  if (wg.dim() != 2 || wg.size(0) == 0) refuse("gated_ff: w_gate: [F, K] tensor with F of at least 1 expected");
  const int64_t hidden = wg.size(0), k = x.size(-1);
  if (k > kMaxWidth || hidden > kMaxWidth) refuse("gated_ff: widths ", k, " and ", hidden, ", expected at most ", kMaxWidth);
  const auto t = x.scalar_type();
  check_param(wg, "gated_ff: w_gate", {hidden, k}, x, t, t);
  check_param(wu, "gated_ff: w_up", {hidden, k}, x, t, t);
  if (bg.defined()) check_param(bg, "gated_ff: b_gate", {hidden}, x, t, t);
  if (bu.defined()) check_param(bu, "gated_ff: b_up", {hidden}, x, t, t);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(wg) || wants_grad(wu) || wants_grad(bg) || wants_grad(bu)))
    return GatedFF::apply(x, wg, wu, maybe(bg), maybe(bu), (int64_t)act);
  return gated_ff_forward(x, wg, wu, bg, bu, act);
}

// ---------------------------------------------------------------------------------------------------------- dropout
Tensor dropout_forward(const Tensor& x_in, const Tensor& residual, double p, const Tensor& rng, int64_t call) {
  const c10::DeviceGuard guard(x_in.device());
  const Tensor x = contiguous(x_in), r = contiguous(residual);
  Tensor y = at::empty_like(x);
  if (x.numel())
    check(api.dropout(x.data_ptr(), address(r), y.data_ptr(), x.numel(), p, rng.data_ptr<int64_t>(), (uint32_t)call,
                      type_code(x.scalar_type()), stream_of(x)),
          "mz_dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, double p, const Tensor& rng, int64_t call) {
    ctx->save_for_backward({rng});
    ctx->saved_data["p"] = p;
    ctx->saved_data["call"] = call;
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["residual"] = residual.has_value();
    return dropout_forward(x, or_none(residual), p, rng, call);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return once(compute(ctx, grads)); }
  static variable_list compute(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();     // raises if rng has changed since
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const at::AutoGradMode raw(false);
    const Tensor g = grad_as(grads[0], (at::ScalarType)ctx->saved_data["type"].toInt());
    Wanted wanted{ctx};
    if (wanted(true))
      out[0] = dropout_forward(g, Tensor(), ctx->saved_data["p"].toDouble(), saved[0], ctx->saved_data["call"].toInt());
    if (wanted(ctx->saved_data["residual"].toBool())) out[1] = g;
    return out;
  }
};

Tensor dropout(py::handle hx, double p, py::handle hrng, int64_t call, py::handle hresidual) {
  const Tensor x = tensor(hx, "dropout: x"), residual = optional_tensor(hresidual, "dropout: residual"),
               rng = tensor(hrng, "dropout: rng");
  const py::gil_scoped_release others_run;
  check_activation(x, "dropout: x");
  if (x.numel() > (int64_t)1 << 35) refuse("dropout: x: at most 2^35 elements");
  if (!(p >= 0.0 && p <= 1.0)) refuse("dropout: p ", p, ", expected 0 to 1");
  if (call < 0 || call >= (int64_t)1 << 32) refuse("dropout: call ", call, ", expected 0 to 2^32 - 1");
  check_param(rng, "dropout: rng", {2}, x, at::kLong, at::kLong);
  if (!rng.is_contiguous()) refuse("dropout: rng: must be contiguous");
  if (residual.defined()) check_param(residual, "dropout: residual", x.sizes(), x, x.scalar_type(), x.scalar_type());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(residual))) return Dropout::apply(x, maybe(residual), p, rng, call);
  return dropout_forward(x, residual, p, rng, call);
}

template <typename F> void take(F& f, const py::dict& entries, const char* name) {
  f = reinterpret_cast<F>(entries[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(_blocks, m) {
  m.def("bind", [](const py::dict& entries, py::object error) {
    take(api.last_error, entries, "mz_last_error");
    take(api.layer_norm_fwd, entries, "mz_layer_norm_fwd");
    take(api.layer_norm_workspace_bytes, entries, "mz_layer_norm_workspace_bytes");
    take(api.layer_norm_bwd, entries, "mz_layer_norm_bwd");
    take(api.gated_ff_workspace_bytes, entries, "mz_gated_ff_workspace_bytes");
    take(api.gated_ff_fwd, entries, "mz_gated_ff_fwd");
    take(api.gated_ff_bwd, entries, "mz_gated_ff_bwd");
    take(api.dropout, entries, "mz_dropout");
    static PyObject* library_error = error.release().ptr();
    py::register_local_exception_translator([](std::exception_ptr p) {
      try {
        if (p) std::rethrow_exception(p);
      } catch (const LibraryError& e) {
        PyErr_SetString(library_error, e.what());
      }
    });
  });
  m.def("layer_norm", &layer_norm);
  m.def("gated_ff", &gated_ff);
  m.def("dropout", &dropout);
}
