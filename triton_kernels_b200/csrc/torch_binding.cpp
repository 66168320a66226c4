// Python binding of the operators whose calls are short next to the host work of a Python wrapper: LayerNorm with its
// gradients, rotary positions from ids, and the adapter projection.  Each function checks its tensors, allocates the
// results, and calls the C ABI (fluxb200.h) on the current stream of the tensors' device.  The autograd nodes live here
// because a backward pass runs on a thread of its own, where Python code waits for the interpreter: a training call of
// the norm took the host 121 us with Python wrappers and takes 67 here.  Nothing here computes anything.
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <atomic>
#include <string>
#include <vector>

#include "fluxb200.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// ---- errors: the exceptions that the Python wrappers raise ---------------------------------------------------
[[noreturn]] void fail(PyObject* type, const std::string& text) {
  if (!PyGILState_Check()) throw std::runtime_error(text);  // a backward thread
  PyErr_SetString(type, text.c_str());
  throw py::error_already_set();
}
void require(bool ok, const char* text) {
  if (!ok) fail(PyExc_AssertionError, text);
}
std::atomic<int64_t> calls{0};  // that returned success
void check(int rc) {
  if (rc == FLUXB_OK) {
    ++calls;
    return;
  }
  const std::string text = fluxb_last_error();
  if (rc == FLUXB_ERR_BAD_ARG) fail(PyExc_ValueError, text);
  if (rc == FLUXB_ERR_UNSUPPORTED) fail(PyExc_NotImplementedError, text);
  const std::string full = "fluxb200 error " + std::to_string(rc) + ": " + text;
  if (!PyGILState_Check()) throw std::runtime_error(full);
  const py::object type = py::module_::import("triton_kernels_b200._lib").attr("FluxbError");
  fail(type.ptr(), full);
}
void require_cuda(const Tensor& t) {
  if (!t.is_cuda())
    fail(PyExc_RuntimeError, "fluxb200 kernels run on CUDA tensors only (no CPU fallback); got a tensor on " + t.device().str());
}
void same_device(const Tensor& first, const Tensor& t) {
  require_cuda(t);
  if (t.device() != first.device())
    fail(PyExc_RuntimeError,
          "fluxb200 kernels take tensors of one device; got " + first.device().str() + " and " + t.device().str());
}
int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return FLUXB_BF16;
  if (t.scalar_type() == at::kFloat) return FLUXB_F32;
  fail(PyExc_NotImplementedError,
        std::string("fluxb200 kernels take float32 or bfloat16 tensors, got ") + c10::toString(t.scalar_type()));
}
fluxb_stream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// ---- tensors ---------------------------------------------------------------------------------------------------
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
int64_t vec(const Tensor& t) { return 16 / t.element_size(); }
Tensor dense16(const Tensor& t) {
  Tensor c = t.contiguous();
  return aligned(c) ? c : c.clone();
}
// Evenly spaced, 16-byte aligned rows of the last dim: the tensor itself where it is contiguous or a 2-D view with a
// row stride, else a copy.
Tensor as_rows(const Tensor& x) {
  if (x.is_contiguous()) return aligned(x) ? x : x.clone();
  if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= x.size(1) && x.stride(0) % vec(x) == 0 && aligned(x)) return x;
  return x.contiguous();
}
int64_t row_stride(const Tensor& x) { return x.is_contiguous() ? x.size(-1) : x.stride(0); }  // of one as above
Tensor empty_as(const Tensor& x) { return at::empty(x.sizes(), x.options()); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Forward-mode tangents would be lost without a word: refused.
void no_tangents(std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      fail(PyExc_NotImplementedError, "fluxb200 kernels have no forward-mode derivative: detach the dual tensor");
}
const Tensor* given(const std::optional<Tensor>& t) {
  static const Tensor none;
  return t.has_value() ? &*t : &none;
}
// Results of a backward pass that somebody wants to differentiate: an error to be raised when they do, not a silent
// zero (what torch.autograd.function.once_differentiable does for Python functions).
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list marked;
  for (const Tensor& g : grads)
    if (g.defined()) marked.push_back(g.detach().set_requires_grad(true));
  if (marked.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int)marked.size());
  marked = (*error)(std::move(marked));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[i++];
  return grads;
}

// ---- LayerNorm ---------------------------------------------------------------------------------------------------
// stats: fp32, the rows' means, then their reciprocal deviations.
Tensor norm_backward(const Tensor& dy_in, const Tensor& x, const Tensor& factor, int64_t factor_stride, const Tensor& stats,
                     float unit, int64_t groups, bool want_dx, const Tensor& df, const Tensor& dof, bool grads_f32) {
  const int64_t C = x.size(-1), rows = x.numel() / C, per_group = groups > 0 ? rows / groups : 0;
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor dy = as_rows(dy_in);
  Tensor dx = want_dx ? empty_as(x) : Tensor(), scratch;
  if (df.defined() || dof.defined())
    scratch = at::empty({fluxb_layer_norm_bwd_scratch(rows, C, per_group)}, stats.options());
  const float* mean = static_cast<const float*>(stats.data_ptr());
  check(fluxb_layer_norm_bwd(dy.data_ptr(), x.data_ptr(), factor.data_ptr(), mean, mean + rows, ptr(dx), ptr(df), ptr(dof),
                             static_cast<float*>(ptr(scratch)), rows, C, per_group, row_stride(dy), row_stride(x), C,
                             factor_stride, unit, grads_f32, dtype_code(x), stream_of(x)));
  return dx;
}

Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, const Tensor& stats) {
  const int64_t C = x.size(-1), rows = x.numel() / C;
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = empty_as(x);
  float* mean = static_cast<float*>(ptr(stats));
  check(fluxb_layer_norm(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), y.data_ptr(), mean, mean != nullptr ? mean + rows : nullptr,
                         rows, C, rows, row_stride(x), C, 0, 0.f, (float)eps, dtype_code(x), stream_of(x)));
  return y;
}

Tensor make_stats(const Tensor& x) {
  c10::cuda::CUDAGuard guard(x.device());
  return at::empty({2 * (x.numel() / x.size(-1))}, x.options().dtype(at::kFloat));
}
Tensor make_grad(at::IntArrayRef shape, const at::TensorOptions& options, bool rows) {
  return rows ? at::empty(shape, options) : at::zeros(shape, options);
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& weight, const Tensor& bias, double eps) {
    const Tensor x = as_rows(x_in), stats = make_stats(x);
    Tensor y = norm_forward(x, weight, bias, eps, stats);
    ctx->save_for_backward({x, weight, stats});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1];
    const bool some = x.numel() > 0;
    Tensor dw = ctx->needs_input_grad(1) ? make_grad(weight.sizes(), weight.options(), some) : Tensor();
    Tensor db = ctx->needs_input_grad(2) ? make_grad(weight.sizes(), weight.options(), some) : Tensor();
    Tensor dx = norm_backward(dy[0], x, weight, 0, saved[2], 0.f, 1, ctx->needs_input_grad(0), dw, db, false);
    return once({dx, dw, db, Tensor()});
  }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight_in, const std::optional<Tensor>& bias_in, double eps) {
  no_tangents({&x, given(weight_in), given(bias_in)});
  require_cuda(x);
  dtype_code(x);
  require(x.dim() > 0 && x.size(-1) > 0, "layer_norm runs over the last dim, which must not be empty");
  const int64_t C = x.size(-1);
  for (const std::optional<Tensor>* p : {&weight_in, &bias_in}) {
    if (!p->has_value()) continue;
    same_device(x, **p);
    require((*p)->dim() == 1 && (*p)->size(0) == C, "weight and bias are vectors of x's last dim");
    require((*p)->scalar_type() == x.scalar_type(), "Incompatible dtypes");
  }
  const Tensor weight = weight_in.has_value() ? dense16(*weight_in) : at::ones({C}, x.options());
  const Tensor bias = bias_in.has_value() ? dense16(*bias_in) : at::zeros({C}, x.options());
  if (wants_grad({&x, &weight, &bias})) return LayerNorm::apply(x, weight, bias, eps);
  return norm_forward(as_rows(x), weight, bias, eps, Tensor());
}

// (scale as [B, C], y) for a contiguous x.
std::pair<Tensor, Tensor> modulated_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, const Tensor& stats) {
  const int64_t B = x.size(0), C = x.size(-1), v = vec(x);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor w = weight.reshape({B, C}).to(x.scalar_type()), b = bias.reshape({B, C}).to(x.scalar_type());
  const auto ok = [&](const Tensor& t) { return t.stride(1) == 1 && t.stride(0) % v == 0 && aligned(t); };
  if (!(ok(w) && ok(b) && (B == 1 || w.stride(0) == b.stride(0)))) {
    w = w.contiguous();
    b = b.contiguous();
  }
  Tensor y = empty_as(x);
  const int64_t rows = x.numel() / C, per_batch = B > 0 ? rows / B : 0, stride = B > 1 ? w.stride(0) : 0;
  float *mean = static_cast<float*>(ptr(stats)), *rstd = mean != nullptr ? mean + rows : nullptr;
  const int code = dtype_code(x);
  if (C % v != 0 || !aligned(x))  // rows that no 16-byte piece fits: the kernels for any width
    check(fluxb_layer_norm(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), mean, rstd, rows, C, per_batch, C, C, stride, 1.f,
                           (float)eps, code, stream_of(x)));
  else if (mean != nullptr)
    check(fluxb_layer_norm_modulation_stats(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), mean, rstd, rows, C, per_batch, C,
                                            C, stride, (float)eps, code, stream_of(x)));
  else
    check(fluxb_layer_norm_modulation(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), rows, C, per_batch, C, C, stride,
                                      (float)eps, code, stream_of(x)));
  return {w, y};
}

struct LayerNormModulation : torch::autograd::Function<LayerNormModulation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& weight, const Tensor& bias, double eps) {
    const Tensor x = x_in.contiguous(), stats = make_stats(x);
    auto [w, y] = modulated_forward(x, weight, bias, eps, stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["w_shape"] = weight.sizes().vec();
    ctx->saved_data["b_shape"] = bias.sizes().vec();
    ctx->saved_data["w_type"] = weight.scalar_type();
    ctx->saved_data["b_type"] = bias.scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    const at::ScalarType w_type = ctx->saved_data["w_type"].toScalarType(), b_type = ctx->saved_data["b_type"].toScalarType();
    // a scale or shift kept in another type than the rows gets its gradient from the fp32 sums
    const bool own = w_type == x.scalar_type() && b_type == x.scalar_type(), some = x.numel() > 0;
    const at::TensorOptions options = x.options().dtype(own ? x.scalar_type() : at::kFloat);
    Tensor dw = ctx->needs_input_grad(1) ? make_grad(ctx->saved_data["w_shape"].toIntVector(), options, some) : Tensor();
    Tensor db = ctx->needs_input_grad(2) ? make_grad(ctx->saved_data["b_shape"].toIntVector(), options, some) : Tensor();
    const int64_t B = w.size(0);
    Tensor dx = norm_backward(dy[0], x, w, B > 1 ? w.stride(0) : 0, saved[2], 1.f, B, ctx->needs_input_grad(0), dw, db,
                              options.dtype() == at::kFloat);
    if (!own) {
      if (dw.defined()) dw = dw.to(w_type);
      if (db.defined()) db = db.to(b_type);
    }
    return once({dx, dw, db, Tensor()});
  }
};

Tensor layer_norm_modulation(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
  no_tangents({&x, &weight, &bias});
  require(x.dim() > 0 && weight.dim() > 0 && bias.dim() > 0 && x.size(0) == weight.size(0) && x.size(0) == bias.size(0),
          "x, weight and bias differ in the batch dim");
  require(x.size(-1) == weight.size(-1) && x.size(-1) == bias.size(-1), "x, weight and bias differ in the last dim");
  require(x.size(-1) > 0, "the last dim must not be empty");
  require_cuda(x);
  same_device(x, weight);
  same_device(x, bias);
  dtype_code(x);
  if (wants_grad({&x, &weight, &bias})) return LayerNormModulation::apply(x, weight, bias, eps);
  return modulated_forward(x.contiguous(), weight, bias, eps, Tensor()).second;
}

// ---- rotary positions --------------------------------------------------------------------------------------------
int id_code(const Tensor& ids) {
  if (ids.scalar_type() == at::kFloat) return FLUXB_ID_F32;
  if (ids.scalar_type() == at::kInt) return FLUXB_ID_I32;
  if (ids.scalar_type() == at::kLong) return FLUXB_ID_I64;
  fail(PyExc_NotImplementedError, std::string("position ids are float32, int32 or int64, got ") + c10::toString(ids.scalar_type()));
}

// q and k (either may be undefined) rotated; the results have their memory layout.
std::pair<Tensor, Tensor> rotate(Tensor q, Tensor k, const Tensor& ids, at::IntArrayRef axes, double theta, bool backward) {
  c10::cuda::CUDAGuard guard(ids.device());
  Tensor out[2], in[2] = {std::move(q), std::move(k)};
  for (int i = 0; i < 2; ++i) {
    if (!in[i].defined()) continue;
    if (in[i].stride(3) != 1) in[i] = in[i].contiguous();
    out[i] = at::empty_like(in[i]);
    if (out[i].stride(3) != 1) out[i] = empty_as(in[i]);  // an input that overlaps itself
  }
  const Tensor& some = in[0].defined() ? in[0] : in[1];
  const auto st = [](const Tensor& t, int d) { return t.defined() ? t.stride(d) : 0; };
  const auto heads = [](const Tensor& t) { return t.defined() ? t.size(1) : 0; };
  check(fluxb_rope_axes(ptr(in[0]), st(in[0], 0), st(in[0], 1), st(in[0], 2), ptr(out[0]), st(out[0], 0), st(out[0], 1), st(out[0], 2),
                        heads(in[0]), ptr(in[1]), st(in[1], 0), st(in[1], 1), st(in[1], 2), ptr(out[1]), st(out[1], 0),
                        st(out[1], 1), st(out[1], 2), heads(in[1]), ids.data_ptr(), id_code(ids),
                        ids.size(0) > 1 ? ids.stride(0) : 0, ids.stride(1), ids.stride(2), some.size(0), some.size(2), some.size(3),
                        axes.data(), (int)axes.size(), theta, backward, dtype_code(some), stream_of(some)));
  return {out[0], out[1]};
}

struct RopeAxes : torch::autograd::Function<RopeAxes> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& ids, std::vector<int64_t> axes,
                               double theta) {
    ctx->set_materialize_grads(false);
    auto [oq, ok] = rotate(q, k, ids, axes, theta, false);
    ctx->save_for_backward({ids});
    ctx->saved_data["axes"] = std::move(axes);
    ctx->saved_data["theta"] = theta;
    return {oq, ok};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    Tensor dq = ctx->needs_input_grad(0) ? d[0] : Tensor(), dk = ctx->needs_input_grad(1) ? d[1] : Tensor();
    if (dq.defined() || dk.defined()) {
      const std::vector<int64_t> axes = ctx->saved_data["axes"].toIntVector();
      std::tie(dq, dk) = rotate(dq, dk, ctx->get_saved_variables()[0], axes, ctx->saved_data["theta"].toDouble(), true);
    }
    return once({dq, dk, Tensor(), Tensor(), Tensor()});
  }
};

std::pair<Tensor, Tensor> apply_rope_axes(const Tensor& q, const Tensor& k, const Tensor& ids, std::vector<int64_t> axes, double theta) {
  no_tangents({&q, &k, &ids});
  require_cuda(q);
  same_device(q, k);
  same_device(q, ids);
  require(q.dim() == 4 && k.dim() == 4 && q.scalar_type() == k.scalar_type(), "xq and xk are 4-D and of one type");
  require(q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3), "xq and xk differ in more than the head count");
  require(ids.dim() == 3 && (ids.size(0) == 1 || ids.size(0) == q.size(0)) && ids.size(1) == q.size(2) &&
              ids.size(2) == (int64_t)axes.size(),
          "ids must be [B or 1, L, number of axes]");
  id_code(ids);
  dtype_code(q);
  if (wants_grad({&ids})) fail(PyExc_NotImplementedError, "position ids get no gradient: detach them");
  if (wants_grad({&q, &k})) {
    variable_list out = RopeAxes::apply(q, k, ids, std::move(axes), theta);
    return {out[0], out[1]};
  }
  return rotate(q, k, ids, axes, theta, false);
}

// ---- adapters ----------------------------------------------------------------------------------------------------
Tensor linear_lora(const Tensor& x, const Tensor& w_in, const std::optional<Tensor>& b_in, const Tensor& lora_a, const Tensor& lora_b_in,
                   const Tensor& adapter, const std::optional<Tensor>& scale_in, bool gelu) {
  const std::initializer_list<const Tensor*> numbers = {&x, &w_in, given(b_in), &lora_a, &lora_b_in, given(scale_in)};
  no_tangents(numbers);
  if (wants_grad(numbers))
    fail(PyExc_NotImplementedError, "linear_lora is forward only: call it under torch.no_grad() or detach its inputs");
  require(x.dim() >= 2 && w_in.dim() == 2 && x.size(-1) == w_in.size(1) && w_in.size(1) > 0, "Incompatible dimensions");
  const int64_t N = w_in.size(0), K = w_in.size(1), n = lora_a.dim() == 3 ? lora_a.size(0) : 0, R = n > 0 ? lora_a.size(1) : 0;
  require(n > 0 && R > 0 && lora_a.size(2) == K && lora_b_in.dim() == 3 && lora_b_in.size(0) == n && lora_b_in.size(1) == N &&
              lora_b_in.size(2) == R,
          "lora_a must be [n, R, K] and lora_b [n, N, R]");
  require(adapter.dim() == 1 && adapter.size(0) == x.size(0), "adapter holds one index per request (x's first dim)");
  require(!b_in.has_value() || (b_in->dim() == 1 && b_in->size(0) == N), "the bias is a vector of w's rows");
  require(!scale_in.has_value() || (scale_in->dim() == 1 && scale_in->size(0) == n), "lora_scale holds one number per adapter");
  require_cuda(x);
  for (const Tensor* t : {&w_in, &lora_a, &lora_b_in, &adapter}) same_device(x, *t);
  if (b_in.has_value()) same_device(x, *b_in);
  if (scale_in.has_value()) same_device(x, *scale_in);
  for (const Tensor* t : {&x, &w_in, &lora_a, &lora_b_in}) {
    if (t->scalar_type() != at::kBFloat16) {
      const py::object type = py::module_::import("triton_kernels_b200.kernels.linear").attr("UnsupportedDtype");
      fail(type.ptr(), c10::toString(t->scalar_type()));
    }
  }
  if (adapter.scalar_type() != at::kInt && adapter.scalar_type() != at::kLong)
    fail(PyExc_TypeError, std::string("adapter indices are int32 or int64, got ") + c10::toString(adapter.scalar_type()));
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(x.device());
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = at::empty(shape, x.options());
  if (y.numel() == 0) return y;
  const int64_t B = x.size(0), M = x.numel() / K;
  Tensor x2 = x.is_contiguous() ? x : x.reshape({M, K});
  int64_t ldx = x2.is_contiguous() ? K : x2.stride(0);
  if (!x2.is_contiguous() && (x2.stride(1) != 1 || ldx % 8 != 0 || ldx < K)) {
    x2 = x2.contiguous();
    ldx = K;
  }
  if (!aligned(x2)) {
    x2 = x2.contiguous().clone();
    ldx = K;
  }
  const bool w_ok = w_in.stride(1) == 1 && w_in.stride(0) % 8 == 0 && w_in.stride(0) >= K && aligned(w_in);
  const Tensor w = w_ok ? w_in : dense16(w_in);
  const Tensor b = b_in.has_value() ? dense16(b_in->to(at::kBFloat16)) : Tensor();
  // rows of B that no 16-byte piece fits are copied into wider ones
  const Tensor lora_b = dense16(R % 8 != 0 ? at::constant_pad_nd(lora_b_in, {0, 8 - R % 8}) : lora_b_in), a = dense16(lora_a);
  const Tensor scale = scale_in.has_value() ? scale_in->to(at::kFloat).contiguous() : Tensor();
  const Tensor index = adapter.contiguous();
  const Tensor scratch = at::empty({fluxb_linear_lora_scratch_bytes(M, N, K, R)}, x.options().dtype(at::kByte));
  check(fluxb_linear_lora(x2.data_ptr(), w.data_ptr(), ptr(b), y.data_ptr(), a.data_ptr(), lora_b.data_ptr(),
                          static_cast<const float*>(ptr(scale)), index.data_ptr(), index.scalar_type() == at::kLong, scratch.data_ptr(),
                          B, M / B, N, K, R, n, ldx, w.stride(0), N, lora_b.size(2), gelu ? FLUXB_EPI_GELU : FLUXB_EPI_NONE,
                          stream_of(x)));
  return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_modulation", &layer_norm_modulation);
  m.def("apply_rope_axes", &apply_rope_axes);
  m.def("linear_lora", &linear_lora);
  m.def("calls", [] { return calls.load(); });
}
