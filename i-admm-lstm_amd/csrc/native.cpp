// iadmm._native: the host side of the operators that take torch tensors in numbers or inside autograd -- layer norm
// with its gradient, the AdamW step and the gradients' norm.  It checks the tensors, allocates what is returned and
// calls libiadmm.so's C entry points (include/iadmm.h), whose addresses iadmm/_abi.py hands over.
//
// Why not Python like the other wrappers: these calls are short.  16 parameters with their gradients and moments
// took 41 us to check and pack in Python against 9 us of GPU work, and a backward pass in Python costs the autograd
// engine's thread the interpreter's lock (154 us for one row's layer norm and gradients).
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "../../include/iadmm.h"

namespace {

using at::Tensor;

struct {
  decltype(&iadmm_layer_norm_fwd) ln_fwd;
  decltype(&iadmm_layer_norm_bwd_ws_bytes) ln_bwd_ws_bytes;
  decltype(&iadmm_layer_norm_bwd) ln_bwd;
  decltype(&iadmm_grad_norm_ws_bytes) norm_ws_bytes;
  decltype(&iadmm_grad_norm) norm;
  decltype(&iadmm_adamw_ws_bytes) adamw_ws_bytes;
  decltype(&iadmm_adamw_step) adamw_step;
} abi;

void done(const char* name, int status) {
  TORCH_CHECK(status == 0, name, " failed: ",
              status == IADMM_E_ARG ? "bad argument" : status == IADMM_E_SIZE ? "size beyond kernel limit"
              : status == IADMM_E_ALIGN ? "misaligned pointer" : "HIP error", " (status ", status, ")");
}

void* stream_of(const c10::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

int type_code(at::ScalarType t) {
  return t == at::kFloat ? IADMM_F32 : t == at::kBFloat16 ? IADMM_BF16 : t == at::kHalf ? IADMM_F16 : -1;
}

void on_device(const Tensor& t, const char* what, const Tensor* like = nullptr) {
  TORCH_CHECK_VALUE(t.is_cuda(), "iadmm kernels need device tensors (no CPU fallback), and ", what, " is on ", t.device());
  TORCH_CHECK_VALUE(!like || t.device() == like->device(), what, " is on ", t.device(), ", not on ", like->device());
  TORCH_CHECK_VALUE(!t.is_neg(), what, " is a view that torch negates on reading: resolve_neg() it first");
  // (a fake tensor of a tracing mode has none, and a null pointer would stand for an operand that is left out)
  TORCH_CHECK_VALUE(t.layout() != at::kStrided || t.numel() == 0 || t.const_data_ptr(), what, " has no memory");
}

// A kernel wrote it behind autograd's back: whoever goes by its version (a graph that saved it, solver.PackedWeights) has
// to see it.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A trace records torch's operations alone: the result would stand in it as a constant.
void not_traced() { TORCH_CHECK(!torch::jit::tracer::isTracing(), "torch.jit.trace cannot record iadmm's kernels"); }

Tensor f32_on(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }

// ----------------------------------------------------------------------------------------------- layer norm
bool has_rows(const Tensor& t) {
  return t.is_contiguous() || (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1));
}

// The tensor, or a copy where its rows are not contiguous or torch negates it on reading.
Tensor plain_rows(const Tensor& t) {
  const Tensor p = t.is_neg() ? t.resolve_neg() : t;
  return has_rows(p) ? p : p.contiguous();
}

struct Rows { int64_t rows, cols, ld; };

Rows rows_of(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.dim() >= 1 && t.size(-1) > 0, what,
                    " needs a last dimension of at least one element, got ", t.sizes());
  const int64_t cols = t.size(-1);
  if (t.is_contiguous()) return {t.numel() / cols, cols, cols};
  TORCH_CHECK_VALUE(has_rows(t), what, " needs contiguous rows, got strides ", t.strides(), " for ", t.sizes());
  return {t.size(0), cols, t.stride(0)};
}

void check_row_vector(const Tensor& w, const Tensor& x, int64_t cols, const char* what) {
  if (!w.defined()) return;
  on_device(w, what, &x);
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == cols && w.is_contiguous(), what, " must be contiguous [", cols, "], got ",
                    w.sizes());
  TORCH_CHECK_TYPE(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), what, " must be float32 or ",
                   x.scalar_type(), ", got ", w.scalar_type());
}

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* address_of(Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// Whether two tensors' memory has a byte in common.
bool overlap(const Tensor& a, const Tensor& b) {
  if (!a.defined() || !b.defined() || !a.numel() || !b.numel()) return false;
  auto end = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return static_cast<const char*>(t.const_data_ptr()) + (last + 1) * static_cast<int64_t>(t.element_size());
  };
  return static_cast<const char*>(a.const_data_ptr()) < end(b) && static_cast<const char*>(b.const_data_ptr()) < end(a);
}

Tensor ln_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor out, Tensor* mean, Tensor* rstd) {
  on_device(x, "x");
  const int t = type_code(x.scalar_type());
  TORCH_CHECK_TYPE(t >= 0, "layer_norm computes on float32, bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(static_cast<float>(eps)), "eps must be finite and not negative, got ", eps);
  const Rows r = rows_of(x, "x");
  check_row_vector(w, x, r.cols, "weight");
  check_row_vector(b, x, r.cols, "bias");
  TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight is ", w.scalar_type(),
                   " and bias ", b.scalar_type(), ": both must be of one type");
  if (out.defined()) {
    on_device(out, "out", &x);
    TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && out.is_contiguous(),
                      "out must be contiguous ", x.sizes(), " ", x.scalar_type());
    TORCH_CHECK_VALUE(!overlap(out, w) && !overlap(out, b) &&
                      (!overlap(out, x) || (x.is_contiguous() && out.const_data_ptr() == x.const_data_ptr())),
                      "out may be x itself, and may not overlap it, weight or bias otherwise");
  } else {
    out = at::empty(x.sizes(), x.options());
  }
  if (mean) {
    *mean = f32_on(x, x.sizes().slice(0, x.dim() - 1));
    *rstd = f32_on(x, x.sizes().slice(0, x.dim() - 1));
  }
  const int wt = w.defined() ? type_code(w.scalar_type()) : b.defined() ? type_code(b.scalar_type()) : IADMM_F32;
  const c10::DeviceGuard guard(x.device());
  done("iadmm_layer_norm_fwd",
       abi.ln_fwd(r.rows, r.cols, t, wt, x.const_data_ptr(), r.ld, address(w), address(b), static_cast<float>(eps),
                  out.mutable_data_ptr(), mean ? mean->mutable_data_ptr<float>() : nullptr,
                  rstd ? rstd->mutable_data_ptr<float>() : nullptr, stream_of(x.device())));
  return out;
}

std::vector<Tensor> ln_backward(const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd, const Tensor& w,
                                at::ScalarType wtype, bool need_x, bool need_w, bool need_b) {
  on_device(x, "x");
  const int t = type_code(x.scalar_type());
  TORCH_CHECK_TYPE(t >= 0 && dy.scalar_type() == x.scalar_type(),
                   "x and dy must be of one type of float32, bfloat16 and float16, got ", x.scalar_type(), ", ",
                   dy.scalar_type());
  on_device(dy, "dy", &x);
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy is ", dy.sizes(), ", x ", x.sizes());
  const Rows r = rows_of(x, "x"), d = rows_of(dy, "dy");
  for (const Tensor* s : {&mean, &rstd}) {
    on_device(*s, "mean or rstd", &x);
    TORCH_CHECK_VALUE(s->scalar_type() == at::kFloat && s->is_contiguous() && s->numel() == r.rows,
                      "mean and rstd must be contiguous float32 with ", r.rows, " values");
  }
  check_row_vector(w, x, r.cols, "weight");
  if (w.defined()) wtype = w.scalar_type();
  TORCH_CHECK_TYPE(wtype == at::kFloat || wtype == x.scalar_type(), "wdtype must be float32 or ", x.scalar_type(), ", got ",
                   wtype);
  Tensor dx, dw, db, ws;
  if (need_x) dx = at::empty(x.sizes(), x.options());
  if (need_w) dw = at::empty({r.cols}, x.options().dtype(wtype));
  if (need_b) db = at::empty({r.cols}, x.options().dtype(wtype));
  int64_t bytes = 0;
  if (need_w || need_b) {
    bytes = abi.ln_bwd_ws_bytes(r.rows, r.cols, t);
    if (bytes) ws = f32_on(x, {bytes / 4});
  }
  const c10::DeviceGuard guard(x.device());
  done("iadmm_layer_norm_bwd",
       abi.ln_bwd(r.rows, r.cols, t, type_code(wtype), dy.const_data_ptr(), d.ld, x.const_data_ptr(), r.ld,
                  mean.const_data_ptr<float>(), rstd.const_data_ptr<float>(), address(w), address_of(dx), address_of(dw),
                  address_of(db), address_of(ws), bytes, stream_of(x.device())));
  return {dx, dw, db};
}

// A leaf's gradients are added up on the stream that its first living graph was made on, which a captured backward pass
// draws into the capture.  Another stream joins it as a fork; the default stream cannot (the process ends): refused before it
// comes to that.
void refuse_default_stream_leaves(const c10::Device& d) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto& edge : node->next_edges()) {
    const auto leaf = std::dynamic_pointer_cast<torch::autograd::AccumulateGrad>(edge.function);
    const auto stream = leaf ? leaf->stream() : std::nullopt;
    TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(d.index()).id(),
                "a captured backward pass of layer_norm: a graph that was made on the default stream from the same leaves is "
                "still alive (delete its outputs, such as a loss, before the capture)");
  }
}

// Saves x and 8 bytes a row.
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor mean, rstd;
    Tensor y = ln_forward(x, w, b, eps, Tensor(), &mean, &rstd);
    ctx->save_for_backward({x, w, mean, rstd});
    ctx->saved_data["bias"] = b.defined();
    ctx->saved_data["wtype"] = static_cast<int64_t>(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat);
    return y;
  }
  static std::vector<Tensor> backward(torch::autograd::AutogradContext* ctx, const std::vector<Tensor>& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    refuse_default_stream_leaves(x.device());
    const Tensor dy = plain_rows(grads[0]);  // (a sum's gradient is expanded)
    std::vector<Tensor> out;
    {
      const at::AutoGradMode off(false);
      out = ln_backward(dy, x, saved[2], saved[3], w, static_cast<at::ScalarType>(ctx->saved_data["wtype"].toInt()),
                        ctx->needs_input_grad(0), w.defined() && ctx->needs_input_grad(1),
                        ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(1 + w.defined()));
    }
    out.emplace_back();
    if (at::GradMode::is_enabled()) {  // the kernels are no graph: whoever differentiates the gradient hears of it
      std::vector<Tensor> all = out;
      for (const Tensor& t : {x, w, grads[0]}) all.push_back(t);  // (what it depends on)
      const size_t n = all.size();
      all = torch::autograd::DelayedError("layer_norm's gradient has no gradient of its own", n).apply(std::move(all));
      std::copy_n(all.begin(), out.size(), out.begin());
    }
    return out;
  }
};

// -------------------------------------------------------------------------------------- the optimizer's step
struct List {
  std::vector<Tensor> t;
  c10::Device device{at::kCPU};
};

// The items that `use` names, contiguous, on one device and of the given types.
List list_of(PyObject* seq, const char* what, std::initializer_list<at::ScalarType> types, const std::vector<int>& use) {
  List l;
  l.t.reserve(use.size());
  for (const int i : use) {
    PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must hold tensors");
    l.t.push_back(THPVariable_Unpack(o));
    const Tensor& t = l.t.back();
    TORCH_CHECK_TYPE(std::find(types.begin(), types.end(), t.scalar_type()) != types.end(), what, " must be ",
                     *types.begin(), types.size() > 1 ? " or " : "", types.size() > 1 ? toString(*(types.end() - 1)) : "",
                     ", got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg(), what, " must be contiguous");
    TORCH_CHECK_VALUE(t.is_cuda(), "iadmm kernels need device tensors (no CPU fallback), and one of ", what, " is on ",
                      t.device());
    TORCH_CHECK_VALUE(l.t.size() == 1 || t.device() == l.device, what, " must be on one device, got ", t.device(), " and ",
                      l.device);
    l.device = t.device();
  }
  return l;
}

Tensor optional_tensor(PyObject* o, const char* what) {
  if (o == Py_None) return Tensor();
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}

struct Fast {  // a list or tuple for as long as it is read
  PyObject* o;
  Fast(PyObject* from, const char* what) : o(PySequence_Fast(from, what)) {
    if (!o) throw python_error();
  }
  ~Fast() { Py_DECREF(o); }
  int size() const { return static_cast<int>(PySequence_Fast_GET_SIZE(o)); }
};

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

PyObject* tuple_of(const Tensor* t, int n) {
  PyObject* out = PyTuple_New(n);
  if (!out) throw python_error();
  for (int i = 0; i < n; ++i) PyTuple_SET_ITEM(out, i, wrap(t[i]));
  return out;
}

void want(Py_ssize_t n, Py_ssize_t count) { TORCH_CHECK_TYPE(n == count, "expected ", count, " arguments, got ", n); }

// ------------------------------------------------------------------------------------------- Python's entries
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 7);
  void* p[7];
  for (int i = 0; i < 7; ++i)
    if (!(p[i] = PyLong_AsVoidPtr(a[i]))) throw python_error();
  abi.ln_fwd = reinterpret_cast<decltype(abi.ln_fwd)>(p[0]);
  abi.ln_bwd_ws_bytes = reinterpret_cast<decltype(abi.ln_bwd_ws_bytes)>(p[1]);
  abi.ln_bwd = reinterpret_cast<decltype(abi.ln_bwd)>(p[2]);
  abi.norm_ws_bytes = reinterpret_cast<decltype(abi.norm_ws_bytes)>(p[3]);
  abi.norm = reinterpret_cast<decltype(abi.norm)>(p[4]);
  abi.adamw_ws_bytes = reinterpret_cast<decltype(abi.adamw_ws_bytes)>(p[5]);
  abi.adamw_step = reinterpret_cast<decltype(abi.adamw_step)>(p[6]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// layer_norm(x, weight, bias, eps, out, stats)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 6);
  not_traced();
  TORCH_CHECK_TYPE(THPVariable_Check(a[0]), "x must be a tensor");
  const Tensor x = THPVariable_Unpack(a[0]), w = optional_tensor(a[1], "weight"), b = optional_tensor(a[2], "bias");
  const double eps = number(a[3]);
  const bool stats = PyObject_IsTrue(a[5]) == 1;
  const at::AutoGradMode off(false);
  Tensor t[3];
  t[0] = ln_forward(x, w, b, eps, optional_tensor(a[4], "out"), stats ? &t[1] : nullptr, stats ? &t[2] : nullptr);
  if (a[4] != Py_None) written(t[0]);
  if (stats) return tuple_of(t, 3);
  return wrap(t[0]);
  END_HANDLE_TH_ERRORS
}

// layer_norm_bwd(dy, x, mean, rstd, weight, type code without a weight, need_x, need_w, need_b)
PyObject* py_layer_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 9);
  not_traced();
  for (int i = 0; i < 4; ++i) TORCH_CHECK_TYPE(THPVariable_Check(a[i]), "dy, x, mean and rstd must be tensors");
  const Tensor w = optional_tensor(a[4], "weight");
  const long half = PyLong_AsLong(a[5]);  // include/iadmm.h's type code
  if (half == -1 && PyErr_Occurred()) throw python_error();
  const at::AutoGradMode off(false);
  const auto out = ln_backward(THPVariable_Unpack(a[0]), THPVariable_Unpack(a[1]), THPVariable_Unpack(a[2]),
                               THPVariable_Unpack(a[3]), w,
                               half == IADMM_BF16 ? at::kBFloat16 : half == IADMM_F16 ? at::kHalf : at::kFloat,
                               PyObject_IsTrue(a[6]) == 1, PyObject_IsTrue(a[7]) == 1, PyObject_IsTrue(a[8]) == 1);
  return tuple_of(out.data(), 3);
  END_HANDLE_TH_ERRORS
}

// layer_norm_grad(x, weight, bias, eps): differentiable
PyObject* py_layer_norm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 4);
  not_traced();
  TORCH_CHECK_TYPE(THPVariable_Check(a[0]), "x must be a tensor");
  const Tensor x = THPVariable_Unpack(a[0]), w = optional_tensor(a[1], "weight"), b = optional_tensor(a[2], "bias");
  const double eps = number(a[3]);
  TORCH_CHECK_VALUE(x.layout() == at::kStrided, "x must be a dense tensor");
  const std::optional<Tensor> weight = w.defined() ? std::optional(w) : std::nullopt,
                              bias = b.defined() ? std::optional(b) : std::nullopt;  // (edges only for those that are)
  return wrap(LayerNorm::apply(plain_rows(x), weight, bias, eps));
  END_HANDLE_TH_ERRORS
}

// grad_norm(grads)
PyObject* py_grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 1);
  not_traced();
  const Fast grads(a[0], "gradients must be a list");
  std::vector<int> use;
  for (int i = 0; i < grads.size(); ++i)
    if (PySequence_Fast_GET_ITEM(grads.o, i) != Py_None) use.push_back(i);
  TORCH_CHECK_VALUE(!use.empty(), "grad_norm needs at least one gradient");
  const List l = list_of(grads.o, "gradients", {at::kFloat, at::kBFloat16}, use);
  std::vector<iadmm_grad_tensor> rec;
  rec.reserve(l.t.size());
  for (const Tensor& t : l.t) rec.push_back({t.const_data_ptr(), t.numel(), type_code(t.scalar_type())});
  const int64_t count = static_cast<int64_t>(rec.size()), bytes = abi.norm_ws_bytes(count);
  const at::AutoGradMode off(false);
  Tensor ws = f32_on(l.t[0], {bytes / 4}), norm = f32_on(l.t[0], {});
  const c10::DeviceGuard guard(l.device);
  done("iadmm_grad_norm", abi.norm(count, rec.data(), norm.mutable_data_ptr<float>(), ws.mutable_data_ptr(), bytes,
                                   stream_of(l.device)));
  return wrap(norm);
  END_HANDLE_TH_ERRORS
}

// The bytes of a tensor, and whether the call writes them.
struct Held {
  uintptr_t from, to;
  bool written;
  Held(const void* p, int64_t bytes, bool w)
      : from(reinterpret_cast<uintptr_t>(p)), to(from + static_cast<uintptr_t>(bytes)), written(w) {}
};
// Whether what is written overlaps nothing else.
bool apart(std::vector<Held>& held) {
  std::sort(held.begin(), held.end(), [](const Held& a, const Held& b) { return a.from < b.from; });
  uintptr_t all = 0, written = 0;  // where the tensors so far end
  for (const Held& h : held) {
    if (h.from < (h.written ? all : written)) return false;
    all = std::max(all, h.to);
    if (h.written) written = std::max(written, h.to);
  }
  return true;
}

// adamw_step(params, grads, exp_avgs, exp_avg_sqs, exponents, step, lr, beta1, beta2, eps, weight_decay, norm,
//            max_norm, seed); step: a number, a list of them or an int64 tensor
PyObject* py_adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 14);
  not_traced();
  const Fast params(a[0], "params must be a list"), grads(a[1], "grads must be a list"),
      avgs(a[2], "exp_avgs must be a list"), sqs(a[3], "exp_avg_sqs must be a list");
  const bool eight = a[4] != Py_None, counted = THPVariable_Check(a[5]), numbers = !counted && !PyIndex_Check(a[5]);
  const Fast exps(eight ? a[4] : a[0], "exponents must be a list");
  const Fast steps(numbers ? a[5] : a[0], "step must be a number, a list of numbers or a tensor");
  const int count = params.size();
  TORCH_CHECK_VALUE(grads.size() == count && avgs.size() == count && sqs.size() == count && exps.size() == count &&
                    steps.size() == count, "the lists must have one entry per parameter");
  TORCH_CHECK_VALUE((a[11] != Py_None) == (a[12] != Py_None), "norm and max_norm belong together");
  std::vector<int> use;
  use.reserve(count);
  for (int i = 0; i < count; ++i)
    if (PySequence_Fast_GET_ITEM(grads.o, i) != Py_None) use.push_back(i);
  if (use.empty()) Py_RETURN_NONE;
  const at::ScalarType state = eight ? at::kByte : at::kFloat;
  const List p = list_of(params.o, "params", {at::kFloat, at::kBFloat16}, use);
  const List g = list_of(grads.o, "grads", {at::kFloat, at::kBFloat16}, use);
  const List m = list_of(avgs.o, "exp_avgs", {state}, use), v = list_of(sqs.o, "exp_avg_sqs", {state}, use);
  const List e = eight ? list_of(exps.o, "exponents", {at::kChar}, use) : List{};
  for (const List* l : {&g, &m, &v, &e})
    TORCH_CHECK_VALUE(l->t.empty() || l->device == p.device, "all tensors must be on one device, got ", l->device, " and ",
                      p.device);
  const double lr = THPVariable_Check(a[6]) ? 0.0 : number(a[6]), b1 = number(a[7]), b2 = number(a[8]), eps = number(a[9]),
               decay = number(a[10]);
  const Tensor lr_dev = THPVariable_Check(a[6]) ? THPVariable_Unpack(a[6]) : Tensor(), norm = optional_tensor(a[11], "norm"),
               counts = counted ? THPVariable_Unpack(a[5]) : Tensor();
  const double most = norm.defined() ? number(a[12]) : 0.0;
  const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[13]);
  if (PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(lr >= 0.0 && std::isfinite(lr) && b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && eps >= 0.0 &&
                    std::isfinite(eps) && decay >= 0.0 && std::isfinite(decay),
                    "lr ", lr, ", betas ", b1, ", ", b2, ", eps ", eps, " or weight_decay ", decay, " is out of range");
  TORCH_CHECK_TYPE(!lr_dev.defined() || counted, "lr on the device needs step on the device");
  for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{lr_dev, "lr"}, {norm, "norm"}})
    TORCH_CHECK_VALUE(!t.defined() || (t.device() == p.device && t.scalar_type() == at::kFloat && t.numel() == 1), what,
                      " must be one float32 value on ", p.device);
  for (const Tensor* t : {&lr_dev, &norm, &counts})
    TORCH_CHECK_VALUE(!t->defined() || t->const_data_ptr(), "lr, norm or step has no memory");
  TORCH_CHECK_VALUE(!norm.defined() || most > 0.0, "max_norm must be positive, got ", most);
  TORCH_CHECK_VALUE(!counted || (counts.device() == p.device && counts.scalar_type() == at::kLong && counts.dim() == 1 &&
                                 counts.size(0) == count && counts.is_contiguous()),
                    "step must be contiguous int64 [", count, "] on ", p.device);
  int64_t step = 0;
  if (!counted && !numbers) step = PyLong_AsLongLong(a[5]);
  std::vector<iadmm_adamw_tensor> rec(use.size());
  std::vector<Held> held;
  held.reserve(use.size() * 5 + 3);
  if (counted) held.emplace_back(counts.const_data_ptr(), count * static_cast<int64_t>(sizeof(int64_t)), true);
  for (const Tensor* t : {&lr_dev, &norm})
    if (t->defined()) held.emplace_back(t->const_data_ptr(), 4, false);
  for (size_t k = 0; k < use.size(); ++k) {
    const int64_t size = p.t[k].numel();
    TORCH_CHECK_VALUE(g.t[k].sizes() == p.t[k].sizes(), "gradient ", use[k], " is ", g.t[k].sizes(), ", its parameter ",
                      p.t[k].sizes());
    TORCH_CHECK_VALUE(m.t[k].numel() == size && v.t[k].numel() == size && (!eight || e.t[k].numel() == (size + 255) / 256 * 2),
                      "the moments of parameter ", use[k], " do not match its size");
    if (numbers) {
      step = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(steps.o, use[k]));
    }
    if (step == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(counted || step >= 1, "steps are counted from 1, got ", step);
    iadmm_adamw_tensor& r = rec[k];
    r.p = p.t[k].mutable_data_ptr();
    r.g = g.t[k].const_data_ptr();
    r.m = m.t[k].mutable_data_ptr();
    r.v = v.t[k].mutable_data_ptr();
    r.e = eight ? e.t[k].mutable_data_ptr() : nullptr;
    r.n = size;
    r.step = step;
    r.slot = use[k];
    r.dtype = static_cast<int16_t>(type_code(p.t[k].scalar_type()));
    r.gdtype = static_cast<int16_t>(type_code(g.t[k].scalar_type()));
    if (size > 0) {
      const int64_t moments = size * (eight ? 1 : 4);
      held.emplace_back(r.p, size * (r.dtype ? 2 : 4), true);
      held.emplace_back(r.g, size * (r.gdtype ? 2 : 4), false);
      held.emplace_back(r.m, moments, true);
      held.emplace_back(r.v, moments, true);
      if (eight) held.emplace_back(r.e, (size + 255) / 256 * 2, true);
    }
  }
  TORCH_CHECK_VALUE(apart(held), "a parameter or its state is in the lists twice, or overlaps another tensor of the call");
  const int64_t many = static_cast<int64_t>(rec.size()), bytes = abi.adamw_ws_bytes(many);
  const at::AutoGradMode off(false);
  Tensor ws = counted || many > 48 ? f32_on(p.t[0], {bytes / 4}) : Tensor();  // (include/iadmm.h: when it is used)
  const c10::DeviceGuard guard(p.device);
  done("iadmm_adamw_step",
       abi.adamw_step(many, rec.data(), eight ? 8 : 32, lr, lr_dev.defined() ? lr_dev.const_data_ptr<float>() : nullptr, b1, b2,
                      eps, decay, norm.defined() ? norm.const_data_ptr<float>() : nullptr, most, seed,
                      counted ? counts.mutable_data_ptr<int64_t>() : nullptr, address_of(ws), bytes, stream_of(p.device)));
  for (const List* l : {&p, &m, &v, &e})
    for (const Tensor& t : l->t) written(t);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define ENTRY(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY("bind", py_bind),
                         ENTRY("layer_norm", py_layer_norm),
                         ENTRY("layer_norm_bwd", py_layer_norm_bwd),
                         ENTRY("layer_norm_grad", py_layer_norm_grad),
                         ENTRY("grad_norm", py_grad_norm),
                         ENTRY("adamw_step", py_adamw_step),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
