// The autograd nodes of the attention ops and of the q / k prologue, and the launch of a
// cached step whose arguments need no conversion, in C++, over
// the C ABI of libmi_attn.so (include/mi_attn.h). flash_cuda.py and prologue.py
// validate, cast and call these; the kernels' arguments, outputs and saved
// tensors are the same as before.
//
// Why: autograd runs a backward on its own device thread. A Python node there
// takes the GIL from the main thread and gives it back, and both threads start
// each half of a step with cold caches, where interpreted code suffers most. A
// small training step is bound by that host path: forward + backward of a small
// attention call 118 -> 74 us, of a small prologue 122 -> 62 us (one box, medians;
// torch's own `mul` takes 55 us forward + backward there). A call that a tracer
// records keeps the Python nodes (flash_cuda._python_node). A cached step is bound by the
// host the same way: decode.attn_tree 18.5 -> 9.1 us, tree_commit 15.6 -> 6.2 us a call.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>

#include "../../include/mi_attn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

void check(int status) { TORCH_CHECK(status == 0, mi_attn_error_string(status)); }

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return MI_F16;
    case at::kBFloat16: return MI_BF16;
    default: return MI_F32;
  }
}

float* floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A gradient as the kernels read it. (It may be a dense piece of a larger tensor's.)
Tensor dense(const Tensor& g, at::ScalarType dt) {
  const Tensor d = g.to(dt).contiguous();
  return aligned16(d) ? d : d.clone();
}

// The node runs once: its gradients cannot be differentiated again
// (torch.autograd.function.once_differentiable).
variable_list once(const variable_list& incoming, variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  bool tracked = false;
  for (const Tensor& g : incoming) tracked = tracked || (g.defined() && g.requires_grad());
  if (!tracked) return out;
  variable_list live;
  for (Tensor& t : out)
    if (t.defined()) live.push_back(t.detach().requires_grad_(true));
  live = torch::autograd::DelayedError(
             "trying to differentiate twice a function that was marked with @once_differentiable",
             static_cast<int64_t>(live.size()))
             .apply(std::move(live));
  size_t i = 0;
  for (Tensor& t : out)
    if (t.defined()) t = live[i++];
  return out;
}

mi_attn_shape shape_of(const Tensor& q, const Tensor& k, int64_t causal, int64_t window, double scale,
                       int64_t sinks, int64_t block) {
  mi_attn_shape s;
  s.B = static_cast<int>(q.size(0));
  s.S = static_cast<int>(q.size(1));
  s.H = static_cast<int>(q.size(2));
  s.Hkv = static_cast<int>(k.size(2));
  s.D = static_cast<int>(q.size(3));
  s.causal = static_cast<int>(causal);
  s.window = static_cast<int>(window);
  s.scale = static_cast<float>(scale);
  s.dtype = code_of(q);
  s.sinks = static_cast<int>(sinks);
  s.block = static_cast<int>(block);
  return s;
}

// Attention on contiguous [B,S,H,D] / [B,S,Hkv,D] tensors returning (O, LSE),
// both differentiable; the LSE's gradient folds into Delta inside the library.
struct Attn : torch::autograd::Function<Attn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const Tensor& v, const MaybeTensor& gate, int64_t causal,
                               int64_t window, int64_t sinks, double scale, int64_t block,
                               bool residual) {
    const c10::DeviceGuard guard(q.device());
    const Tensor z = gate.value_or(Tensor());
    const mi_attn_shape s = shape_of(q, k, causal, window, scale, sinks, block);
    Tensor o = at::empty_like(q), o_res;
    if (residual) o_res = at::empty_like(q);
    Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    hipStream_t st = stream_of(q);
    if (residual)
      check(mi_attn_fwd_res(ptr(q), ptr(k), ptr(v), ptr(o), ptr(o_res), floats(lse), &s, st));
    else if (z.defined())
      check(mi_attn_fwd_gated(ptr(q), ptr(k), ptr(v), floats(z), ptr(o), floats(lse), &s, st));
    else
      check(mi_attn_fwd(ptr(q), ptr(k), ptr(v), ptr(o), floats(lse), &s, st));
    ctx->save_for_backward({q, k, v, o, lse, z, o_res});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["block"] = block;
    ctx->set_materialize_grads(false);
    return {o, lse};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out;
    {
      at::NoGradGuard no_grad;
      const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lse = saved[4],
                   &gate = saved[5], &res = saved[6];
      auto& d = ctx->saved_data;
      const mi_attn_shape s = shape_of(q, k, d["causal"].toInt(), d["window"].toInt(),
                                       d["scale"].toDouble(), d["sinks"].toInt(), d["block"].toInt());
      const c10::DeviceGuard guard(q.device());
      const Tensor dy = grads[0].defined() ? dense(grads[0], q.scalar_type()) : at::zeros_like(o);
      const Tensor dl = grads[1].defined() ? dense(grads[1], at::kFloat) : Tensor();
      Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v), dz;
      long long n = 0;
      check(mi_attn_bwd_workspace(&s, &n));
      const Tensor ws = at::empty({static_cast<int64_t>(n)}, lse.options());
      hipStream_t st = stream_of(q);
      if (res.defined()) {
        check(mi_attn_bwd_res(ptr(q), ptr(k), ptr(v), ptr(o), ptr(res), ptr(dy), floats(lse),
                              floats(dl), floats(ws), ptr(dq), ptr(dk), ptr(dv), &s, st));
      } else if (!gate.defined()) {
        check(mi_attn_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(dy), floats(lse), floats(dl),
                          floats(ws), ptr(dq), ptr(dk), ptr(dv), &s, st));
      } else {
        const Tensor dy_attn = at::empty_like(dy);   // the gradient of O as dK/dV reads it
        dz = at::empty_like(gate);
        if (!dl.defined() && s.dtype == MI_BF16)
          check(mi_attn_bwd_gated_direct(ptr(q), ptr(k), ptr(v), floats(gate), ptr(o), ptr(dy),
                                         floats(lse), floats(ws), ptr(dy_attn), ptr(dq), ptr(dk),
                                         ptr(dv), floats(dz), &s, st));
        else
          check(mi_attn_bwd_gated(ptr(q), ptr(k), ptr(v), floats(gate), ptr(o), ptr(dy), floats(lse),
                                  floats(dl), floats(ws), ptr(dy_attn), ptr(dq), ptr(dk), ptr(dv),
                                  floats(dz), &s, st));
      }
      out = {dq, dk, dv, dz};
    }
    out = once(grads, std::move(out));
    out.resize(10);   // causal .. residual take no gradient
    return out;
  }
};

mi_prologue_shape prologue_shape(const Tensor& x, int out_code, bool norm, bool rope, double eps) {
  mi_prologue_shape s;
  s.B = static_cast<int>(x.size(0));
  s.T = static_cast<int>(x.size(1));
  s.H = static_cast<int>(x.size(2));
  s.D = static_cast<int>(x.size(3));
  s.dtype_in = code_of(x);
  s.dtype_out = out_code;
  s.norm = norm;
  s.rope = rope;
  s.eps = static_cast<float>(eps);
  return s;
}

at::ScalarType type_of(int64_t code) {
  return code == MI_F16 ? at::kHalf : code == MI_BF16 ? at::kBFloat16 : at::kFloat;
}

struct Prologue : torch::autograd::Function<Prologue> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight,
                        const MaybeTensor& cos, const MaybeTensor& sin, double eps, int64_t out_code) {
    const c10::DeviceGuard guard(x.device());
    const Tensor w = weight.value_or(Tensor()), c = cos.value_or(Tensor()), s = sin.value_or(Tensor());
    const mi_prologue_shape shp =
        prologue_shape(x, static_cast<int>(out_code), w.defined(), c.defined(), eps);
    Tensor out = at::empty(x.sizes(), x.options().dtype(type_of(out_code))), rstd;
    if (w.defined())
      rstd = at::empty({x.size(0), x.size(1), x.size(2)}, x.options().dtype(at::kFloat));
    check(mi_qk_prologue_fwd(ptr(x), floats(w), floats(c), floats(s), ptr(out), floats(rstd), &shp,
                             stream_of(x)));
    ctx->save_for_backward({x, w, c, s, rstd});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["out"] = out_code;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out;
    {
      at::NoGradGuard no_grad;
      const Tensor &x = saved[0], &w = saved[1], &c = saved[2], &s = saved[3], &rstd = saved[4];
      const int64_t code = ctx->saved_data["out"].toInt();
      const mi_prologue_shape shp = prologue_shape(x, static_cast<int>(code), w.defined(), c.defined(),
                                                   ctx->saved_data["eps"].toDouble());
      const c10::DeviceGuard guard(x.device());
      const Tensor g = dense(grads[0], type_of(code));
      Tensor dx = at::empty_like(x), dw;
      if (w.defined()) dw = at::empty({x.size(3)}, x.options().dtype(at::kFloat));
      long long n = 0;
      check(mi_qk_prologue_workspace(&shp, &n));
      const Tensor ws = at::empty({static_cast<int64_t>(n > 0 ? n : 1)}, x.options().dtype(at::kFloat));
      check(mi_qk_prologue_bwd(ptr(g), ptr(x), floats(w), floats(c), floats(s), floats(rstd), ptr(dx),
                               floats(dw), floats(ws), &shp, stream_of(x)));
      out = {dx, dw};
    }
    out = once(grads, std::move(out));
    out.resize(6);
    return out;
  }
};

// Differential attention on contiguous [B,S,H,E] / [B,S,Hkv,E] tensors; lam [H].
struct Diff : torch::autograd::Function<Diff> {
  static mi_diff_shape shape(const Tensor& q, const Tensor& k, const Tensor& lam, int64_t causal,
                             double scale) {
    mi_diff_shape s;
    s.B = static_cast<int>(q.size(0));
    s.S = static_cast<int>(q.size(1));
    s.H = static_cast<int>(q.size(2));
    s.Hkv = static_cast<int>(k.size(2));
    s.E = static_cast<int>(q.size(3));
    s.causal = static_cast<int>(causal);
    s.scale = static_cast<float>(scale);
    s.dtype = code_of(q);
    s.lam_dtype = code_of(lam);
    return s;
  }

  static Tensor run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, int64_t causal,
                    double scale, const Tensor& o2, const Tensor& lse) {
    const mi_diff_shape s = shape(q, k, lam, causal, scale);
    Tensor out = at::empty_like(q);
    check(mi_attn_diff_fwd(ptr(q), ptr(k), ptr(v), ptr(lam), ptr(out), ptr(o2), floats(lse), &s,
                           stream_of(q)));
    return out;
  }

  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Tensor& lam, int64_t causal, double scale) {
    const c10::DeviceGuard guard(q.device());
    // What the backward reads.
    const Tensor o2 = at::empty_like(q);
    const Tensor lse = at::empty({2, q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    Tensor out = run(q, k, v, lam, causal, scale, o2, lse);
    ctx->save_for_backward({q, k, v, lam, out, o2, lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out;
    {
      at::NoGradGuard no_grad;
      const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &lam = saved[3], &o = saved[4],
                   &o2 = saved[5], &lse = saved[6];
      const mi_diff_shape s = shape(q, k, lam, ctx->saved_data["causal"].toInt(),
                                    ctx->saved_data["scale"].toDouble());
      const c10::DeviceGuard guard(q.device());
      const Tensor dy = dense(grads[0], q.scalar_type());
      Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
      // Nothing is written for an empty input.
      Tensor dlam = q.numel() ? at::empty_like(lam) : at::zeros_like(lam);
      long long n = 0;
      check(mi_attn_diff_bwd_workspace(&s, &n));
      const Tensor ws = at::empty({static_cast<int64_t>(n)}, lse.options());
      check(mi_attn_diff_bwd(ptr(q), ptr(k), ptr(v), ptr(lam), ptr(o), ptr(o2), ptr(dy), floats(lse),
                             floats(ws), ptr(dq), ptr(dk), ptr(dv), ptr(dlam), &s, stream_of(q)));
      out = {dq, dk, dv, dlam};
    }
    out = once(grads, std::move(out));
    out.resize(6);
    return out;
  }
};

// ---------------------------------------------------------------------------
// Python entry points (validated by the callers)
// ---------------------------------------------------------------------------
bool tensor_arg(PyObject* o, Tensor& out) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  out = THPVariable_Unpack(o);
  return true;
}
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

// attn(q, k, v, gate | None, causal, window, sinks, scale, block, residual) -> (O, LSE).
// `residual` asks for O's rounding residual where the call will be differentiated.
PyObject* py_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, gate;
  TORCH_CHECK_TYPE(n == 10 && tensor_arg(args[0], q) && tensor_arg(args[1], k) &&
                       tensor_arg(args[2], v) && tensor_arg(args[3], gate) && q.defined() &&
                       k.defined() && v.defined(),
                   "attn(q, k, v, gate, causal, window, sinks, scale, block, residual)");
  const int64_t causal = PyLong_AsLongLong(args[4]), window = PyLong_AsLongLong(args[5]),
                sinks = PyLong_AsLongLong(args[6]);
  const double scale = PyFloat_AsDouble(args[7]);
  const int64_t block = PyLong_AsLongLong(args[8]), res = PyLong_AsLongLong(args[9]);
  if (PyErr_Occurred()) throw python_error();
  const bool keep = res && at::GradMode::is_enabled() &&
                    (q.requires_grad() || k.requires_grad() || v.requires_grad());
  variable_list out;
  {
    // As torch's own operators: an allocation may block, or want the GIL for a
    // callback under the allocator's lock.
    pybind11::gil_scoped_release no_gil;
    out = Attn::apply(q, k, v, maybe(gate), causal, window, sinks, scale, block, keep);
  }
  PyObject* o = THPVariable_Wrap(std::move(out[0]));
  if (!o) throw python_error();
  PyObject* lse = THPVariable_Wrap(std::move(out[1]));
  if (!lse) {
    Py_DECREF(o);
    throw python_error();
  }
  PyObject* t = PyTuple_New(2);
  if (!t) {
    Py_DECREF(o);
    Py_DECREF(lse);
    throw python_error();
  }
  PyTuple_SET_ITEM(t, 0, o);
  PyTuple_SET_ITEM(t, 1, lse);
  return t;
  END_HANDLE_TH_ERRORS
}

// prologue(x, weight | None, cos | None, sin | None, eps, out dtype code) -> out.
PyObject* py_prologue(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w, c, s;
  TORCH_CHECK_TYPE(n == 6 && tensor_arg(args[0], x) && tensor_arg(args[1], w) &&
                       tensor_arg(args[2], c) && tensor_arg(args[3], s) && x.defined(),
                   "prologue(x, weight, cos, sin, eps, out_dtype)");
  const double eps = PyFloat_AsDouble(args[4]);
  const int64_t code = PyLong_AsLongLong(args[5]);
  if (PyErr_Occurred()) throw python_error();
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = Prologue::apply(x, maybe(w), maybe(c), maybe(s), eps, code);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

Tensor diff_out(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, int64_t causal,
                double scale) {
  // A node only where one is needed (a forward-mode tangent is the node's to refuse).
  bool node = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() ||
                                             v.requires_grad() || lam.requires_grad());
  for (const Tensor* t : {&q, &k, &v, &lam}) node = node || torch::autograd::isFwGradDefined(*t);
  pybind11::gil_scoped_release no_gil;
  if (node) return Diff::apply(q, k, v, lam, causal, scale);
  at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(q.device());
  return Diff::run(q, k, v, lam, causal, scale, Tensor(), Tensor());
}

// diff_attn(q, k, v, lam, causal, scale) -> out.
PyObject* py_diff_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, lam;
  TORCH_CHECK_TYPE(n == 6 && tensor_arg(args[0], q) && tensor_arg(args[1], k) &&
                       tensor_arg(args[2], v) && tensor_arg(args[3], lam) && q.defined() &&
                       k.defined() && v.defined() && lam.defined(),
                   "diff_attn(q, k, v, lam, causal, scale)");
  const int64_t causal = PyLong_AsLongLong(args[4]);
  const double scale = PyFloat_AsDouble(args[5]);
  if (PyErr_Occurred()) throw python_error();
  Tensor out = diff_out(q, k, v, lam, causal, scale);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// Differential attention and cached steps, for arguments that need no conversion. These
// return None for anything else, refusals included: the Python then converts, or says what is
// wrong.
// ---------------------------------------------------------------------------
bool plain_arg(PyObject* o, Tensor& out) {      // a Tensor itself, or None
  if (o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  out = THPVariable_Unpack(o);
  return true;
}

bool kernel_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// A dense tensor of `dtype` on q's device with these sizes.
bool dense_like(const Tensor& t, const Tensor& q, at::ScalarType dtype, at::IntArrayRef sizes) {
  return t.defined() && t.scalar_type() == dtype && t.device() == q.device() && t.sizes() == sizes &&
         t.is_contiguous();
}

// Cache rows as the kernels read them: D apart, strides and address in 16-byte chunks.
bool cache_ok(const Tensor& t, const Tensor& k) {
  if (!t.defined() || t.dim() != 4 || t.scalar_type() != k.scalar_type() || t.device() != k.device())
    return false;
  const int64_t D = k.size(3), chunk = 16 / t.element_size();
  return t.size(0) == k.size(0) && t.size(1) == k.size(2) && t.size(3) == D && t.stride(3) == 1 &&
         t.stride(2) == D && t.stride(0) % chunk == 0 && t.stride(1) % chunk == 0 && aligned16(t);
}

bool tracked(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Whether k, v [B,T,Hkv,D] are what the kernels read, with nothing for autocast to do.
bool rows_ok(const Tensor& k, const Tensor& v) {
  if (!k.defined() || k.dim() != 4 || !k.is_cuda() || !kernel_type(k.scalar_type()) || !k.is_contiguous())
    return false;
  if (!dense_like(v, k, k.scalar_type(), k.sizes())) return false;
  const int64_t D = k.size(3);
  return (D == 32 || D == 64 || D == 128) && k.size(2) != 0 && aligned16(k) && aligned16(v) && !at::autocast::is_autocast_enabled(at::kCUDA);
}
// ... on the current device, with nothing for autograd to do either.
bool block_ok(const Tensor& k, const Tensor& v) {
  if (!rows_ok(k, v) || k.get_device() != c10::hip::current_device()) return false;
  return !at::GradMode::is_enabled() || (!tracked(k) && !tracked(v));
}

bool fits_int(int64_t n) { return n <= 0x7fffffff; }

mi_step_shape step_shape(const Tensor& q, const Tensor& k, const Tensor& ck, const Tensor& cv) {
  mi_step_shape s = {};
  s.B = static_cast<int>(k.size(0));
  s.T = static_cast<int>(k.size(1));
  s.H = static_cast<int>(q.size(2));
  s.Hkv = static_cast<int>(k.size(2));
  s.D = static_cast<int>(k.size(3));
  s.maps = 1;
  s.scale = 1.f;
  s.dtype = code_of(k);
  if (ck.defined()) {
    s.rows = static_cast<int>(ck.size(2));
    s.k_batch_stride = ck.stride(0);
    s.k_head_stride = ck.stride(1);
    s.v_batch_stride = cv.stride(0);
    s.v_head_stride = cv.stride(1);
  }
  return s;
}

// step(q, k, v, cache k, cache v, lens, parents, lam, gate, causal, scale, return_lse)
// -> out, (out, lse) or None.
PyObject* py_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, ck, cv, lens, parents, lam, gate;
  TORCH_CHECK_TYPE(n == 12, "step(q, k, v, cache_k, cache_v, lens, parents, lam, gate, causal, scale, return_lse)");
  if (!plain_arg(args[0], q) || !plain_arg(args[1], k) || !plain_arg(args[2], v) || !plain_arg(args[3], ck) ||
      !plain_arg(args[4], cv) || !plain_arg(args[5], lens) || !plain_arg(args[6], parents) ||
      !plain_arg(args[7], lam) || !plain_arg(args[8], gate))
    Py_RETURN_NONE;
  const int64_t causal = PyObject_IsTrue(args[9]), want_lse = PyObject_IsTrue(args[11]);
  double scale = 0.0;
  if (args[10] != Py_None) scale = PyFloat_AsDouble(args[10]);
  if (PyErr_Occurred()) throw python_error();
  if (!q.defined() || q.dim() != 4 || !block_ok(k, v) || ck.defined() != cv.defined()) Py_RETURN_NONE;
  const int64_t B = k.size(0), T = k.size(1), Hkv = k.size(2), D = k.size(3), H = q.size(2);
  if (!dense_like(q, k, k.scalar_type(), {B, T, H, D}) || H % Hkv || !aligned16(q)) Py_RETURN_NONE;
  if (ck.defined() && (!cache_ok(ck, k) || !cache_ok(cv, k) || ck.size(2) != cv.size(2) || !fits_int(ck.size(2))))
    Py_RETURN_NONE;
  if (lens.defined() && !dense_like(lens, k, at::kInt, {B})) Py_RETURN_NONE;
  const bool one_tree = parents.defined() && parents.dim() == 1;
  if (parents.defined() && (T > MI_TREE_MAX || !(one_tree ? dense_like(parents, k, at::kInt, {T})
                                                          : dense_like(parents, k, at::kInt, {B, T}))))
    Py_RETURN_NONE;
  if (lam.defined() && (want_lse || !kernel_type(lam.scalar_type()) || !dense_like(lam, k, lam.scalar_type(), {H})))
    Py_RETURN_NONE;
  if (gate.defined() && !dense_like(gate, k, at::kFloat, {B, T, H})) Py_RETURN_NONE;
  if (at::GradMode::is_enabled() && (tracked(q) || tracked(lam) || tracked(gate))) Py_RETURN_NONE;
  if (args[10] == Py_None) scale = std::sqrt((lam.defined() ? 2.0 : 1.0) / static_cast<double>(D));
  if (!std::isfinite(scale) || !(scale > 0.0) || !fits_int(B) || !fits_int(T) || !fits_int(H)) Py_RETURN_NONE;
  mi_step_shape s = step_shape(q, k, ck, cv);
  s.causal = static_cast<int>(causal);
  s.one_tree = one_tree;
  s.scale = static_cast<float>(scale);
  if (lam.defined()) {
    s.maps = 2;
    s.lam_dtype = code_of(lam);
  }
  Tensor out, lse;
  {
    pybind11::gil_scoped_release no_gil;
    at::NoGradGuard no_grad;
    long long floats_ws = 0;
    check(mi_attn_step_workspace(&s, &floats_ws));
    out = at::empty_like(q);
    // From torch's allocator at every call: a captured graph gets one of its own.
    const Tensor ws = floats_ws ? at::empty({static_cast<int64_t>(floats_ws)}, q.options().dtype(at::kFloat))
                                : Tensor();
    if (want_lse) lse = at::empty({B, H, T}, q.options().dtype(at::kFloat));
    check(mi_attn_step(ptr(q), ptr(k), ptr(v), ptr(ck), ptr(cv), static_cast<const int*>(ptr(lens)),
                       static_cast<const int*>(ptr(parents)), ptr(lam), floats(gate), ptr(out), floats(lse),
                       floats(ws), &s, stream_of(q)));
  }
  PyObject* o = THPVariable_Wrap(std::move(out));
  if (!o) throw python_error();
  if (!want_lse) return o;
  PyObject* l = THPVariable_Wrap(std::move(lse));
  PyObject* t = l ? PyTuple_Pack(2, o, l) : nullptr;
  Py_DECREF(o);
  Py_XDECREF(l);
  if (!t) throw python_error();
  return t;
  END_HANDLE_TH_ERRORS
}

// diff(q, k, v, lam, scale or None, causal) -> out, or None.
PyObject* py_diff(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, lam;
  TORCH_CHECK_TYPE(n == 6, "diff(q, k, v, lam, scale, causal)");
  if (!plain_arg(args[0], q) || !plain_arg(args[1], k) || !plain_arg(args[2], v) || !plain_arg(args[3], lam))
    Py_RETURN_NONE;
  const int causal = PyObject_IsTrue(args[5]);
  double scale = 0.0;
  if (args[4] != Py_None) scale = PyFloat_AsDouble(args[4]);
  if (PyErr_Occurred()) throw python_error();
  if (!q.defined() || q.dim() != 4 || !lam.defined() || !rows_ok(k, v)) Py_RETURN_NONE;
  const int64_t H = q.size(2), E = k.size(3);
  if (!dense_like(q, k, k.scalar_type(), {k.size(0), k.size(1), H, E}) || H % k.size(2) || q.numel() == 0 || !aligned16(q) ||
      !kernel_type(lam.scalar_type()) || !dense_like(lam, k, lam.scalar_type(), {H}))
    Py_RETURN_NONE;
  if (args[4] == Py_None) scale = std::sqrt(2.0 / static_cast<double>(E));
  if (!std::isfinite(scale) || !(scale > 0.0)) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i)
    if (!fits_int(q.size(i))) Py_RETURN_NONE;
  return THPVariable_Wrap(diff_out(q, k, v, lam, causal, scale));
  END_HANDLE_TH_ERRORS
}

// tree_commit(k, v, cache k, cache v, lens, path, count) -> the new lens or None.
PyObject* py_tree_commit(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor k, v, ck, cv, lens, path, count;
  TORCH_CHECK_TYPE(n == 7, "tree_commit(k, v, cache_k, cache_v, lens, path, count)");
  if (!plain_arg(args[0], k) || !plain_arg(args[1], v) || !plain_arg(args[2], ck) || !plain_arg(args[3], cv) ||
      !plain_arg(args[4], lens) || !plain_arg(args[5], path) || !plain_arg(args[6], count))
    Py_RETURN_NONE;
  if (!block_ok(k, v) || !cache_ok(ck, k) || !cache_ok(cv, k) || ck.size(2) != cv.size(2)) Py_RETURN_NONE;
  for (const Tensor* t : {&ck, &cv})             // sequences or heads that share their rows
    if ((t->size(0) > 1 && t->stride(0) == 0) || (t->size(1) > 1 && t->stride(1) == 0)) Py_RETURN_NONE;
  const int64_t B = k.size(0);
  if (!path.defined() || path.dim() != 2) Py_RETURN_NONE;
  const int64_t P = path.size(1);
  if (!dense_like(lens, k, at::kInt, {B}) || !dense_like(path, k, at::kInt, {B, P}) ||
      !dense_like(count, k, at::kInt, {B}) || !fits_int(B) || !fits_int(k.size(1)) || !fits_int(P) ||
      !fits_int(ck.size(2)))
    Py_RETURN_NONE;
  const mi_step_shape s = step_shape(k, k, ck, cv);
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    at::NoGradGuard no_grad;
    out = at::empty_like(lens);
    check(mi_attn_tree_commit(ptr(k), ptr(v), ptr(ck), ptr(cv), static_cast<const int*>(ptr(lens)),
                              static_cast<const int*>(ptr(path)), static_cast<const int*>(ptr(count)),
                              static_cast<int*>(ptr(out)), static_cast<int>(P), &s, stream_of(k)));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_attn)), METH_FASTCALL,
     "attn(q, k, v, gate, causal, window, sinks, scale, block, residual) -> (O, LSE)"},
    {"prologue", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_prologue)), METH_FASTCALL,
     "prologue(x, weight, cos, sin, eps, out_dtype) -> out"},
    {"diff_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_diff_attn)), METH_FASTCALL,
     "diff_attn(q, k, v, lam, causal, scale) -> out"},
    {"diff", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_diff)), METH_FASTCALL,
     "diff(q, k, v, lam, scale, causal) -> out or None"},
    {"step", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_step)), METH_FASTCALL,
     "step(q, k, v, cache_k, cache_v, lens, parents, lam, gate, causal, scale, return_lse) -> out, (out, lse) or None"},
    {"tree_commit", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_tree_commit)), METH_FASTCALL,
     "tree_commit(k, v, cache_k, cache_v, lens, path, count) -> lens or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mi_torch", nullptr, -1, methods, nullptr, nullptr,
                      nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mi_torch(void) { return PyModule_Create(&module); }
