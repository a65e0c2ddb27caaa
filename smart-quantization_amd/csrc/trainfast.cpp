// trainfast.cpp — the eager host path of the training-step operators on at::Tensor (module _smqtrain,
// built next to libsmq.so and linked to it and to libtorch): allocation, launch and autograd node of
//
//   group_norm(x, weight | None, bias | None, groups, eps, activation)
//   linear_ce(hidden, weight, bias | None, target, ignore_index, reduction, piece)
//   orthogonalize(x, steps, a, b, c, eps)
//
// in one C call each. Small tensors are bound by the host: the Python autograd Functions of
// util/pytorch/{norm,loss}.py, which do the same through ctypes and serve where this module is absent,
// cost 20-40 us a pass more. The callers there have checked the arguments. Workspaces come from
// torch's allocator per call: returned in stream order, private to a graph's pool during a capture.
// Nothing here crosses the C-ABI (include/smq.h); exceptions end at the entry points.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "smq.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<at::Tensor>;

int code_of(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat  ? SMQ_DTYPE_F32
         : t.scalar_type() == at::kHalf ? SMQ_DTYPE_F16
                                        : SMQ_DTYPE_BF16;
}
void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
at::Tensor buffer(const at::Tensor& like, size_t bytes, const char* who) {
  TORCH_CHECK(bytes > 0, who, ": ", smq_last_error());
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}
void ok(int rc, const char* who) { TORCH_CHECK(rc == SMQ_OK, who, " failed (rc=", rc, "): ", smq_last_error()); }
at::Tensor f32(const at::Tensor& t) {
  return t.defined() ? t.detach().to(at::kFloat).contiguous() : at::Tensor();
}
const float* fptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
float* fout(at::Tensor& t) { return t.defined() ? t.mutable_data_ptr<float>() : nullptr; }
void only_once(const char* who) {
  TORCH_CHECK(!at::GradMode::is_enabled(), who, " has no second derivative (create_graph=True)");
}

// ---- group norm -----------------------------------------------------------------------------------
// A new tensor of x's shape in channels-last memory. No view: autograd refuses to change a view that a
// custom function returns in place, and what follows a normalisation often does (out += identity).
at::Tensor channels_last_like(const at::Tensor& x) {
  at::DimVector strides(x.dim());
  int64_t step = x.size(1);
  strides[1] = 1;
  for (int64_t d = x.dim() - 1; d > 1; d--) strides[d] = step, step *= x.size(d);
  strides[0] = step;
  return at::empty_strided(x.sizes(), strides, x.options());
}

struct GroupNorm : Function<GroupNorm> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& weight_,
                            const MaybeTensor& bias_, int64_t groups, double eps, int64_t act) {
    const at::Tensor weight = weight_.value_or(at::Tensor()), bias = bias_.value_or(at::Tensor());
    const at::Tensor xl = x.detach().movedim(1, -1).contiguous();
    const int64_t n = xl.size(0), c = xl.size(-1), s = xl.numel() / (n * c);
    const c10::DeviceGuard guard(x.device());
    at::Tensor y = channels_last_like(x);
    at::Tensor stats = at::empty({2, n, groups}, x.options().dtype(at::kFloat));
    const size_t need = smq_group_norm_workspace_bytes(code_of(x), n, s, c, groups, 0);
    const at::Tensor ws = buffer(x, need, "group_norm_act"), w = f32(weight), b = f32(bias);
    float* st = stats.mutable_data_ptr<float>();
    ok(smq_group_norm_act(xl.const_data_ptr(), code_of(x), y.mutable_data_ptr(), n, s, c, groups, fptr(w),
                          fptr(b), eps, (int)act, st, st + n * groups, ws.data_ptr(), need, stream_of(x)),
       "group_norm_act");
    ctx->save_for_backward({x, weight, bias, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    only_once("group_norm_act");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    const int64_t groups = ctx->saved_data["groups"].toInt();
    const at::Tensor xl = x.detach().movedim(1, -1).contiguous(), dl = grads[0].movedim(1, -1).contiguous();
    const int64_t n = xl.size(0), c = xl.size(-1), s = xl.numel() / (n * c);
    const c10::DeviceGuard guard(x.device());
    at::Tensor dx = channels_last_like(x), dw, db;
    const auto fopt = x.options().dtype(at::kFloat);
    // (edges are counted over the tensors that are there)
    if (weight.defined() && ctx->needs_input_grad(1)) dw = at::empty({c}, fopt);
    if (bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1)) db = at::empty({c}, fopt);
    const size_t need = smq_group_norm_workspace_bytes(code_of(x), n, s, c, groups, 1);
    const at::Tensor ws = buffer(x, need, "group_norm_act backward"), w = f32(weight), b = f32(bias);
    const float* st = stats.const_data_ptr<float>();
    ok(smq_group_norm_act_backward(xl.const_data_ptr(), dl.const_data_ptr(), code_of(x),
                                   dx.mutable_data_ptr(), n, s, c, groups, fptr(w), fptr(b),
                                   (int)ctx->saved_data["act"].toInt(), st, st + n * groups, fout(dw),
                                   fout(db), ws.data_ptr(), need, stream_of(x)),
       "group_norm_act backward");
    if (dw.defined()) dw = dw.to(weight.scalar_type());
    if (db.defined()) db = db.to(bias.scalar_type());
    return {dx, dw, db, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ---- cross entropy of a linear head -----------------------------------------------------------------
// The matrix with unit column stride and rows that do not overlap (a copy where it has not).
at::Tensor rows_of(const at::Tensor& t) {
  const bool cols = t.size(1) == 1 || t.stride(1) == 1;
  const bool rows = t.size(0) == 1 || t.stride(0) >= t.size(1);
  return cols && rows ? t.detach() : t.detach().contiguous();
}
int64_t pitch_of(const at::Tensor& t) {
  return t.size(0) > 1 && t.stride(0) > t.size(1) ? t.stride(0) : t.size(1);
}

struct LinearCe : Function<LinearCe> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& hidden, const at::Tensor& weight,
                            const MaybeTensor& bias_, const at::Tensor& target, int64_t ignore,
                            int64_t reduction, int64_t piece) {
    const at::Tensor bias = bias_.value_or(at::Tensor());
    const at::Tensor h = rows_of(hidden), w = rows_of(weight), b = f32(bias), t = target.contiguous();
    const int64_t tokens = h.size(0), dim = h.size(1), vocab = w.size(0);
    const c10::DeviceGuard guard(h.device());
    const auto fopt = h.options().dtype(at::kFloat);
    at::Tensor loss = reduction == SMQ_REDUCE_NONE ? at::empty({tokens}, fopt) : at::empty({}, fopt);
    at::Tensor lse = at::empty({tokens}, fopt);
    at::Tensor head = at::empty({SMQ_CE_HEAD_BYTES}, h.options().dtype(at::kByte));
    const size_t need = smq_linear_ce_workspace_bytes(h.const_data_ptr(), pitch_of(h), w.const_data_ptr(),
                                                      pitch_of(w), code_of(h), tokens, dim, vocab, 0, 0);
    const at::Tensor ws = buffer(h, need, "linear_cross_entropy");
    ok(smq_linear_ce_forward(h.const_data_ptr(), pitch_of(h), w.const_data_ptr(), pitch_of(w), code_of(h),
                             t.const_data_ptr<int64_t>(), fptr(b), tokens, dim, vocab, ignore,
                             (int)reduction, loss.mutable_data_ptr<float>(), lse.mutable_data_ptr<float>(),
                             head.data_ptr(), ws.data_ptr(), need, stream_of(h)),
       "linear_cross_entropy");
    ctx->save_for_backward({hidden, weight, bias, t, lse, head});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["piece"] = piece;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    only_once("linear_cross_entropy");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &bias = saved[2], &t = saved[3], &lse = saved[4], &head = saved[5];
    const at::Tensor h = rows_of(saved[0]), w = rows_of(saved[1]), b = f32(bias), g = f32(grads[0]);
    const int64_t tokens = h.size(0), dim = h.size(1), vocab = w.size(0);
    const int64_t piece = ctx->saved_data["piece"].toInt();
    const c10::DeviceGuard guard(h.device());
    at::Tensor dh, dw, db;
    int flags = 0;
    if (ctx->needs_input_grad(0)) dh = at::empty({tokens, dim}, h.options()), flags |= SMQ_CE_GRAD_HIDDEN;
    if (ctx->needs_input_grad(1)) dw = at::empty({vocab, dim}, w.options()), flags |= SMQ_CE_GRAD_WEIGHT;
    if (bias.defined() && ctx->needs_input_grad(2))
      db = at::empty({vocab}, h.options().dtype(at::kFloat)), flags |= SMQ_CE_GRAD_BIAS;
    const size_t need =
        smq_linear_ce_workspace_bytes(h.const_data_ptr(), pitch_of(h), w.const_data_ptr(), pitch_of(w),
                                      code_of(h), tokens, dim, vocab, piece, flags);
    const at::Tensor ws = buffer(h, need, "linear_cross_entropy backward");
    ok(smq_linear_ce_backward(h.const_data_ptr(), pitch_of(h), w.const_data_ptr(), pitch_of(w), code_of(h),
                              t.const_data_ptr<int64_t>(), fptr(b), tokens, dim, vocab,
                              ctx->saved_data["ignore"].toInt(), (int)ctx->saved_data["reduction"].toInt(),
                              lse.const_data_ptr<float>(), head.data_ptr(), fptr(g),
                              dh.defined() ? dh.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr,
                              fout(db), piece, ws.data_ptr(), need, stream_of(h)),
       "linear_cross_entropy backward");
    if (db.defined()) db = db.to(bias.scalar_type());
    return {dh, dw, db, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ---- entry points -----------------------------------------------------------------------------------
template <typename T>  // at::Tensor, or MaybeTensor where None may stand
bool tensor_arg(PyObject* o, T* t, bool optional) {
  if (optional && o == Py_None) return true;
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "tensor expected");
    return false;
  }
  *t = THPVariable_Unpack(o);
  return true;
}
// Errors become Python's: what a saved-tensor hook raised as it is, no memory as OutOfMemoryError.
template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  return THPVariable_Wrap(f());
  END_HANDLE_TH_ERRORS
}

PyObject* group_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "group_norm(x, weight, bias, groups, eps, activation)");
    return nullptr;
  }
  at::Tensor x;
  MaybeTensor w, b;
  if (!tensor_arg(a[0], &x, false) || !tensor_arg(a[1], &w, true) || !tensor_arg(a[2], &b, true)) return nullptr;
  const int64_t groups = PyLong_AsLongLong(a[3]);
  const double eps = PyFloat_AsDouble(a[4]);
  const int64_t act = PyLong_AsLongLong(a[5]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&] { return GroupNorm::apply(x, w, b, groups, eps, act); });
}

PyObject* linear_ce(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "linear_ce(hidden, weight, bias, target, ignore_index, reduction, piece)");
    return nullptr;
  }
  at::Tensor h, w, t;
  MaybeTensor b;
  if (!tensor_arg(a[0], &h, false) || !tensor_arg(a[1], &w, false) || !tensor_arg(a[2], &b, true) ||
      !tensor_arg(a[3], &t, false))
    return nullptr;
  const int64_t ignore = PyLong_AsLongLong(a[4]), red = PyLong_AsLongLong(a[5]), piece = PyLong_AsLongLong(a[6]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&] { return LinearCe::apply(h, w, b, t, ignore, red, piece); });
}

PyObject* orthogonalize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "orthogonalize(x, steps, a, b, c, eps)");
    return nullptr;
  }
  at::Tensor u;
  if (!tensor_arg(a[0], &u, false)) return nullptr;
  const int64_t steps = PyLong_AsLongLong(a[1]);
  const double c[3] = {PyFloat_AsDouble(a[2]), PyFloat_AsDouble(a[3]), PyFloat_AsDouble(a[4])};
  const double eps = PyFloat_AsDouble(a[5]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&] {
    const at::NoGradGuard no_grad;
    at::Tensor x = u.detach();
    at::Tensor out = at::empty(x.sizes(), x.options());
    if (x.dim() == 2) x = x.unsqueeze(0);
    const int64_t batch = x.size(0), rows = x.size(1), cols = x.size(2);
    if ((cols > 1 && x.stride(2) != 1) || (rows > 1 && x.stride(1) < cols)) x = x.contiguous();
    const int64_t ld = rows > 1 && x.stride(1) > cols ? x.stride(1) : cols;
    const c10::DeviceGuard guard(x.device());
    const size_t need = smq_orthogonalize_workspace_bytes(code_of(x), batch, rows, cols);
    const at::Tensor ws = buffer(x, need, "orthogonalize");
    ok(smq_orthogonalize(x.const_data_ptr(), ld, x.stride(0), code_of(x), out.mutable_data_ptr(), batch,
                         rows, cols, steps < 1 || steps > 64 ? 0 : (int)steps, c, eps, ws.data_ptr(), need,
                         stream_of(x)),
       "orthogonalize");
    return out;
  });
}

#define SMQ_METHOD(name, doc) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, doc}
PyMethodDef kMethods[] = {
    SMQ_METHOD(group_norm, "group norm + activation with its autograd node (smq_group_norm_act)"),
    SMQ_METHOD(linear_ce, "linear cross entropy with its autograd node (smq_linear_ce_forward)"),
    SMQ_METHOD(orthogonalize, "Newton-Schulz orthogonalisation (smq_orthogonalize)"),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_smqtrain", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__smqtrain(void) { return PyModule_Create(&kModule); }
