// mi_operator_call.cpp -- the ordinary calls of the operators that take
// argument structures (layer_norm, matmul_epilogue, newton_schulz and the
// gradients), from torch tensors to the C ABI launch, in native code.
//
// Each function does what the Python body of its operator does for plain
// contiguous tensors on one device, in 4 to 6 us of host time instead of 15
// to 25, and returns None for everything else: another type, layout, device,
// shape or mode, an argument that is to be refused, or a library that
// bind_operators() was not told of.  The Python body then runs, checks
// everything and raises what is to be raised.  Nothing is kept between calls
// but the entry points.
#include <c10/core/GradMode.h>

#include <climits>
#include <cstdlib>
#include <initializer_list>
#include <string>
#include <vector>

#include "../../../include/mi_kernels.h"
#include "mi_torch_plain.hpp"

extern PyMethodDef kOperatorMethods[];

// The same words as the Python bodies' (_operands.warn_detached).
#define MI_DETACHED                                                                                          \
  "%s records nothing for autograd, and an operand requires a gradient: it will not reach it through this " \
  "result. Call %s under torch.no_grad() and take the gradients from the operator's own call."

namespace {

using mi_torch::disjoint;
using mi_torch::no_mode;
using mi_torch::plain;

struct Operators {
  decltype(&mi_layer_norm) layer_norm = nullptr;
  decltype(&mi_layer_norm_backward_workspace) layer_norm_backward_workspace = nullptr;
  decltype(&mi_layer_norm_backward) layer_norm_backward = nullptr;
  decltype(&mi_matmul_epilogue_workspace) matmul_epilogue_workspace = nullptr;
  decltype(&mi_matmul_epilogue_bf16) matmul_epilogue = nullptr;
  decltype(&mi_matmul_epilogue_backward_workspace) matmul_epilogue_backward_workspace = nullptr;
  decltype(&mi_matmul_epilogue_backward_bf16) matmul_epilogue_backward = nullptr;
  decltype(&mi_newton_schulz_workspace) newton_schulz_workspace = nullptr;
  decltype(&mi_newton_schulz) newton_schulz = nullptr;
  std::string env;               // MI_KERNELS_LIB when the library was bound ("" if unset)
  PyObject* check_rc = nullptr;  // raises the error of a return code
} g_ops;

// The bound library is the one in use, and nothing intercepts calls.
bool ready() {
  if (!g_ops.check_rc || !no_mode()) return false;
  const char* env = std::getenv("MI_KERNELS_LIB");
  return g_ops.env == (env ? env : "");
}

// An argument that may be None: a plain tensor of `device` or nothing; false
// for anything else.
bool optional(PyObject* o, const c10::Device& device, const at::Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return true;
  *t = plain(o);
  return *t && (*t)->device() == device;
}
bool number(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
at::Tensor like(const at::Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }
at::Tensor make(const at::Tensor& on, at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::empty(sizes, on.options().dtype(dtype).requires_grad(false));
}

// Raises the error of a return code.
PyObject* raise(int rc, const char* what) {
  PyObject* r = PyObject_CallFunction(g_ops.check_rc, "is", rc, what);
  if (r) {  // check_rc raises for every code but 0
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, what);
  }
  return nullptr;
}

// Warns where autograd records and an operand requires a gradient: the result
// will not.  False where the warning is an error.
bool warn_detached(const char* what, std::initializer_list<const at::Tensor*> operands) {
  if (!c10::GradMode::is_enabled()) return true;
  for (const at::Tensor* t : operands)
    if (t && t->requires_grad()) return PyErr_WarnFormat(PyExc_UserWarning, 2, MI_DETACHED, what, what) == 0;
  return true;
}

// fn(stream) without the GIL; fn reads nothing shared.
template <class F>
int launch(const c10::Device& dev, F&& fn) {
  void* stream = (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(stream);
  Py_END_ALLOW_THREADS
  return rc;
}
// The same with the workspace that query(&bytes) asks for.
template <class Q, class F>
int launch_with(const at::Tensor& on, Q&& query, F&& fn) {
  unsigned long long bytes = 0;
  const int rc = query(&bytes);
  if (rc != 0) return rc;
  at::Tensor ws;
  if (bytes) ws = make(on, {(int64_t)bytes}, at::kByte);
  void* p = bytes ? ws.data_ptr() : nullptr;
  return launch(on.device(), [&](void* stream) { return fn(p, bytes, stream); });
}

PyObject* wrap_or_none(at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(std::move(t));
  Py_RETURN_NONE;
}
PyObject* three(at::Tensor& a, at::Tensor& b, at::Tensor& c) {
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  at::Tensor* t[] = {&a, &b, &c};
  for (int i = 0; i < 3; ++i) {
    PyObject* o = wrap_or_none(*t[i]);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, o);
  }
  return r;
}

#define MI_TAKES(N)                                              \
  if (n != N) {                                                  \
    PyErr_SetString(PyExc_TypeError, "takes " #N " arguments");  \
    return nullptr;                                              \
  }
#define MI_OR_PYTHON(COND) \
  if (!(COND)) Py_RETURN_NONE

int norm_dtype(const at::Tensor& x) {
  switch (x.scalar_type()) {
    case at::kBFloat16: return MI_DTYPE_BF16;
    case at::kHalf: return MI_DTYPE_F16;
    case at::kFloat: return MI_DTYPE_F32;
    default: return -1;
  }
}
// weight and bias of rows of D: both x's type or both fp32.
bool params(const at::Tensor& x, int64_t D, const at::Tensor* w, const at::Tensor* b, int* f32) {
  *f32 = 0;
  for (const at::Tensor* t : {w, b}) {
    if (!t) continue;
    if (t->dim() != 1 || t->size(0) != D) return false;
    if (t->scalar_type() != x.scalar_type() && t->scalar_type() != at::kFloat) return false;
    if (t->scalar_type() == at::kFloat) *f32 = 1;
  }
  return !w || !b || w->scalar_type() == b->scalar_type();
}

// layer_norm(x, weight | None, bias | None, eps, out | None, stats)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  MI_TAKES(6)
  HANDLE_TH_ERRORS
  {
    MI_OR_PYTHON(ready());
    const at::Tensor *x = plain(args[0]), *w, *b, *given;
    MI_OR_PYTHON(x && x->dim() >= 1 && x->numel() > 0);
    const c10::Device dev = x->device();
    const int dtype = norm_dtype(*x);
    const int64_t D = x->size(-1), rows = x->numel() / D;
    int f32;
    double eps;
    MI_OR_PYTHON(dtype >= 0 && D <= INT_MAX && optional(args[1], dev, &w) && optional(args[2], dev, &b) &&
                 optional(args[4], dev, &given) && params(*x, D, w, b, &f32) && number(args[3], &eps) && eps >= 0.0 &&
                 eps < 3e38);
    if (given)
      MI_OR_PYTHON(given->scalar_type() == x->scalar_type() && given->sizes() == x->sizes() && disjoint(*given, *x) &&
                   (!w || disjoint(*given, *w)) && (!b || disjoint(*given, *b)));
    const int stats = PyObject_IsTrue(args[5]);
    if (stats < 0 || !warn_detached("layer_norm", {x, w, b})) return nullptr;
    const c10::OptionalDeviceGuard guard(dev);
    at::Tensor out = given ? *given : like(*x), mean, rstd;
    if (stats) {
      mean = make(*x, x->sizes().slice(0, x->dim() - 1), at::kFloat);
      rstd = make(*x, x->sizes().slice(0, x->dim() - 1), at::kFloat);
    }
    const mi_layer_norm_args a = {x->data_ptr(), ptr(w), ptr(b), out.data_ptr(), stats ? mean.data_ptr<float>() : nullptr,
                                  stats ? rstd.data_ptr<float>() : nullptr, rows, D, (int)D, dtype, f32, (float)eps};
    const auto fn = g_ops.layer_norm;
    const int rc = launch(dev, [&](void* s) { return fn(&a, s); });
    if (rc != 0) return raise(rc, "layer_norm");
    if (stats) return three(out, mean, rstd);
    return THPVariable_Wrap(std::move(out));
  }
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(dout, x, mean, rstd, weight | None, bias | None, need_dx)
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  MI_TAKES(7)
  HANDLE_TH_ERRORS
  {
    MI_OR_PYTHON(ready());
    const at::Tensor *dout = plain(args[0]), *x = plain(args[1]), *mean = plain(args[2], at::kFloat),
                     *rstd = plain(args[3], at::kFloat), *w, *b;
    MI_OR_PYTHON(dout && x && mean && rstd && x->dim() >= 1 && x->numel() > 0);
    const c10::Device dev = x->device();
    const int dtype = norm_dtype(*x);
    const int64_t D = x->size(-1), rows = x->numel() / D;
    const auto lead = x->sizes().slice(0, x->dim() - 1);
    int f32;
    MI_OR_PYTHON(dtype >= 0 && D <= INT_MAX && dout->scalar_type() == x->scalar_type() && dout->sizes() == x->sizes() &&
                 dout->device() == dev && mean->device() == dev && rstd->device() == dev && mean->sizes() == lead &&
                 rstd->sizes() == lead && optional(args[4], dev, &w) && optional(args[5], dev, &b) &&
                 params(*x, D, w, b, &f32));
    const int need_dx = PyObject_IsTrue(args[6]);
    if (need_dx < 0) return nullptr;
    const c10::OptionalDeviceGuard guard(dev);
    at::Tensor dx, dw, db;
    if (need_dx) dx = like(*x);
    if (w) dw = like(*w);
    if (b) db = like(*b);
    const mi_layer_norm_grad_args a = {dout->data_ptr(), x->data_ptr(), ptr(w), mean->data_ptr<float>(),
                                       rstd->data_ptr<float>(), need_dx ? dx.data_ptr() : nullptr,
                                       w ? dw.data_ptr() : nullptr, b ? db.data_ptr() : nullptr, rows, D, D, (int)D, dtype,
                                       f32};
    const auto query = g_ops.layer_norm_backward_workspace;
    const auto fn = g_ops.layer_norm_backward;
    const int rc = launch_with(*x, [&](unsigned long long* need) { return query(&a, need); },
                               [&](void* ws, unsigned long long bytes, void* s) { return fn(&a, ws, bytes, s); });
    if (rc != 0) return raise(rc, "layer_norm_backward");
    return three(dx, dw, db);
  }
  END_HANDLE_TH_ERRORS
}

bool matrix(const at::Tensor* t, int64_t M, int64_t N) {
  return t->scalar_type() == at::kBFloat16 && t->dim() == 2 && t->size(0) == M && t->size(1) == N;
}
// The product's sizes and its bias; false where the Python body has to look.
struct Sizes {
  int64_t M, N, K;
  int transposed, act, f32;
};
bool product(const at::Tensor* lhs, const at::Tensor* rhs, PyObject* transposed, PyObject* act, const at::Tensor* bias,
             Sizes* s) {
  if (!lhs || !rhs || lhs->dim() != 2 || rhs->dim() != 2 || rhs->device() != lhs->device()) return false;
  s->transposed = PyObject_IsTrue(transposed);
  if (s->transposed < 0) {
    PyErr_Clear();
    return false;
  }
  s->M = lhs->size(0);
  s->K = lhs->size(1);
  s->N = rhs->size(s->transposed ? 0 : 1);
  if (rhs->size(s->transposed ? 1 : 0) != s->K || s->M < 1 || s->N < 1 || s->K < 1 || s->M > INT_MAX || s->N > INT_MAX ||
      s->K > INT_MAX)
    return false;
  if (!PyLong_Check(act)) return false;
  s->act = (int)PyLong_AsLong(act);
  s->f32 = bias && bias->scalar_type() == at::kFloat;
  return !bias || (bias->dim() == 1 && bias->size(0) == s->N && (s->f32 || bias->scalar_type() == at::kBFloat16));
}

// matmul_epilogue(lhs, rhs, bias | None, activation, residual | None, rhs_transposed, pre | None, out | None)
PyObject* matmul_epilogue(PyObject*, PyObject* const* args, Py_ssize_t n) {
  MI_TAKES(8)
  HANDLE_TH_ERRORS
  {
    MI_OR_PYTHON(ready());
    const at::Tensor *lhs = plain(args[0], at::kBFloat16), *rhs = plain(args[1], at::kBFloat16), *bias, *res, *pre, *given;
    MI_OR_PYTHON(lhs && rhs);
    const c10::Device dev = lhs->device();
    Sizes z;
    MI_OR_PYTHON(optional(args[2], dev, &bias) && optional(args[4], dev, &res) && optional(args[6], dev, &pre) &&
                 optional(args[7], dev, &given) && product(lhs, rhs, args[5], args[3], bias, &z) &&
                 (!res || matrix(res, z.M, z.N)));
    for (const at::Tensor* o : {pre, given}) {
      if (!o) continue;
      MI_OR_PYTHON(matrix(o, z.M, z.N));
      for (const at::Tensor* i : {lhs, rhs, bias, res}) MI_OR_PYTHON(!i || disjoint(*o, *i));
    }
    MI_OR_PYTHON(!pre || !given || disjoint(*pre, *given));
    if (!warn_detached("matmul_epilogue", {lhs, rhs, bias, res})) return nullptr;
    const c10::OptionalDeviceGuard guard(dev);
    at::Tensor out = given ? *given : make(*lhs, {z.M, z.N}, at::kBFloat16);
    const mi_epilogue_args a = {lhs->data_ptr(), rhs->data_ptr(), ptr(bias), ptr(res), out.data_ptr(), ptr(pre), (int)z.M,
                                (int)z.N, (int)z.K, z.transposed, z.act, z.f32};
    const auto query = g_ops.matmul_epilogue_workspace;
    const auto fn = g_ops.matmul_epilogue;
    const int rc = launch_with(*lhs, [&](unsigned long long* need) { return query(&a, nullptr, need); },
                               [&](void* ws, unsigned long long bytes, void* s) { return fn(&a, nullptr, ws, bytes, s); });
    if (rc != 0) return raise(rc, "matmul_epilogue");
    return THPVariable_Wrap(std::move(out));
  }
  END_HANDLE_TH_ERRORS
}

// matmul_epilogue_backward(dout, lhs, rhs, activation, pre | None, bias | None, rhs_transposed, need_dlhs, need_drhs)
PyObject* matmul_epilogue_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  MI_TAKES(9)
  HANDLE_TH_ERRORS
  {
    MI_OR_PYTHON(ready());
    const at::Tensor *dout = plain(args[0]), *lhs = plain(args[1], at::kBFloat16), *rhs = plain(args[2], at::kBFloat16),
                     *pre, *bias;
    MI_OR_PYTHON(dout && lhs && rhs && dout->device() == lhs->device());
    const c10::Device dev = lhs->device();
    Sizes z;
    MI_OR_PYTHON(optional(args[4], dev, &pre) && optional(args[5], dev, &bias) &&
                 product(lhs, rhs, args[6], args[3], bias, &z) && matrix(dout, z.M, z.N));
    if (z.act == MI_ACT_NONE) pre = nullptr;
    else MI_OR_PYTHON(pre && matrix(pre, z.M, z.N));
    const int need_l = PyObject_IsTrue(args[7]), need_r = PyObject_IsTrue(args[8]);
    if (need_l < 0 || need_r < 0) return nullptr;
    const c10::OptionalDeviceGuard guard(dev);
    at::Tensor dl, dr, db;
    if (need_l) dl = like(*lhs);
    if (need_r) dr = like(*rhs);
    if (bias) db = like(*bias);
    const mi_epilogue_grad_args a = {dout->data_ptr(), lhs->data_ptr(), rhs->data_ptr(), ptr(pre),
                                     need_l ? dl.data_ptr() : nullptr, need_r ? dr.data_ptr() : nullptr,
                                     bias ? db.data_ptr() : nullptr, (int)z.M, (int)z.N, (int)z.K, z.transposed, z.act, z.f32};
    const auto query = g_ops.matmul_epilogue_backward_workspace;
    const auto fn = g_ops.matmul_epilogue_backward;
    const int rc = launch_with(*lhs, [&](unsigned long long* need) { return query(&a, need); },
                               [&](void* ws, unsigned long long bytes, void* s) { return fn(&a, ws, bytes, s); });
    if (rc != 0) return raise(rc, "matmul_epilogue_backward");
    return three(dl, dr, db);
  }
  END_HANDLE_TH_ERRORS
}

// newton_schulz(grad, steps, a, b, c, eps, out | None)
PyObject* newton_schulz(PyObject*, PyObject* const* args, Py_ssize_t n) {
  MI_TAKES(7)
  HANDLE_TH_ERRORS
  {
    MI_OR_PYTHON(ready());
    const at::Tensor *g = plain(args[0]), *given;
    MI_OR_PYTHON(g && (g->dim() == 2 || g->dim() == 3) && g->numel() > 0);
    const int dtype = norm_dtype(*g);
    double v[4];
    MI_OR_PYTHON((dtype == MI_DTYPE_BF16 || dtype == MI_DTYPE_F32) && optional(args[6], g->device(), &given) &&
                 PyLong_Check(args[1]));
    for (int i = 0; i < 4; ++i) MI_OR_PYTHON(number(args[2 + i], &v[i]));
    const long steps = PyLong_AsLong(args[1]);
    if (steps == -1 && PyErr_Occurred()) PyErr_Clear();
    const int64_t batch = g->dim() == 3 ? g->size(0) : 1, m = g->size(-2), k = g->size(-1);
    MI_OR_PYTHON(steps >= 0 && steps <= INT_MAX && v[3] >= 0.0 && v[3] < 3e38 && batch <= INT_MAX && m <= INT_MAX &&
                 k <= INT_MAX);
    if (given)
      MI_OR_PYTHON(given->scalar_type() == at::kBFloat16 && given->sizes() == g->sizes() && disjoint(*given, *g));
    if (!warn_detached("newton_schulz", {g})) return nullptr;
    const c10::OptionalDeviceGuard guard(g->device());
    at::Tensor out = given ? *given : make(*g, g->sizes(), at::kBFloat16);
    const mi_newton_schulz_args a = {g->data_ptr(), out.data_ptr(), (int)batch, (int)m, (int)k, (int)steps, dtype,
                                     (float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    const auto query = g_ops.newton_schulz_workspace;
    const auto fn = g_ops.newton_schulz;
    const int rc = launch_with(*g, [&](unsigned long long* need) { return query(&a, need); },
                               [&](void* ws, unsigned long long bytes, void* s) { return fn(&a, ws, bytes, s); });
    if (rc != 0) return raise(rc, "newton_schulz");
    return THPVariable_Wrap(std::move(out));
  }
  END_HANDLE_TH_ERRORS
}

// bind_operators(env, the entry points' addresses in the order of Operators, check_rc): the library that the calls
// go to, and the value of MI_KERNELS_LIB it was found with.
PyObject* bind_operators(PyObject*, PyObject* args) {
  const char* env;
  unsigned long long p[9];
  PyObject* check_rc;
  if (!PyArg_ParseTuple(args, "sKKKKKKKKKO", &env, p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7, p + 8, &check_rc))
    return nullptr;
  const auto to = [&](auto& f, int i) { f = (std::remove_reference_t<decltype(f)>)(uintptr_t)p[i]; };
  to(g_ops.layer_norm, 0);
  to(g_ops.layer_norm_backward_workspace, 1);
  to(g_ops.layer_norm_backward, 2);
  to(g_ops.matmul_epilogue_workspace, 3);
  to(g_ops.matmul_epilogue, 4);
  to(g_ops.matmul_epilogue_backward_workspace, 5);
  to(g_ops.matmul_epilogue_backward, 6);
  to(g_ops.newton_schulz_workspace, 7);
  to(g_ops.newton_schulz, 8);
  g_ops.env = env;
  Py_INCREF(check_rc);
  PyObject* const before = g_ops.check_rc;
  g_ops.check_rc = check_rc;
  Py_XDECREF(before);
  Py_RETURN_NONE;
}

// knows_operators(): whether the library in use is bound.
PyObject* knows_operators(PyObject*, PyObject*) {
  const char* env = std::getenv("MI_KERNELS_LIB");
  return PyBool_FromLong(g_ops.check_rc && g_ops.env == (env ? env : ""));
}

#define MI_FAST(F) (PyCFunction)(void (*)(void))F, METH_FASTCALL, nullptr

}  // namespace

PyMethodDef kOperatorMethods[] = {{"layer_norm", MI_FAST(layer_norm)},
                                  {"layer_norm_backward", MI_FAST(layer_norm_backward)},
                                  {"matmul_epilogue", MI_FAST(matmul_epilogue)},
                                  {"matmul_epilogue_backward", MI_FAST(matmul_epilogue_backward)},
                                  {"newton_schulz", MI_FAST(newton_schulz)},
                                  {"bind_operators", bind_operators, METH_VARARGS, nullptr},
                                  {"knows_operators", knows_operators, METH_NOARGS, nullptr},
                                  {nullptr, nullptr, 0, nullptr}};
