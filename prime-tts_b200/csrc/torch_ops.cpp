// torch_ops.cpp -- the operators' entry points on torch tensors (the module _pt_b200_torch, which
// pt_b200.Operators calls): argument checks, output allocation and marshalling into the C ABI.
//
// It is native because small calls are bound by it: a single token's layer norm spends 2 us on the
// device, and the same checks and allocations made from Python took 12 us a call (this takes 5).
// Nothing is computed here.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>
#include <string>

#include "pt_b200.h"

namespace {

PyObject *g_error = nullptr;   // pt_b200.PtB200Error

// A refused argument, or a call that the library refused; becomes a PtB200Error.
struct Refused {
  std::string what;
};
template <class... A>
[[noreturn]] void refuse(const A &...a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused{s.str()};
}
void check(int rc, const char *what) {
  if (rc == 0) return;
  const char *m = pt_b200_last_error();
  refuse(what, " failed: ", m ? m : "");
}

std::string type_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    default: return c10::toString(t);
  }
}
std::string describe(const at::Tensor &t) {
  std::ostringstream s;
  s << "(";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << (t.dim() == 1 ? ",) " : ") ") << type_name(t.scalar_type()) << " on " << t.device().str();
  return s.str();
}

const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) refuse(name, ": needs a tensor");
  return THPVariable_Unpack(o);
}

// What the tensors of a call share.
struct Call {
  pt_b200_ops *h;
  int device, code, bytes;
  at::ScalarType type;
  Call(PyObject *handle, PyObject *dev, const at::Tensor &t, const char *name) {
    h = static_cast<pt_b200_ops *>(PyLong_AsVoidPtr(handle));
    device = static_cast<int>(PyLong_AsLong(dev));
    if (!h) refuse(name, ": the operators have been closed");
    type = t.scalar_type();
    code = type == at::kFloat ? PT_B200_F32 : type == at::kBFloat16 ? PT_B200_BF16 : type == at::kHalf ? PT_B200_F16 : -1;
    bytes = code == PT_B200_F32 ? 4 : 2;
    if (code < 0 || !here(t))
      refuse(name, ": needs a float32, bfloat16 or float16 tensor on cuda:", device, ", got ", type_name(type), " on ",
             t.device().str());
  }
  bool here(const at::Tensor &t) const { return t.is_cuda() && t.get_device() == device; }
  cudaStream_t stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

  // Tensors whose values are not what lies in memory: torch keeps a pending minus sign (x.conj().imag), or
  // no memory at all for zeros.
  static void in_memory(const at::Tensor &t, const char *name) {
    if (t.is_neg()) refuse(name, ": is a negated view, whose sign is not in memory (resolve_neg() puts it there)");
    if (t._is_zerotensor()) refuse(name, ": is a tensor of zeros without memory (clone() gives it some)");
  }

  // A [..., cols] tensor seen as [rows][cols] with one stride for its rows.
  const void *rows(const at::Tensor &t, const char *name, int64_t n, int64_t cols, int64_t *ld) const {
    if (t.scalar_type() != type || !here(t) || t.dim() == 0 || t.size(-1) != cols || t.numel() != n * cols)
      refuse(name, ": needs ", n, " rows of ", cols, " ", type_name(type), " on cuda:", device, ", got ", describe(t));
    in_memory(t, name);
    *ld = cols;
    if (t.is_contiguous()) return t.const_data_ptr();
    int64_t stride = 0, step = 0;
    if (t.dim() == 2) {
      stride = t.stride(0);
      step = t.stride(1);
    } else {
      try {
        const at::Tensor v = t.view({n, cols});
        stride = v.stride(0);
        step = v.stride(1);
      } catch (const c10::Error &) {
        refuse(name, ": its leading dimensions have no common row stride");
      }
    }
    if (step != 1 && cols > 1) refuse(name, ": its columns are not contiguous (stride ", step, ")");
    if (n > 1 && stride < cols) refuse(name, ": its rows overlap (stride ", stride, " for ", cols, " columns)");
    if (n > 1) *ld = stride;
    return t.const_data_ptr();
  }
  // A contiguous tensor of n elements; None gives NULL.
  const void *vector(PyObject *o, const char *name, at::ScalarType want, int64_t n) const {
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != want || !here(t) || t.numel() != n || !t.is_contiguous())
      refuse(name, ": needs ", n, " contiguous ", type_name(want), " on cuda:", device, ", got ", describe(t));
    in_memory(t, name);
    return t.const_data_ptr();
  }
};

// New tensors on like's device, from the allocator itself: the dispatcher's way to it takes as long.
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}
// like's leading dimensions with `cols` columns.
at::Tensor empty_rows(const at::Tensor &like, int64_t cols) {
  at::DimVector shape(like.sizes().begin(), like.sizes().end());
  shape.back() = cols;
  return empty(shape, like.scalar_type(), like);
}
at::Tensor workspace(const at::Tensor &like, int64_t bytes) { return empty({bytes}, at::kByte, like); }

PyObject *wrap(at::Tensor t) { return t.defined() ? THPVariable_Wrap(std::move(t)) : Py_NewRef(Py_None); }
PyObject *tuple3(at::Tensor a, at::Tensor b, at::Tensor c) {
  return Py_BuildValue("(NNN)", wrap(std::move(a)), wrap(std::move(b)), wrap(std::move(c)));
}

template <class F>
int without_gil(F &&fn) {
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = fn();
  Py_END_ALLOW_THREADS return rc;
}

// linear(handle, device, x, w, bias, residual, act, slope, save_pre) -> y or (y, pre)
PyObject *linear(PyObject *const *o) {
  const at::Tensor &x = tensor(o[2], "x"), &w = tensor(o[3], "w");
  const Call c(o[0], o[1], x, "x");
  if (w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(1))
    refuse("linear: x ", describe(x), " and w ", describe(w), " do not fit");
  pt_b200_linear_args a{};
  a.dtype = c.code;
  a.act = static_cast<int32_t>(PyLong_AsLong(o[6]));
  a.out = w.size(0);
  a.in = w.size(1);
  if (a.in == 0 || a.out == 0) refuse("linear: w ", describe(w), " is empty");
  a.rows = x.numel() / a.in;
  a.x = c.rows(x, "x", a.rows, a.in, &a.ldx);
  a.w = c.rows(w, "w", a.out, a.in, &a.ldw);
  a.bias = c.vector(o[4], "bias", c.type, a.out);
  if (o[5] != Py_None) a.residual = c.rows(tensor(o[5], "residual"), "residual", a.rows, a.out, &a.ldr);
  a.slope = static_cast<float>(PyFloat_AsDouble(o[7]));
  const int save = PyObject_IsTrue(o[8]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor y = empty_rows(x, a.out), pre, work;
  a.y = y.mutable_data_ptr();
  a.ldy = a.ldp = a.out;
  if (save) {
    pre = empty_rows(x, a.out);
    a.pre = pre.mutable_data_ptr();
  }
  a.work_bytes = pt_b200_linear_work(c.h, &a);
  if (a.work_bytes) {
    work = workspace(x, a.work_bytes);
    a.work = work.mutable_data_ptr();
  }
  check(without_gil([&] { return pt_b200_linear(c.h, c.stream(), &a); }), "pt_b200_linear");
  return save ? Py_BuildValue("(NN)", wrap(std::move(y)), wrap(std::move(pre))) : wrap(std::move(y));
}

// linear_backward(handle, device, dy, x, w, pre, act, slope, need_dx, need_dw, need_db) -> (dx, dw, db)
PyObject *linear_backward(PyObject *const *o) {
  const at::Tensor &dy = tensor(o[2], "dy"), &x = tensor(o[3], "x"), &w = tensor(o[4], "w");
  const Call c(o[0], o[1], dy, "dy");
  if (w.dim() != 2 || dy.dim() < 1 || dy.size(-1) != w.size(0))
    refuse("linear_backward: dy ", describe(dy), " and w ", describe(w), " do not fit");
  pt_b200_linear_grad_args a{};
  a.dtype = c.code;
  a.act = static_cast<int32_t>(PyLong_AsLong(o[6]));
  a.slope = static_cast<float>(PyFloat_AsDouble(o[7]));
  const int need_dx = PyObject_IsTrue(o[8]), need_dw = PyObject_IsTrue(o[9]), need_db = PyObject_IsTrue(o[10]);
  if (PyErr_Occurred()) return nullptr;
  a.out = w.size(0);
  a.in = w.size(1);
  if (a.in == 0 || a.out == 0) refuse("linear_backward: w ", describe(w), " is empty");
  if (!need_dx && !need_dw && !need_db) refuse("linear_backward: nothing to compute");
  if (a.act != PT_B200_ACT_NONE && o[5] == Py_None) refuse("linear_backward: an activation needs pre");
  a.rows = dy.numel() / a.out;
  a.dy = c.rows(dy, "dy", a.rows, a.out, &a.lddy);
  a.x = c.rows(x, "x", a.rows, a.in, &a.ldx);
  a.w = c.rows(w, "w", a.out, a.in, &a.ldw);
  if (a.act != PT_B200_ACT_NONE) a.pre = c.rows(tensor(o[5], "pre"), "pre", a.rows, a.out, &a.ldp);
  at::Tensor dx, dw, db, work;
  if (need_dx) {
    dx = empty_rows(dy, a.in);
    a.dx = dx.mutable_data_ptr();
  }
  if (need_dw) {
    dw = empty({a.out, a.in}, c.type, dy);
    a.dw = dw.mutable_data_ptr();
  }
  if (need_db) {
    db = empty({a.out}, c.type, dy);
    a.db = db.mutable_data_ptr();
  }
  a.lddx = a.lddw = a.in;
  // (a tensor without elements has no address, and an output without rows nothing to write)
  if (a.rows == 0 && !need_dw && !need_db) return tuple3(std::move(dx), std::move(dw), std::move(db));
  a.work_bytes = pt_b200_linear_backward_work(c.h, &a);
  if (a.work_bytes) {
    work = workspace(dy, a.work_bytes);
    a.work = work.mutable_data_ptr();
  }
  check(without_gil([&] { return pt_b200_linear_backward(c.h, c.stream(), &a); }), "pt_b200_linear_backward");
  return tuple3(std::move(dx), std::move(dw), std::move(db));
}

// layer_norm(handle, device, x, gamma, beta, eps) -> (y, mean, rstd)
PyObject *layer_norm(PyObject *const *o) {
  const at::Tensor &x = tensor(o[2], "x");
  const Call c(o[0], o[1], x, "x");
  pt_b200_norm_args a{};
  a.dtype = c.code;
  a.eps = static_cast<float>(PyFloat_AsDouble(o[5]));
  if (PyErr_Occurred()) return nullptr;
  a.cols = x.dim() ? x.size(-1) : 0;
  if (a.cols == 0) refuse("layer_norm: x ", describe(x), " has no columns");
  a.rows = x.numel() / a.cols;
  a.x = c.rows(x, "x", a.rows, a.cols, &a.ldx);
  a.gamma = c.vector(o[3], "gamma", c.type, a.cols);
  a.beta = c.vector(o[4], "beta", c.type, a.cols);
  at::Tensor y = empty(x.sizes(), c.type, x);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  at::Tensor mean = empty(lead, at::kFloat, x), rstd = empty(lead, at::kFloat, x);
  a.y = y.mutable_data_ptr();
  a.ldy = a.cols;
  a.mean = mean.mutable_data_ptr<float>();
  a.rstd = rstd.mutable_data_ptr<float>();
  check(without_gil([&] { return pt_b200_layer_norm(c.h, c.stream(), &a); }), "pt_b200_layer_norm");
  return tuple3(std::move(y), std::move(mean), std::move(rstd));
}

// layer_norm_backward(handle, device, dy, x, gamma, mean, rstd, need_dx, need_dgamma, need_dbeta)
PyObject *layer_norm_backward(PyObject *const *o) {
  const at::Tensor &dy = tensor(o[2], "dy"), &x = tensor(o[3], "x");
  const Call c(o[0], o[1], dy, "dy");
  pt_b200_norm_grad_args a{};
  a.dtype = c.code;
  a.cols = dy.dim() ? dy.size(-1) : 0;
  if (a.cols == 0) refuse("layer_norm_backward: dy ", describe(dy), " has no columns");
  const int need_dx = PyObject_IsTrue(o[7]), need_dg = PyObject_IsTrue(o[8]), need_db = PyObject_IsTrue(o[9]);
  if (PyErr_Occurred()) return nullptr;
  if (!need_dx && !need_dg && !need_db) refuse("layer_norm_backward: nothing to compute");
  a.rows = dy.numel() / a.cols;
  a.dy = c.rows(dy, "dy", a.rows, a.cols, &a.lddy);
  a.x = c.rows(x, "x", a.rows, a.cols, &a.ldx);
  a.gamma = c.vector(o[4], "gamma", c.type, a.cols);
  a.mean = static_cast<const float *>(c.vector(o[5], "mean", at::kFloat, a.rows));
  a.rstd = static_cast<const float *>(c.vector(o[6], "rstd", at::kFloat, a.rows));
  at::Tensor dx, dgamma, dbeta, work;
  if (need_dx) {
    dx = empty(dy.sizes(), c.type, dy);
    a.dx = dx.mutable_data_ptr();
    a.lddx = a.cols;
  }
  if (need_dg) {
    dgamma = empty({a.cols}, c.type, dy);
    a.dgamma = dgamma.mutable_data_ptr();
  }
  if (need_db) {
    dbeta = empty({a.cols}, c.type, dy);
    a.dbeta = dbeta.mutable_data_ptr();
  }
  if (need_dg || need_db) a.work_bytes = pt_b200_layer_norm_backward_work(c.h, a.rows, a.cols);
  if (a.work_bytes) {
    work = workspace(dy, a.work_bytes);
    a.work = work.mutable_data_ptr();
  }
  check(without_gil([&] { return pt_b200_layer_norm_backward(c.h, c.stream(), &a); }), "pt_b200_layer_norm_backward");
  return tuple3(std::move(dx), std::move(dgamma), std::move(dbeta));
}

template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments are needed, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused &r) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, r.what.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject *set_error_class(PyObject *, PyObject *cls) {
  Py_XSETREF(g_error, Py_NewRef(cls));
  Py_RETURN_NONE;
}

#define PTB_ENTRY(fn, n) \
  {#fn, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&entry<fn, n>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {PTB_ENTRY(linear, 9),
                           PTB_ENTRY(linear_backward, 11),
                           PTB_ENTRY(layer_norm, 6),
                           PTB_ENTRY(layer_norm_backward, 10),
                           {"set_error_class", set_error_class, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_pt_b200_torch", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__pt_b200_torch(void) { return PyModule_Create(&g_module); }
