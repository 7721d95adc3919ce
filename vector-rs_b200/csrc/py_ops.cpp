// py_ops.cpp -- the torch side of vector_cuda.ops as a Python extension: checks
// of arguments, outputs and workspaces, and the call into libvrs on the current
// stream. (The same steps in Python took 10 to 20 us a call, several times what
// the small operators take on the GPU.)
//
// It has no link to libvrs: bind() gets the entry points' addresses from the
// library that vector_cuda loaded, and the function that turns a status into a
// CudaError.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <optional>
#include <sstream>
#include <string>

#include "vrs.h"

namespace {

struct Bound {
  decltype(&vrs_layer_norm_forward) norm_forward;
  decltype(&vrs_layer_norm_backward) norm_backward;
  decltype(&vrs_layer_norm_backward_workspace) norm_workspace;
  decltype(&vrs_linear_cross_entropy_forward) loss_forward;
  decltype(&vrs_linear_cross_entropy_backward_with_loss) loss_backward;
  decltype(&vrs_linear_cross_entropy_workspace) loss_workspace;
  PyObject* check;  // raises CudaError for a status
} g{};

// Thrown for a wrong argument (ValueError), and after a Python error was set.
struct BadArgument {
  std::string what;
};
struct PythonError {};

template <class... A>
[[noreturn]] void bad(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw BadArgument{s.str()};
}

void check_status(int status) {
  if (status == VRS_OK) return;
  PyObject* r = PyObject_CallFunction(g.check, "i", status);
  if (r) {
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, "vector_cuda.ops: a failing status raised nothing");
  }
  throw PythonError{};
}

std::string name_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}

int code_of(at::ScalarType t) { return t == at::kFloat ? VRS_F32 : t == at::kHalf ? VRS_F16 : VRS_BF16; }

const at::Tensor& tensor_arg(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) bad(name, " must be a torch tensor");
  return THPVariable_Unpack(o);
}

std::optional<at::Tensor> optional_arg(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor_arg(o, name);
}

double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
  return v;
}

bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError{};
  return v != 0;
}

// A tensor as rows of its last dimension. Rows that are contiguous and evenly
// spaced are used where they are, others are copied.
struct Rows {
  at::Tensor t;
  int64_t n, d, stride;
};

Rows rows_of(const at::Tensor& in, const char* name, int64_t want = -1) {
  if (!in.is_cuda()) bad(name, " must be a CUDA tensor (there is no CPU fallback)");
  const auto type = in.scalar_type();
  if (in.dim() < 1 || (type != at::kFloat && type != at::kHalf && type != at::kBFloat16))
    bad(name, " must have rows of float32, float16 or bfloat16, got ", name_of(type));
  const int64_t d = in.size(-1);
  if (want >= 0 && d != want) bad(name, " has rows of ", d, " elements, expected ", want);
  if (d < 1) bad(name, " has rows of no elements");
  Rows r{in.dim() == 2 ? in : in.reshape({-1, d}), 0, d, 0};
  r.n = r.t.size(0);
  r.stride = r.t.stride(0);
  if ((d > 1 && r.t.stride(1) != 1) || (r.n > 1 && r.stride < d)) {
    r.t = r.t.contiguous();
    r.stride = d;
  }
  if (r.stride < d) r.stride = d;  // a single row
  return r;
}

// n values beside `like`, contiguous.
at::Tensor beside(const at::Tensor& t, const at::Tensor& like, const char* name, int64_t n, at::ScalarType type) {
  if (t.scalar_type() != type) bad(name, " must be ", name_of(type), ", got ", name_of(t.scalar_type()));
  if (t.numel() != n) bad(name, " holds ", t.numel(), " values, expected ", n);
  if (t.device() != like.device()) bad(name, " is on ", t.device().str(), ", expected ", like.device().str());
  return t.is_contiguous() ? t : t.contiguous();
}

void* ptr(const std::optional<at::Tensor>& t) { return t ? t->data_ptr() : nullptr; }

// The shape of x without its last dimension.
at::Tensor column_of(const at::Tensor& x, const at::Tensor& like) {
  return at::empty(x.sizes().slice(0, x.dim() - 1), like.options().dtype(at::kFloat));
}

PyObject* to_tuple(std::initializer_list<std::optional<at::Tensor>> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) throw PythonError{};
  Py_ssize_t i = 0;
  for (const auto& t : ts) {
    PyObject* o;
    if (t) {
      o = THPVariable_Wrap(*t);
    } else {
      o = Py_None;
      Py_INCREF(o);
    }
    if (!o) {
      Py_DECREF(r);
      throw PythonError{};
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

template <class F>
int unlocked(F f) {
  int status;
  Py_BEGIN_ALLOW_THREADS status = f();
  Py_END_ALLOW_THREADS return status;
}

// The parameters' type (the rows', or float32), checked.
at::ScalarType check_params(std::optional<at::Tensor>& weight, std::optional<at::Tensor>& bias, const Rows& x) {
  auto type = x.t.scalar_type();
  std::pair<const char*, std::optional<at::Tensor>*> both[] = {{"weight", &weight}, {"bias", &bias}};
  for (auto& [name, p] : both)
    if (*p) {
      const auto t = (*p)->scalar_type();
      if (t != x.t.scalar_type() && t != at::kFloat)
        bad(name, " must be ", name_of(x.t.scalar_type()), " or torch.float32, got ", name_of(t));
      type = t;
    }
  for (auto& [name, p] : both)
    if (*p) *p = beside(**p, x.t, name, x.d, type);
  return type;
}

// (x, weight, bias, eps) -> (y, mean, rstd)
PyObject* layer_norm_forward(PyObject* const* args) {
  const at::Tensor& x = tensor_arg(args[0], "x");
  const Rows r = rows_of(x, "x");
  auto weight = optional_arg(args[1], "weight"), bias = optional_arg(args[2], "bias");
  const float eps = (float)float_arg(args[3]);
  const auto pt = check_params(weight, bias, r);
  at::Tensor y = at::empty(x.sizes(), r.t.options());
  at::Tensor mean = column_of(x, r.t), rstd = column_of(x, r.t);
  const c10::cuda::CUDAGuard guard(r.t.device());
  void* stream = c10::cuda::getCurrentCUDAStream(r.t.get_device()).stream();
  check_status(unlocked([&] {
    return g.norm_forward(r.t.data_ptr(), r.stride, r.n, r.d, code_of(r.t.scalar_type()), ptr(weight), ptr(bias),
                          code_of(pt), eps, y.data_ptr(), r.d, (float*)mean.data_ptr(), (float*)rstd.data_ptr(), stream);
  }));
  return to_tuple({y, mean, rstd});
}

// (dy, x, weight, mean, rstd, params in 32 bits where there is no weight,
// want params) -> (dx, dweight, dbias)
PyObject* layer_norm_backward(PyObject* const* args) {
  const at::Tensor &dy = tensor_arg(args[0], "dy"), &x = tensor_arg(args[1], "x");
  const Rows r = rows_of(x, "x");
  if (dy.sizes() != x.sizes() || dy.scalar_type() != r.t.scalar_type() || dy.device() != r.t.device())
    bad("dy must be like x (", x.sizes(), ", ", name_of(r.t.scalar_type()), "), got ", dy.sizes(), ", ",
        name_of(dy.scalar_type()));
  const Rows q = rows_of(dy, "dy", r.d);
  auto weight = optional_arg(args[2], "weight");
  std::optional<at::Tensor> none;
  auto pt = check_params(weight, none, r);
  const at::Tensor mean = beside(tensor_arg(args[3], "mean"), r.t, "mean", r.n, at::kFloat);
  const at::Tensor rstd = beside(tensor_arg(args[4], "rstd"), r.t, "rstd", r.n, at::kFloat);
  if (!weight && bool_arg(args[5])) pt = at::kFloat;
  const bool params = bool_arg(args[6]);
  at::Tensor dx = at::empty(x.sizes(), r.t.options());
  const c10::cuda::CUDAGuard guard(r.t.device());
  std::optional<at::Tensor> dw, db, ws;
  int64_t need = 0;
  if (params) {
    check_status(g.norm_workspace(r.n, r.d, &need));
    dw = at::empty({r.d}, r.t.options().dtype(pt));
    db = at::empty({r.d}, r.t.options().dtype(pt));
    ws = at::empty({need}, r.t.options().dtype(at::kByte));
  }
  void* stream = c10::cuda::getCurrentCUDAStream(r.t.get_device()).stream();
  check_status(unlocked([&] {
    return g.norm_backward(q.t.data_ptr(), q.stride, r.t.data_ptr(), r.stride, r.n, r.d, code_of(r.t.scalar_type()),
                           ptr(weight), code_of(pt), (const float*)mean.data_ptr(), (const float*)rstd.data_ptr(),
                           dx.data_ptr(), r.d, ptr(dw), ptr(db), ptr(ws), need, stream);
  }));
  return to_tuple({dx, dw, db});
}

struct LossArgs {
  Rows x, table;
  at::Tensor targets;
  float scale;
  bool aligned;
};

LossArgs loss_args(PyObject* x_, PyObject* table_, PyObject* targets_, PyObject* scale_) {
  const at::Tensor &x = tensor_arg(x_, "x"), &table = tensor_arg(table_, "table"),
                   &targets = tensor_arg(targets_, "targets");
  LossArgs a;
  a.x = rows_of(x, "x");
  if (table.dim() != 2) bad("table must be classes x d, got ", table.sizes());
  a.table = rows_of(table, "table", a.x.d);
  const auto type = a.x.t.scalar_type();
  if (a.table.t.scalar_type() != type || a.table.t.device() != a.x.t.device())
    bad("table must be ", name_of(type), " on ", a.x.t.device().str(), ", got ", name_of(a.table.t.scalar_type()),
        " on ", a.table.t.device().str());
  if (type == at::kFloat) bad("x and table must be float16 or bfloat16 (operands of the tensor cores)");
  if (a.table.n < 1) bad("table has no rows");
  if (targets.sizes() != x.sizes().slice(0, x.dim() - 1))
    bad("targets have shape ", targets.sizes(), ", expected ", x.sizes().slice(0, x.dim() - 1));
  a.targets = beside(targets, a.x.t, "targets", a.x.n, at::kLong);
  const double scale = float_arg(scale_);
  a.scale = (float)scale;
  if (!(scale > 0.0) || !(a.scale > 0.0f) || !(a.scale < INFINITY)) bad("scale must be positive and finite, got ", scale);
  a.aligned = (uintptr_t)a.table.t.data_ptr() % 16 == 0 && a.table.stride % 8 == 0;
  return a;
}

at::Tensor loss_workspace(const LossArgs& a, bool backward, int64_t* need) {
  check_status(g.loss_workspace(a.x.n, a.table.n, a.x.d, code_of(a.x.t.scalar_type()), backward, a.aligned, need));
  return at::empty({*need}, a.x.t.options().dtype(at::kByte));
}

// (x, table, targets, scale) -> (loss, lse)
PyObject* linear_cross_entropy_forward(PyObject* const* args) {
  const LossArgs a = loss_args(args[0], args[1], args[2], args[3]);
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  at::Tensor loss = column_of(x, a.x.t), lse = column_of(x, a.x.t);
  const c10::cuda::CUDAGuard guard(a.x.t.device());
  int64_t need = 0;
  const at::Tensor ws = loss_workspace(a, false, &need);
  void* stream = c10::cuda::getCurrentCUDAStream(a.x.t.get_device()).stream();
  check_status(unlocked([&] {
    return g.loss_forward(a.x.t.data_ptr(), a.x.stride, a.x.n, a.table.t.data_ptr(), a.table.stride, a.table.n, a.x.d,
                          code_of(a.x.t.scalar_type()), (const int64_t*)a.targets.data_ptr(), a.scale,
                          (float*)loss.data_ptr(), (float*)lse.data_ptr(), ws.data_ptr(), need, stream);
  }));
  return to_tuple({loss, lse});
}

// (dloss, x, table, targets, lse, scale, need dx, need dtable, loss or None) -> (dx, dtable)
PyObject* linear_cross_entropy_backward(PyObject* const* args) {
  const LossArgs a = loss_args(args[1], args[2], args[3], args[5]);
  const at::Tensor &x = THPVariable_Unpack(args[1]), &table = THPVariable_Unpack(args[2]);
  const at::Tensor dloss = beside(tensor_arg(args[0], "dloss"), a.x.t, "dloss", a.x.n, at::kFloat);
  const at::Tensor lse = beside(tensor_arg(args[4], "lse"), a.x.t, "lse", a.x.n, at::kFloat);
  auto loss = optional_arg(args[8], "loss");
  if (loss) loss = beside(*loss, a.x.t, "loss", a.x.n, at::kFloat);
  std::optional<at::Tensor> dx, dtable;
  if (bool_arg(args[6])) dx = at::empty(x.sizes(), a.x.t.options());
  if (bool_arg(args[7])) dtable = at::empty(table.sizes(), a.table.t.options());
  const c10::cuda::CUDAGuard guard(a.x.t.device());
  int64_t need = 0;
  const at::Tensor ws = loss_workspace(a, true, &need);
  void* stream = c10::cuda::getCurrentCUDAStream(a.x.t.get_device()).stream();
  check_status(unlocked([&] {
    return g.loss_backward((const float*)dloss.data_ptr(), a.x.t.data_ptr(), a.x.stride, a.x.n, a.table.t.data_ptr(),
                           a.table.stride, a.table.n, a.x.d, code_of(a.x.t.scalar_type()),
                           (const int64_t*)a.targets.data_ptr(), a.scale, (const float*)lse.data_ptr(),
                           (const float*)ptr(loss), ptr(dx), a.x.d, ptr(dtable), a.x.d, ws.data_ptr(), need, stream);
  }));
  return to_tuple({dx, dtable});
}

// Every call: the argument count, no autograd inside, C++ errors as Python's.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  if (!g.check) {
    PyErr_SetString(PyExc_RuntimeError, "vector_cuda._ops is not bound to libvrs");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    return F(args);
  } catch (const BadArgument& e) {
    PyErr_SetString(PyExc_ValueError, e.what.c_str());
    return nullptr;
  } catch (const PythonError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the six entry points in the order of Bound, check)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes six addresses and a function");
    return nullptr;
  }
  void* at[6];
  for (int i = 0; i < 6; i++) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  g.norm_forward = (decltype(g.norm_forward))at[0];
  g.norm_backward = (decltype(g.norm_backward))at[1];
  g.norm_workspace = (decltype(g.norm_workspace))at[2];
  g.loss_forward = (decltype(g.loss_forward))at[3];
  g.loss_backward = (decltype(g.loss_backward))at[4];
  g.loss_workspace = (decltype(g.loss_workspace))at[5];
  Py_INCREF(args[6]);
  Py_XDECREF(g.check);
  g.check = args[6];
  Py_RETURN_NONE;
}

#define VRS_METHOD(name, count) \
  {#name, (PyCFunction)(void (*)())(&entry<name, count>), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
                         VRS_METHOD(layer_norm_forward, 4),
                         VRS_METHOD(layer_norm_backward, 7),
                         VRS_METHOD(linear_cross_entropy_forward, 4),
                         VRS_METHOD(linear_cross_entropy_backward, 9),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&module); }
