// torch_calls.cpp - the operators' calls on well-formed CUDA tensors, straight
// from Python to the C ABI.
//
// operators.py checks its arguments through some forty attribute reads, which
// take longer than the smallest kernels.  These functions make the same checks
// on the tensors themselves, allocate the result and launch; they return None,
// having launched nothing, for every call that is not plainly in order, and
// operators.py then finds out what is wrong with it, or handles it.  A launch
// that failed is reported at once (on_failure): it is not tried again, since a
// call may add to its own output.  There is no computation here.  The pointers,
// sizes and pitches that reach the library are
// the same either way.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "int8conv.h"

namespace {

// What a tensor argument turned out to be.
enum class Arg { kNone, kTensor, kOther };

Arg tensor(PyObject *o, at::Tensor &t) {
  if (o == Py_None) return Arg::kNone;
  if (!THPVariable_CheckExact(o)) return Arg::kOther;
  t = THPVariable_Unpack(o);
  return Arg::kTensor;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16:
      return INT8CONV_BF16;
    case at::kHalf:
      return INT8CONV_FP16;
    case at::kFloat:
      return INT8CONV_FP32;
    case at::kChar:
      return INT8CONV_INT8;
    case at::kInt:
      return INT8CONV_INT32;
    default:
      return -1;
  }
}

at::ScalarType scalar_type(long code) {
  static const at::ScalarType types[] = {at::kBFloat16, at::kHalf, at::kFloat, at::kChar, at::kInt};
  return types[code];
}

bool on(const at::Tensor &t, int device) { return t.is_cuda() && t.get_device() == device; }

// A contiguous vector of `count` entries, or nothing.
bool vector(PyObject *o, at::ScalarType type, int64_t count, int device, const void **p) {
  at::Tensor t;
  *p = nullptr;
  const Arg a = tensor(o, t);
  if (a == Arg::kNone) return true;
  if (a == Arg::kOther || t.scalar_type() != type || t.numel() != count || !t.is_contiguous() ||
      !on(t, device))
    return false;
  *p = t.data_ptr();
  return true;
}

struct Matrix {
  void *p = nullptr;
  int64_t rows = 0, cols = 0, pitch = 0;
};

bool matrix(const at::Tensor &t, int device, Matrix &m) {
  if (t.dim() != 2 || !on(t, device)) return false;
  m.rows = t.size(0);
  m.cols = t.size(1);
  if (t.stride(1) != 1 && m.cols > 1) return false;
  m.pitch = m.rows > 1 ? t.stride(0) : m.cols;   // one row has no pitch of its own
  if (m.pitch < m.cols) return false;
  m.p = t.data_ptr();
  return true;
}

bool int8_matrix(const at::Tensor &t, int device, Matrix &m) {
  if (t.scalar_type() != at::kChar || !matrix(t, device, m)) return false;
  if (m.rows <= 1) m.pitch = (m.pitch + 15) & -16;
  return (m.pitch & 15) == 0;
}

// int8 rows get a pitch that is a multiple of 16.
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int device) {
  const auto options = at::TensorOptions().dtype(type).device(at::kCUDA, device);
  const int64_t cols = shape.back();
  if (type != at::kChar || (cols & 15) == 0) return at::empty(shape, options);
  c10::SmallVector<int64_t, 6> wide(shape.begin(), shape.end());
  wide.back() = (cols + 15) & -16;
  return at::empty(wide, options).narrow(static_cast<int64_t>(shape.size()) - 1, 0, cols);
}

void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

PyObject *declined() { Py_RETURN_NONE; }

// operators.py's report of a status: raises.
PyObject *report = nullptr;

PyObject *on_failure(PyObject *, PyObject *callable) {
  Py_INCREF(callable);
  Py_XSETREF(report, callable);
  Py_RETURN_NONE;
}

// What a call returns whose launch had another status than OK: None for those
// that the library's checks of arguments give, before anything is launched.
PyObject *refused(int8conv_status st, const char *what) {
  if (st == INT8CONV_BAD_ARGUMENT || st == INT8CONV_BAD_POINTER || report == nullptr)
    return declined();
  PyObject *r = PyObject_CallFunction(report, "is", static_cast<int>(st), what);
  Py_XDECREF(r);
  if (r != nullptr) PyErr_Format(PyExc_RuntimeError, "%s: status %d", what, static_cast<int>(st));
  return nullptr;
}

// (a, b, offsets, y, row_scale, col_scale, bias, residual, activation, dtype, out_scale)
// -> y, or None.  offsets None: the plain product.  y None: a new result of type `dtype`.
PyObject *matmul(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  at::Tensor a, b, y, residual;
  if (count != 11 || tensor(args[0], a) != Arg::kTensor || tensor(args[1], b) != Arg::kTensor ||
      !a.is_cuda())
    return declined();
  const int device = c10::cuda::current_device();
  const bool grouped = args[2] != Py_None;
  int8conv_matmul d{};
  Matrix ma, mb, my, mr;
  if (!int8_matrix(a, device, ma)) return declined();
  int64_t groups = 1, group_stride = 0;
  if (grouped) {
    if (b.dim() != 3 || b.scalar_type() != at::kChar || !on(b, device)) return declined();
    groups = b.size(0);
    mb.rows = b.size(1);
    mb.cols = b.size(2);
    if (groups < 1 || groups > INT8CONV_MAX_GROUPS || (b.stride(2) != 1 && mb.cols > 1))
      return declined();
    mb.pitch = mb.rows > 1 ? b.stride(1) : (mb.cols + 15) & -16;
    if (mb.pitch < mb.cols || (mb.pitch & 15) != 0) return declined();
    if (groups > 1) {
      group_stride = b.stride(0);
      if ((group_stride & 15) != 0 || group_stride < (mb.rows - 1) * mb.pitch + mb.cols)
        return declined();
    }
    mb.p = b.data_ptr();
  } else if (!int8_matrix(b, device, mb)) {
    return declined();
  }
  if (ma.cols != mb.cols) return declined();
  const int64_t m = ma.rows, n = mb.rows;
  const void *offsets = nullptr, *row = nullptr, *col = nullptr, *bias = nullptr;
  if (!vector(args[2], at::kInt, groups + 1, device, &offsets) ||
      !vector(args[4], at::kFloat, m, device, &row) ||
      !vector(args[5], at::kFloat, n * groups, device, &col) ||
      !vector(args[6], at::kFloat, n * groups, device, &bias))
    return declined();
  const Arg res = tensor(args[7], residual);
  const long activation = PyLong_AsLong(args[8]);
  if (res == Arg::kOther) return declined();
  switch (tensor(args[3], y)) {
    case Arg::kOther:
      return declined();
    case Arg::kNone: {
      const long type = PyLong_AsLong(args[9]);
      if (type < 0 || type > INT8CONV_INT8) return declined();
      y = empty({m, n}, scalar_type(type), device);
      break;
    }
    default:
      break;
  }
  if (!matrix(y, device, my) || my.rows != m || my.cols != n) return declined();
  if (res == Arg::kTensor && (residual.scalar_type() != y.scalar_type() ||
                              !matrix(residual, device, mr) || mr.rows != m || mr.cols != n))
    return declined();
  d.m = m;
  d.n = n;
  d.k = ma.cols;
  d.lda = ma.pitch;
  d.ldb = mb.pitch;
  d.ldy = my.pitch;
  d.ldr = mr.pitch;
  d.row_scale = static_cast<const float *>(row);
  d.col_scale = static_cast<const float *>(col);
  d.bias = static_cast<const float *>(bias);
  d.residual = mr.p;
  d.activation = static_cast<int32_t>(activation);
  d.y_dtype = dtype_code(y.scalar_type());
  if ((d.y_dtype == INT8CONV_INT8) != (args[10] != Py_None)) return declined();
  if (args[10] != Py_None) d.out_scale = static_cast<float>(PyFloat_AsDouble(args[10]));
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return declined();
  }
  void *stream = stream_of(device);
  const auto *pa = static_cast<const int8_t *>(ma.p), *pb = static_cast<const int8_t *>(mb.p);
  int8conv_status st;
  Py_BEGIN_ALLOW_THREADS
  st = grouped ? int8conv_launch_grouped_matmul(&d, pa, pb, group_stride,
                                                static_cast<const int32_t *>(offsets),
                                                static_cast<int32_t>(groups), my.p, stream)
               : int8conv_launch_matmul(&d, pa, pb, my.p, stream);
  Py_END_ALLOW_THREADS
  if (st != INT8CONV_OK) return refused(st, grouped ? "grouped_matmul" : "matmul");
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (x, index, q, scale) -> (q, scale), or None.  q None: new buffers.
PyObject *quantize_rows(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  at::Tensor x, index, q, scale;
  if (count != 4 || tensor(args[0], x) != Arg::kTensor || !x.is_cuda()) return declined();
  const int device = c10::cuda::current_device();
  Matrix mx, mq;
  if (!matrix(x, device, mx)) return declined();
  const int code = dtype_code(x.scalar_type());
  int64_t m = mx.rows;
  const void *pi = nullptr;
  if (args[1] != Py_None) {
    if (tensor(args[1], index) != Arg::kTensor) return declined();
    m = index.numel();
    if (!vector(args[1], at::kInt, m, device, &pi)) return declined();
  }
  if (args[2] == Py_None) {
    q = empty({m, mx.cols}, at::kChar, device);
    scale = empty({m}, at::kFloat, device);
  } else if (tensor(args[2], q) != Arg::kTensor || tensor(args[3], scale) != Arg::kTensor) {
    return declined();
  }
  if (q.scalar_type() != at::kChar || !matrix(q, device, mq) || mq.rows != m || mq.cols != mx.cols)
    return declined();
  if (scale.scalar_type() != at::kFloat || scale.numel() != m || !scale.is_contiguous() ||
      !on(scale, device))
    return declined();
  void *stream = stream_of(device);
  int8conv_status st;
  Py_BEGIN_ALLOW_THREADS
  st = int8conv_launch_quantize_rows(m, mx.cols, code, mx.p, mx.rows, mx.pitch,
                                     static_cast<const int32_t *>(pi), static_cast<int8_t *>(mq.p),
                                     mq.pitch, static_cast<float *>(scale.data_ptr()), stream);
  Py_END_ALLOW_THREADS
  if (st != INT8CONV_OK) return refused(st, "quantize_rows");
  PyObject *pair = PyTuple_New(2);
  if (pair == nullptr) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(scale)));
  return pair;
  END_HANDLE_TH_ERRORS
}

// A channels-last tensor [n, ..., c] whose positions are evenly spaced.
struct Pixels {
  void *p = nullptr;
  int64_t n = 0, pixels = 0, c = 0, pitch = 0;
};

bool pixels(const at::Tensor &t, int device, Pixels &x) {
  const int64_t dims = t.dim();
  if (dims < 2 || !on(t, device)) return false;
  x.c = t.size(dims - 1);
  if (t.stride(dims - 1) != 1 && x.c > 1) return false;
  int64_t positions = 1, pitch = -1;
  for (int64_t i = dims - 2; i >= 0; --i) {
    if (t.size(i) > 1) {
      if (pitch < 0)
        pitch = t.stride(i);
      else if (t.stride(i) != pitch * positions)
        return false;
    }
    positions *= t.size(i);
  }
  x.pitch = pitch < 0 ? x.c : pitch;
  if (x.pitch < x.c) return false;
  x.n = t.size(0);
  x.pixels = x.n > 0 ? positions / x.n : 0;
  x.p = t.data_ptr();
  return true;
}

// (x, groups, gamma, beta, scale, eps, activation, dtype, out_scale) -> y, or None.
PyObject *group_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  at::Tensor x;
  if (count != 9 || tensor(args[0], x) != Arg::kTensor || !x.is_cuda()) return declined();
  const int device = c10::cuda::current_device();
  Pixels px, py;
  int8conv_group_norm d{};
  // The descriptor's channels are 32 bits wide.
  if (!pixels(x, device, px) || px.c > INT8CONV_MAX_NORM_CHANNELS) return declined();
  const void *gamma = nullptr, *beta = nullptr, *scale = nullptr;
  if (!vector(args[2], at::kFloat, px.c, device, &gamma) ||
      !vector(args[3], at::kFloat, px.c, device, &beta) ||
      !vector(args[4], at::kFloat, px.c, device, &scale))
    return declined();
  const long groups = PyLong_AsLong(args[1]);
  const double eps = PyFloat_AsDouble(args[5]);
  const long activation = PyLong_AsLong(args[6]);
  const long type = PyLong_AsLong(args[7]);
  double step = 0.0;
  if (args[8] != Py_None) step = PyFloat_AsDouble(args[8]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return declined();
  }
  if (type < 0 || type > INT8CONV_INT8 || (type == INT8CONV_INT8) != (args[8] != Py_None) ||
      groups < 1 || groups > px.c)
    return declined();
  at::Tensor y = empty(x.sizes(), scalar_type(type), device);
  if (!pixels(y, device, py)) return declined();
  d.n = px.n;
  d.pixels = px.pixels;
  d.channels = static_cast<int32_t>(px.c);
  d.groups = static_cast<int32_t>(groups);
  d.ldx = px.pitch;
  d.ldy = py.pitch;
  d.scale = static_cast<const float *>(scale);
  d.gamma = static_cast<const float *>(gamma);
  d.beta = static_cast<const float *>(beta);
  d.eps = static_cast<float>(eps);
  d.activation = static_cast<int32_t>(activation);
  d.x_dtype = dtype_code(x.scalar_type());
  d.y_dtype = static_cast<int32_t>(type);
  d.out_scale = static_cast<float>(step);
  const size_t bytes = int8conv_group_norm_workspace_bytes(&d);
  at::Tensor workspace;
  if (bytes > 0) workspace = empty({static_cast<int64_t>(bytes)}, at::kByte, device);
  void *stream = stream_of(device), *ws = bytes > 0 ? workspace.data_ptr() : nullptr;
  int8conv_status st;
  Py_BEGIN_ALLOW_THREADS
  st = int8conv_launch_group_norm(&d, px.p, py.p, ws, bytes, stream);
  Py_END_ALLOW_THREADS
  if (st != INT8CONV_OK) return refused(st, "group_norm");
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

template <class F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(f));
}

PyMethodDef methods[] = {
    {"matmul", fast(&matmul), METH_FASTCALL, nullptr},
    {"quantize_rows", fast(&quantize_rows), METH_FASTCALL, nullptr},
    {"group_norm", fast(&group_norm), METH_FASTCALL, nullptr},
    {"on_failure", &on_failure, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "torch_calls", nullptr, -1, methods,
                      nullptr,               nullptr,       nullptr, nullptr};

}  // namespace

#ifndef BUILT_FOR_TORCH
#define BUILT_FOR_TORCH "unknown"
#endif
#define TEXT_OF(x) #x
#define VERSION_TEXT(major, minor) TEXT_OF(major) "." TEXT_OF(minor)

// Nothing of torch is touched here: operators.py compares `built_for` with what
// runs before it calls anything.
PyMODINIT_FUNC PyInit_torch_calls(void) {
  PyObject *m = PyModule_Create(&module);
  if (m != nullptr &&
      PyModule_AddStringConstant(m, "built_for", "torch " BUILT_FOR_TORCH ", Python " VERSION_TEXT(
                                     PY_MAJOR_VERSION, PY_MINOR_VERSION)) != 0)
    Py_CLEAR(m);
  return m;
}
