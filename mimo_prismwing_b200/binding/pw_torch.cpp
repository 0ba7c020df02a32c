// pw_torch.cpp -- the host side of the norm and linear calls on torch tensors.
//
// For a single token these calls take 2 to 11 us on the device, and Python code that
// looks at every tensor, allocates the outputs and goes through ctypes took 9.5 to 14.5
// us per call (4.5 to 7.5 here, 3 of them the launch).  Here an asynchronous call's
// checks, descriptors and allocations are one step.  A call that is not the ordinary
// one (host rows, a shape or type to be refused, a tensor subclass) is not taken: the
// methods return None and the caller's own path, which words the refusals, runs.  A
// status is returned as an int.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_strided.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "pw_cuda.h"

namespace {

using NormFn = decltype(&pw_add_rms_norm);
using LinearFn = decltype(&pw_linear);
using CodesFn = decltype(&pw_fp8_linear_codes);

// A runtime handle, its device (-1: host tensors) and the library's entry points.
struct Calls {
  PyObject_HEAD
  pw_runtime *rt;
  int device;
  NormFn norm;
  LinearFn linear;
  CodesFn codes;
};

// PW_DTYPE_*, or -1.
int dtype_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PW_DTYPE_F32;
    case at::kBFloat16: return PW_DTYPE_BF16;
    case at::kHalf: return PW_DTYPE_F16;
    default: return -1;
  }
}

bool here(const Calls *c, const at::Tensor &t) {
  if (t.layout() != at::kStrided) return false;
  return c->device < 0 ? t.is_cpu() : t.is_cuda() && t.get_device() == c->device;
}

// An argument's tensor (not a subclass other than Parameter), or nullptr.
const at::Tensor *tensor(PyObject *o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// A 2-D tensor whose rows are contiguous and apart.
bool rows(const Calls *c, const at::Tensor &t, pw_rows &r) {
  const int d = dtype_of(t.scalar_type());
  if (d < 0 || t.dim() != 2 || !here(c, t)) return false;
  const int64_t n = t.size(0), len = t.size(1);
  int64_t stride = t.stride(0);
  if (n <= 1) stride = 0;  // one row may have any stride in torch
  if ((t.stride(1) != 1 && len > 1) || (stride < len && n > 1) || n > INT32_MAX || len > INT32_MAX) return false;
  r = pw_rows{t.data_ptr(), (uint64_t)stride, (uint32_t)d, 0u};
  return true;
}

// A contiguous vector of n.
bool vector(const Calls *c, const at::Tensor &t, int64_t n, const void *&at, uint32_t &dtype) {
  const int d = dtype_of(t.scalar_type());
  if (d < 0 || t.dim() != 1 || t.size(0) != n || !here(c, t) || !t.is_contiguous()) return false;
  at = t.data_ptr();
  dtype = (uint32_t)d;
  return true;
}

at::Tensor empty(const Calls *c, int64_t n, int64_t len, at::ScalarType t) {
  const c10::Device d = c->device < 0 ? c10::Device(c10::kCPU) : c10::Device(c10::kCUDA, (c10::DeviceIndex)c->device);
  return at::empty_strided({n, len}, {len, 1}, at::TensorOptions().dtype(t).device(d));
}

// A linear call's epilogue and output: bias, activation, residual, out_dtype, out.
bool epilogue(const Calls *c, PyObject *const *a, int64_t width, int64_t cols, at::ScalarType default_type, pw_epilogue &e,
              pw_rows &y, at::Tensor &out) {
  e = pw_epilogue{};
  if (a[0] != Py_None) {
    const at::Tensor *t = tensor(a[0]);
    if (!t || !vector(c, *t, cols, e.bias, e.bias_dtype)) return false;
  }
  if (!PyLong_Check(a[1])) return false;
  e.activation = (uint32_t)PyLong_AsUnsignedLongMask(a[1]);
  if (a[2] != Py_None) {
    const at::Tensor *t = tensor(a[2]);
    if (!t || !rows(c, *t, e.residual) || t->size(0) != width || t->size(1) != cols) return false;
  }
  if (a[4] != Py_None) {
    const at::Tensor *t = tensor(a[4]);
    if (!t || !rows(c, *t, y) || t->size(0) != width || t->size(1) != cols) return false;
    out = *t;
    return true;
  }
  at::ScalarType type = default_type;
  if (a[3] != Py_None) {
    if (!THPDtype_Check(a[3])) return false;
    type = reinterpret_cast<THPDtype *>(a[3])->scalar_type;
  }
  if (dtype_of(type) < 0) return false;
  out = empty(c, width, cols, type);
  return rows(c, out, y);
}

// What a C++ exception becomes: before the call was made, a call not taken.
PyObject *failed(bool called) {
  if (!called) Py_RETURN_NONE;
  PyErr_SetString(PyExc_RuntimeError, "the outputs of a call that was made could not be returned");
  return nullptr;
}

// A status as the methods return it, or the tensor.
PyObject *answer(int status, const at::Tensor &out) {
  return status == PW_OK ? THPVariable_Wrap(out) : PyLong_FromLong(status);
}

// linear(x, weight, bias, activation, residual, out_dtype, out)
PyObject *linear(PyObject *self, PyObject *const *a, Py_ssize_t n) {
  const Calls *c = reinterpret_cast<Calls *>(self);
  bool called = false;
  try {
    const at::Tensor *x = n == 7 ? tensor(a[0]) : nullptr, *w = x ? tensor(a[1]) : nullptr;
    pw_rows xr, wr, yr;
    pw_epilogue e;
    at::Tensor out;
    if (!w || !rows(c, *x, xr) || !rows(c, *w, wr) || x->size(1) != w->size(1) ||
        !epilogue(c, a + 2, x->size(0), w->size(0), x->scalar_type(), e, yr, out))
      Py_RETURN_NONE;
    const pw_dense d{wr.data, wr.stride, (uint32_t)w->size(0), (uint32_t)w->size(1), wr.dtype, 0u};
    const uint32_t width = (uint32_t)x->size(0);
    int status;
    called = true;
    Py_BEGIN_ALLOW_THREADS;
    status = c->linear(c->rt, &d, &xr, width, &e, &yr, PW_MEM_DEVICE | PW_MEM_ASYNC, nullptr);
    Py_END_ALLOW_THREADS;
    return answer(status, out);
  } catch (...) {
    return failed(called);
  }
}

// fp8_linear_codes(codes, scales, weight, weight_scale, layout, bias, activation, residual, out_dtype, out)
PyObject *fp8_linear_codes(PyObject *self, PyObject *const *a, Py_ssize_t n) {
  const Calls *c = reinterpret_cast<Calls *>(self);
  bool called = false;
  try {
    const at::Tensor *t[4];
    for (int i = 0; i < 4; ++i)
      if (n != 10 || !(t[i] = tensor(a[i])) || t[i]->dim() != 2 || !here(c, *t[i]) || !t[i]->is_contiguous() ||
          t[i]->size(0) > INT32_MAX || t[i]->size(1) > INT32_MAX)
        Py_RETURN_NONE;
    const int64_t width = t[0]->size(0), cols = t[0]->size(1);
    if (t[0]->scalar_type() != at::kByte || t[1]->scalar_type() != at::kFloat || t[2]->scalar_type() != at::kByte ||
        t[3]->scalar_type() != at::kFloat || t[2]->size(1) != cols || t[1]->size(0) != width ||
        t[1]->size(1) != cols / 128 || !PyLong_Check(a[4]))
      Py_RETURN_NONE;
    pw_rows yr;
    pw_epilogue e;
    at::Tensor out;
    if (!epilogue(c, a + 5, width, t[2]->size(0), at::kFloat, e, yr, out)) Py_RETURN_NONE;
    const pw_fp8_tensor w{static_cast<const uint8_t *>(t[2]->data_ptr()), static_cast<const float *>(t[3]->data_ptr()),
                          (uint32_t)t[2]->size(0),                        (uint32_t)cols,
                          (uint32_t)t[3]->size(0),                        (uint32_t)t[3]->size(1)};
    const uint32_t layout = (uint32_t)PyLong_AsUnsignedLongMask(a[4]);
    const uint8_t *codes = static_cast<const uint8_t *>(t[0]->data_ptr());
    const float *scales = static_cast<const float *>(t[1]->data_ptr());
    int status;
    called = true;
    Py_BEGIN_ALLOW_THREADS;
    status = c->codes(c->rt, &w, layout, codes, scales, (uint32_t)width, &e, &yr, PW_MEM_DEVICE | PW_MEM_ASYNC, nullptr);
    Py_END_ALLOW_THREADS;
    return answer(status, out);
  } catch (...) {
    return failed(called);
  }
}

// add_rms_norm(x, weight, epsilon, residual, want_y, want_codes, out_dtype, in_place): (sum, y, codes, scales)
PyObject *add_rms_norm(PyObject *self, PyObject *const *a, Py_ssize_t n) {
  const Calls *c = reinterpret_cast<Calls *>(self);
  bool called = false;
  try {
    const at::Tensor *x = n == 8 ? tensor(a[0]) : nullptr, *w = x ? tensor(a[1]) : nullptr;
    pw_rows xr, rr, sr, yr;
    const void *weight;
    uint32_t w_dtype;
    if (!w || !rows(c, *x, xr) || !vector(c, *w, x->size(1), weight, w_dtype) || !PyFloat_Check(a[2])) Py_RETURN_NONE;
    const int64_t T = x->size(0), H = x->size(1);
    const pw_norm norm{weight, (uint32_t)H, w_dtype, (float)PyFloat_AS_DOUBLE(a[2])};
    // the flags' truth as Python has it; -1: an error in asking
    const int want_y = PyObject_IsTrue(a[4]), want_codes = PyObject_IsTrue(a[5]), in_place = PyObject_IsTrue(a[7]);
    if (want_y < 0 || want_codes < 0 || in_place < 0) return nullptr;
    at::Tensor sum, y, codes, scales;
    if (a[3] != Py_None) {
      const at::Tensor *r = tensor(a[3]);
      if (!r || !rows(c, *r, rr) || rr.dtype != xr.dtype || r->size(0) != T || r->size(1) != H) Py_RETURN_NONE;
      sum = in_place ? *r : empty(c, T, H, x->scalar_type());
      if (!rows(c, sum, sr)) Py_RETURN_NONE;
    }
    if (want_y) {
      at::ScalarType type = x->scalar_type();
      if (a[6] != Py_None) {
        if (!THPDtype_Check(a[6])) Py_RETURN_NONE;
        type = reinterpret_cast<THPDtype *>(a[6])->scalar_type;
      }
      if (dtype_of(type) < 0) Py_RETURN_NONE;
      y = empty(c, T, H, type);
      if (!rows(c, y, yr)) Py_RETURN_NONE;
    }
    uint8_t *cp = nullptr;
    float *sp = nullptr;
    if (want_codes) {
      codes = empty(c, T, H, at::kByte);
      scales = empty(c, T, (H + 127) / 128, at::kFloat);
      cp = static_cast<uint8_t *>(codes.data_ptr());
      sp = static_cast<float *>(scales.data_ptr());
    }
    const bool add = sum.defined();
    int status;
    called = true;
    Py_BEGIN_ALLOW_THREADS;
    status = c->norm(c->rt, &norm, &xr, add ? &rr : nullptr, (uint32_t)T, add ? &sr : nullptr, want_y ? &yr : nullptr, cp,
                     sp, PW_MEM_DEVICE | PW_MEM_ASYNC, nullptr);
    Py_END_ALLOW_THREADS;
    if (status != PW_OK) return PyLong_FromLong(status);
    PyObject *result = PyTuple_New(4);
    if (!result) return nullptr;
    const at::Tensor *parts[4] = {&sum, &y, &codes, &scales};
    for (int i = 0; i < 4; ++i) {
      PyObject *o = parts[i]->defined() ? THPVariable_Wrap(*parts[i]) : Py_NewRef(Py_None);
      if (!o) {
        Py_DECREF(result);
        return nullptr;
      }
      PyTuple_SET_ITEM(result, i, o);
    }
    return result;
  } catch (...) {
    return failed(called);
  }
}

PyMethodDef methods[] = {
    {"add_rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(add_rms_norm)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
    {"fp8_linear_codes", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fp8_linear_codes)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};

// Calls(runtime, device, pw_add_rms_norm, pw_linear, pw_fp8_linear_codes): addresses as ints.
PyObject *calls_new(PyTypeObject *type, PyObject *args, PyObject *) {
  unsigned long long rt, norm, lin, codes;
  int device;
  if (!PyArg_ParseTuple(args, "KiKKK", &rt, &device, &norm, &lin, &codes)) return nullptr;
  Calls *c = reinterpret_cast<Calls *>(type->tp_alloc(type, 0));
  if (!c) return nullptr;
  c->rt = reinterpret_cast<pw_runtime *>(rt);
  c->device = device;
  c->norm = reinterpret_cast<NormFn>(norm);
  c->linear = reinterpret_cast<LinearFn>(lin);
  c->codes = reinterpret_cast<CodesFn>(codes);
  return reinterpret_cast<PyObject *>(c);
}

PyTypeObject calls_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pw_torch", nullptr, -1, nullptr, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pw_torch() {
  calls_type.tp_name = "_pw_torch.Calls";
  calls_type.tp_basicsize = sizeof(Calls);
  calls_type.tp_flags = Py_TPFLAGS_DEFAULT;
  calls_type.tp_methods = methods;
  calls_type.tp_new = calls_new;
  if (PyType_Ready(&calls_type) < 0) return nullptr;
  PyObject *m = PyModule_Create(&module);
  if (!m) return nullptr;
  if (PyModule_AddObjectRef(m, "Calls", reinterpret_cast<PyObject *>(&calls_type)) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
