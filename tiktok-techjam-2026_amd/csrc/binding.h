// What the Python calls of the operators share: checks of their tensors, the
// launch on the current stream of the tensors' device, errors as TjkError.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/tjk.h"

namespace {

PyObject* tjk_error = nullptr;  // tjkernels._lib.TjkError

// Its own message, raised as TjkError.
struct Refusal {
  char text[256];
};

[[noreturn]] void refuse(const char* fmt, ...) {
  Refusal r;
  va_list args;
  va_start(args, fmt);
  vsnprintf(r.text, sizeof(r.text), fmt, args);
  va_end(args);
  throw r;
}

const at::Tensor* tensor_or_none(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse("%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
  return &THPVariable_Unpack(o);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  const at::Tensor* t = tensor_or_none(o, name);
  if (!t) refuse("%s must be a tensor, got None", name);
  return *t;
}

int dtype_code(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return TJK_F32;
    case at::kHalf: return TJK_F16;
    case at::kBFloat16: return TJK_BF16;
    case at::kFloat8_e4m3fn: return TJK_E4M3;
    default: refuse("%s: unsupported dtype %s", name, c10::toString(t.scalar_type()));
  }
}

// A 2-D row-major view.  (A single row, and an empty one, may have any stride.)
struct Matrix {
  int64_t rows, cols, ld;
  int dtype;
  void* data;
};

Matrix matrix(const at::Tensor& t, const char* name) {
  if (t.dim() != 2 || (t.stride(1) != 1 && t.size(1) != 1))
    refuse("%s must be a 2-D row-major view", name);
  return {t.size(0), t.size(1), t.size(0) > 1 && t.size(1) > 0 ? t.stride(0) : t.size(1), dtype_code(t, name), t.data_ptr()};
}

void* vector_of(const at::Tensor& t, int64_t n, at::ScalarType dtype, const char* name) {
  if (t.scalar_type() != dtype || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse("%s must be a contiguous %s vector of %lld elements", name, c10::toString(dtype), (long long)n);
  return t.data_ptr();
}

// The device that all tensors lie on.
template <size_t N>
c10::DeviceIndex one_device(const at::Tensor* const (&ts)[N]) {
  const c10::Device d = ts[0]->device();
  if (!d.is_cuda()) refuse("tjkernels ops need ROCm device tensors (no CPU path)");
  for (const at::Tensor* t : ts)
    if (t && t->device() != d) refuse("tensors on %s and %s", d.str().c_str(), t->device().str().c_str());
  return d.index();
}

int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  if (v != (int)v) refuse("%s: %lld is out of range", name, v);
  return v;
}

// Calls an entry point on the device's current stream, with that device as the
// current one (a launch goes to the current device).
template <typename F>
PyObject* launch(c10::DeviceIndex device, const char* what, F call) {
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    void* const stream = c10::hip::getCurrentHIPStream(device).stream();
    const c10::DeviceIndex before = c10::hip::current_device();
    if (before != device) c10::hip::set_device(device);
    status = call(stream);
    if (before != device) c10::hip::set_device(before);
  }
  if (status) refuse("%s failed with status %d: %s", what, status, tjk_last_error_string());
  Py_RETURN_NONE;
}

// C++ exceptions end at the Python call.
template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F body) {
  HANDLE_TH_ERRORS
  try {
    if (given != wanted) refuse("%lld arguments given, %lld wanted", (long long)given, (long long)wanted);
    return body();
  } catch (const Refusal& r) {
    PyErr_SetString(tjk_error, r.text);
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// The module, if the library is the one that it was built for.
PyObject* make_module(PyModuleDef* def) {
  PyObject* const lib = PyImport_ImportModule("tjkernels._lib");
  if (!lib) return nullptr;
  tjk_error = PyObject_GetAttrString(lib, "TjkError");
  Py_DECREF(lib);
  if (!tjk_error) return nullptr;
  if (tjk_abi_version() != TJK_ABI_VERSION) {
    PyErr_Format(tjk_error, "libtjk ABI version %d, tjkernels.%s was built for %d", tjk_abi_version(), def->m_name,
                 TJK_ABI_VERSION);
    return nullptr;
  }
  return PyModule_Create(def);
}

}  // namespace
