// What the extension module's functions share: checks of arguments, and the call of an entry point of the C ABI.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "../../include/cswap_b200.h"

namespace cswext {

inline PyObject* g_check = nullptr;  // cswap_b200._lib.check: raises CswapError for a status

// false with a Python exception set
inline bool status_ok(csw_status st, const char* what) {
  if (st == CSW_OK) return true;
  PyObject* r = PyObject_CallFunction(g_check, "is", st, what);
  Py_XDECREF(r);
  return false;
}
inline bool value_error(const char* fmt, const char* name = nullptr) {
  PyErr_Format(PyExc_ValueError, fmt, name);  // `fmt` names one %s where `name` is given
  return false;
}
inline bool arg_count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

inline const at::Tensor* as_tensor(PyObject* o, const char* name) {
  if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
  PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
  return nullptr;
}
inline bool require_cuda_f32(const at::Tensor& t, const char* name) {
  if (!t.is_cuda()) return value_error("%s must be a CUDA tensor (this path has no CPU implementation)", name);
  if (t.scalar_type() != at::kFloat) return value_error("%s must be float32", name);
  if (!t.is_contiguous()) return value_error("%s must be contiguous", name);
  return true;
}
inline bool as_size(PyObject* o, size_t* v) {
  const Py_ssize_t x = PyNumber_AsSsize_t(o, PyExc_OverflowError);
  if (x == -1 && PyErr_Occurred()) return false;
  *v = (size_t)x;
  return true;
}

inline at::Tensor new_on(const at::Tensor& like, int64_t n, at::ScalarType type) {
  return at::empty({n}, at::TensorOptions().dtype(type).device(like.device()));
}

// What every call ends with: the ABI call on the tensor's device and torch's
// current stream there, without the interpreter lock.
template <class F>
bool launch(const at::Tensor& t, const char* what, F&& call) {
  const c10::cuda::CUDAGuard on(t.device());
  const csw_stream_t stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
  csw_status st;
  Py_BEGIN_ALLOW_THREADS;
  st = call(stream);
  Py_END_ALLOW_THREADS;
  return status_ok(st, what);
}

// C++ exceptions (an allocation that failed, say) become torch's Python ones
template <class F>
PyObject* guarded(F&& body) {
  HANDLE_TH_ERRORS
  return body();
  END_HANDLE_TH_ERRORS
}

}  // namespace cswext

extern PyMethodDef cswap_ops_methods[];  // ops_ext.cpp
