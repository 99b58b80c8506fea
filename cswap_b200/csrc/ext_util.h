// What the extension module's functions share: checks of arguments, and the call of an entry point of the C ABI.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
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

// The same outside of Python's calls, in a thread of autograd's: the exception that g_check raises, thrown
inline void require_ok(csw_status st, const char* what) {
  if (st == CSW_OK) return;
  PyGILState_STATE gil = PyGILState_Ensure();
  python_error err;
  if (!status_ok(st, what)) err.persist();
  PyGILState_Release(gil);
  throw err;
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

// ---- tensors of the training operators -------------------------------------------------------------------------------
// The CSW_TYPE_* code of a tensor's type, -1 for another one
inline int type_code(at::ScalarType t) {
  return t == at::kFloat ? CSW_TYPE_F32 : t == at::kHalf ? CSW_TYPE_F16 : t == at::kBFloat16 ? CSW_TYPE_BF16 : -1;
}
inline bool require_values(const at::Tensor& t, const char* name, int* type) {
  if (!t.is_cuda()) return value_error("%s must be a CUDA tensor (this path has no CPU implementation)", name);
  *type = type_code(t.scalar_type());
  if (*type < 0) return value_error("%s must be float32, float16 or bfloat16", name);
  return true;
}
inline bool require_flat(const at::Tensor& t, const char* name) {
  if (!t.is_contiguous()) return value_error("%s must be contiguous", name);
  return true;
}
inline bool same_device(const at::Tensor& t, const at::Tensor& as, const char* name) {
  if (t.device() != as.device()) return value_error("%s is on another device", name);
  return true;
}
inline bool optional_tensor(PyObject* o, const char* name, const at::Tensor** t) {
  *t = nullptr;
  return o == Py_None || (*t = as_tensor(o, name)) != nullptr;
}
inline void* ptr(const at::Tensor& t) { return t.numel() ? const_cast<void*>(t.const_data_ptr()) : nullptr; }
inline void* out(at::Tensor& t) { return t.numel() ? t.mutable_data_ptr() : nullptr; }

// New tensors on a tensor's device, without the way through torch's dispatcher: the smallest calls are as long as their
// allocations.
inline at::Tensor fresh(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}
inline at::Tensor fresh(const at::Tensor& like) { return fresh(like, like.sizes(), like.scalar_type()); }

// A new tuple of the tensors; an undefined one becomes None
inline PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = nullptr;
    if (r) o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) {
      Py_XDECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// While a graph is captured, refuses a leaf, also behind views and copies, whose gradient accumulator a graph of another
// stream keeps (with a Python exception set).  Backward would hand the gradient over to that stream in the middle of the
// capture, an error that autograd's threads do not survive.  (ops_ext.cpp)
bool capture_allows(const at::Tensor& t);

#define CSW_METHOD(name, doc) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, doc}

}  // namespace cswext

extern PyMethodDef cswap_ops_methods[];   // ops_ext.cpp
extern PyMethodDef cswap_step_methods[];  // step_ext.cpp
