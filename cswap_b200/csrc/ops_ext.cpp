// Tensor-level front end of the training operators (the wrappers in ops.py keep the documented signatures; these
// functions take every argument by position).  As with the codecs it is there for host time: the smallest calls run
// 3 us on the GPU.
#include "ext_util.h"

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cmath>

using namespace cswext;

namespace {
std::shared_ptr<torch::autograd::Node> accumulator_of(const at::Tensor& t);
}  // namespace

bool cswext::capture_allows(const at::Tensor& t) {
  if (!t.is_cuda() || !t.requires_grad()) return true;
  const c10::cuda::CUDAGuard on(t.device());  // the operands of a call are on one device, and refused otherwise
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return true;
  const auto node = accumulator_of(t);
  if (!node) return true;
  const auto stream = node->stream();
  if (!stream || *stream == c10::cuda::getCurrentCUDAStream(t.device().index()).unwrap()) return true;
  PyErr_SetString(PyExc_RuntimeError,
                  "a leaf of this captured step is also a leaf of a live graph of another stream: "
                  "let go of that graph (its outputs and losses) before the capture");
  return false;
}

namespace {

bool require_like(const at::Tensor& t, const at::Tensor& as, const char* name) {
  if (!same_device(t, as, name)) return false;
  if (t.scalar_type() != as.scalar_type()) return value_error("%s has another type than the input", name);
  if (!t.sizes().equals(as.sizes())) return value_error("%s has another shape than the input", name);
  return require_flat(t, name);
}
bool require_f32(const at::Tensor& t, const at::Tensor& as, int64_t n, const char* name) {
  if (!same_device(t, as, name)) return false;
  if (t.scalar_type() != at::kFloat) return value_error("%s must be float32", name);
  if (t.numel() != n) return value_error("%s has the wrong number of values", name);
  return require_flat(t, name);
}
// an output that the caller gives, of which `written` bytes are written while others of `read` may not have been read
bool require_apart(const at::Tensor& out, size_t written, const at::Tensor& in, size_t read) {
  const char *a = static_cast<const char*>(out.const_data_ptr()), *b = static_cast<const char*>(in.const_data_ptr());
  const bool apart = written == 0 || read == 0 || a + written <= b || b + read <= a;
  return apart || value_error("%s overlaps the input", "out");
}
// ---- 8-bit checkpoints ---------------------------------------------------------------------------------------------
bool q8_bytes(size_t n, size_t* need) { return status_ok(csw_q8_bytes(n, need), "csw_q8_bytes"); }
bool packed_out(PyObject* o, const at::Tensor& like, size_t n, at::Tensor* packed) {
  size_t need;
  if (!q8_bytes(n, &need)) return false;
  if (o == Py_None) {
    *packed = fresh(like, {(int64_t)need}, at::kByte);
    return true;
  }
  const at::Tensor* t = as_tensor(o, "out");
  if (!t) return false;
  if (t->scalar_type() != at::kByte) return value_error("%s must be uint8", "out");
  if (!same_device(*t, like, "out") || !require_flat(*t, "out") || !require_apart(*t, need, like, like.nbytes()))
    return false;
  *packed = *t;
  return true;
}
bool packed_in(const at::Tensor& t) {
  if (!t.is_cuda()) return value_error("%s must be a CUDA tensor (this path has no CPU implementation)", "packed");
  if (t.scalar_type() != at::kByte) return value_error("%s must be uint8", "packed");
  return require_flat(t, "packed");
}

// q8_compress(t, out) -> packed
PyObject* q8_compress(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int type;
    at::Tensor packed;
    if (!arg_count(n, 2)) return nullptr;
    const at::Tensor* t = as_tensor(a[0], "t");
    if (!t || !require_values(*t, "t", &type) || !require_flat(*t, "t") || !packed_out(a[1], *t, t->numel(), &packed))
      return nullptr;
    const void* src = ptr(*t);
    void* dst = out(packed);
    if (!launch(*t, "csw_q8_compress", [&](csw_stream_t s) {
          return csw_q8_compress(src, type, (size_t)t->numel(), dst, (size_t)packed.numel(), s);
        }))
      return nullptr;
    return THPVariable_Wrap(packed);
  });
}

// q8_decompress(packed, numel, dtype, out) -> tensor
PyObject* q8_decompress(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    size_t numel, need;
    int type;
    if (!arg_count(n, 4)) return nullptr;
    const at::Tensor* packed = as_tensor(a[0], "packed");
    if (!packed || !packed_in(*packed) || !as_size(a[1], &numel)) return nullptr;
    if ((Py_ssize_t)numel < 0) {
      value_error("numel must not be negative");
      return nullptr;
    }
    at::Tensor dst;
    if (a[3] == Py_None) {
      if (!THPDtype_Check(a[2])) {
        PyErr_SetString(PyExc_TypeError, "dtype must be a torch.dtype");
        return nullptr;
      }
      const at::ScalarType kind = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
      if (type_code(kind) < 0) {
        value_error("%s must be float32, float16 or bfloat16", "dtype");
        return nullptr;
      }
      if (!q8_bytes(numel, &need)) return nullptr;
      if ((size_t)packed->numel() < need) {
        status_ok(CSW_ERR_SIZE, "csw_q8_decompress");
        return nullptr;
      }
      dst = fresh(*packed, {(int64_t)numel}, kind);
    } else {
      const at::Tensor* o = as_tensor(a[3], "out");
      if (!o || !same_device(*o, *packed, "out") || !require_flat(*o, "out") || !q8_bytes(numel, &need) ||
          !require_apart(*o, o->nbytes(), *packed, std::min<size_t>(need, packed->nbytes())))
        return nullptr;
      if ((size_t)o->numel() != numel) {
        value_error("%s has the wrong number of values", "out");
        return nullptr;
      }
      dst = *o;
    }
    if (!require_values(dst, "out", &type)) return nullptr;
    const void* src = ptr(*packed);
    void* to = out(dst);
    if (!launch(*packed, "csw_q8_decompress", [&](csw_stream_t s) {
          return csw_q8_decompress(src, (size_t)packed->numel(), numel, to, type, s);
        }))
      return nullptr;
    return THPVariable_Wrap(dst);
  });
}

// gelu_forward(x) -> (y, packed)
PyObject* gelu_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int type;
    at::Tensor packed;
    if (!arg_count(n, 1)) return nullptr;
    const at::Tensor* x = as_tensor(a[0], "x");
    if (!x || !require_values(*x, "x", &type) || !require_flat(*x, "x") ||
        !packed_out(Py_None, *x, x->numel(), &packed))
      return nullptr;
    at::Tensor y = fresh(*x);
    const void* src = ptr(*x);
    void *dst = out(y), *codes = out(packed);
    if (!launch(*x, "csw_gelu_forward", [&](csw_stream_t s) {
          return csw_gelu_forward(src, type, (size_t)x->numel(), dst, codes, (size_t)packed.numel(), s);
        }))
      return nullptr;
    return tuple_of({y, packed});
  });
}

// gelu_backward(dy, packed, recompute) -> dx, or (dx, y)
PyObject* gelu_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int type;
    if (!arg_count(n, 3)) return nullptr;
    const at::Tensor* dy = as_tensor(a[0], "dy");
    const at::Tensor* packed = dy ? as_tensor(a[1], "packed") : nullptr;
    if (!packed || !require_values(*dy, "dy", &type) || !require_flat(*dy, "dy") || !packed_in(*packed) ||
        !same_device(*packed, *dy, "packed"))
      return nullptr;
    const int recompute = PyObject_IsTrue(a[2]);
    if (recompute < 0) return nullptr;
    at::Tensor dx = fresh(*dy), y;
    if (recompute) y = fresh(*dy);
    const void *src = ptr(*dy), *codes = ptr(*packed);
    void *dst = out(dx), *again = recompute ? out(y) : nullptr;
    if (!launch(*dy, "csw_gelu_backward", [&](csw_stream_t s) {
          return csw_gelu_backward(src, type, codes, (size_t)packed->numel(), (size_t)dy->numel(), dst, again, s);
        }))
      return nullptr;
    return recompute ? tuple_of({dx, y}) : THPVariable_Wrap(dx);
  });
}

// ---- layer norm ----------------------------------------------------------------------------------------------------
// rows and columns of a tensor normed over its last axis, and its parameters' type
bool norm_shape(const at::Tensor& x, const at::Tensor* weight, const at::Tensor* bias, int type, int64_t* rows,
                int64_t* cols, int* param_type) {
  if (x.dim() < 1 || x.size(-1) < 1) return value_error("x needs a last axis of at least one value");
  *cols = x.size(-1);
  *rows = x.numel() / *cols;
  *param_type = type;
  if (bias && !weight) return value_error("a bias needs a weight");
  for (const at::Tensor* p : {weight, bias}) {
    if (!p) continue;
    const char* name = p == weight ? "weight" : "bias";
    if (!require_values(*p, name, param_type) || !same_device(*p, x, name) || !require_flat(*p, name)) return false;
    if (p->dim() != 1 || p->numel() != *cols) return value_error("%s must hold one value for each column", name);
    if (*param_type != type && *param_type != CSW_TYPE_F32)
      return value_error("%s must have the input's type, or float32", name);
  }
  if (weight && bias && weight->scalar_type() != bias->scalar_type())
    return value_error("weight and bias have different types");
  return true;
}

// layer_norm_forward(x, weight, bias, eps, residual) -> (y, sum, mean, rstd)
PyObject* layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int type, param_type;
    int64_t rows, cols;
    const at::Tensor *weight, *bias, *residual;
    if (!arg_count(n, 5)) return nullptr;
    const at::Tensor* x = as_tensor(a[0], "x");
    if (!x || !optional_tensor(a[1], "weight", &weight) || !optional_tensor(a[2], "bias", &bias) ||
        !optional_tensor(a[4], "residual", &residual) || !require_values(*x, "x", &type) || !require_flat(*x, "x") ||
        !norm_shape(*x, weight, bias, type, &rows, &cols, &param_type) ||
        (residual && !require_like(*residual, *x, "residual")))
      return nullptr;
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    if (!(eps >= 0.0)) {
      value_error("eps must not be negative");
      return nullptr;
    }
    at::Tensor y = fresh(*x), sum = *x;
    if (residual) sum = fresh(*x);
    at::Tensor mean = fresh(*x, {rows}, at::kFloat), rstd = fresh(*x, {rows}, at::kFloat);
    const void *src = ptr(*x), *r = residual ? ptr(*residual) : nullptr, *w = weight ? ptr(*weight) : nullptr,
               *b = bias ? ptr(*bias) : nullptr;
    void *to = out(y), *held = residual ? out(sum) : nullptr;
    float *m = static_cast<float*>(out(mean)), *d = static_cast<float*>(out(rstd));
    if (!launch(*x, "csw_layer_norm_forward", [&](csw_stream_t s) {
          return csw_layer_norm_forward(src, r, w, b, type, param_type, rows, cols, (float)eps, to, held, m, d, s);
        }))
      return nullptr;
    return tuple_of({y, sum, mean, rstd});
  });
}

// layer_norm_backward(dy, x, mean, rstd, weight, sums) -> (dx, dweight, dbias); sums: whether the last two are wanted
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int type, param_type;
    int64_t rows, cols;
    const at::Tensor* weight;
    if (!arg_count(n, 6)) return nullptr;
    const at::Tensor* dy = as_tensor(a[0], "dy");
    const at::Tensor* x = dy ? as_tensor(a[1], "x") : nullptr;
    const at::Tensor* mean = x ? as_tensor(a[2], "mean") : nullptr;
    const at::Tensor* rstd = mean ? as_tensor(a[3], "rstd") : nullptr;
    if (!rstd || !optional_tensor(a[4], "weight", &weight) || !require_values(*x, "x", &type) ||
        !require_flat(*x, "x") || !norm_shape(*x, weight, nullptr, type, &rows, &cols, &param_type) ||
        !require_like(*dy, *x, "dy") || !require_f32(*mean, *x, rows, "mean") || !require_f32(*rstd, *x, rows, "rstd"))
      return nullptr;
    const int wanted = PyObject_IsTrue(a[5]);
    if (wanted < 0) return nullptr;
    at::Tensor dx = fresh(*x), dw, db, space;
    void *pw = nullptr, *pb = nullptr, *ws = nullptr;
    size_t need = 0;
    if (weight && wanted) {
      const c10::cuda::CUDAGuard on(x->device());  // the size goes by the device's SMs
      if (!status_ok(csw_layer_norm_workspace(rows, cols, &need), "csw_layer_norm_workspace")) return nullptr;
      dw = fresh(*weight);
      db = fresh(*weight);
      space = fresh(*x, {(int64_t)need}, at::kByte);
      pw = out(dw), pb = out(db), ws = out(space);
    }
    const void *g = ptr(*dy), *src = ptr(*x), *w = weight ? ptr(*weight) : nullptr;
    const float *m = static_cast<float*>(ptr(*mean)), *d = static_cast<float*>(ptr(*rstd));
    void* to = out(dx);
    if (!launch(*x, "csw_layer_norm_backward", [&](csw_stream_t s) {
          return csw_layer_norm_backward(g, src, m, d, w, type, param_type, rows, cols, to, pw, pb, ws, need, s);
        }))
      return nullptr;
    return tuple_of({dx, dw, db});
  });
}

// ---- attention -----------------------------------------------------------------------------------------------------
// A tensor [batch, heads, tokens, dim] as the kernels take it; one that lies otherwise (values of a head apart,
// strides that are no multiple of 16 bytes, an expanded axis) is copied.
struct Operand {
  at::Tensor t;
  csw_attention_operand o;
};
Operand operand_of(const at::Tensor& given) {
  Operand r;
  r.t = given;
  auto lies = [](const at::Tensor& t) {
    if (t.numel() == 0) return true;
    if (t.stride(3) != 1 && t.size(3) != 1) return false;
    for (int i = 0; i < 3; ++i)
      if (t.size(i) > 1 && (t.stride(i) % 8 || t.stride(i) == 0)) return false;
    return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  };
  if (!lies(r.t)) r.t = given.clone(at::MemoryFormat::Contiguous);
  auto stride = [&](int i) { return r.t.size(i) > 1 ? (ptrdiff_t)r.t.stride(i) : 0; };
  r.o = {ptr(r.t), stride(0), stride(1), stride(2)};
  return r;
}
// A new tensor of like's shape, its tokens in front of its heads where they lie so in `like`
Operand new_operand(const at::Tensor& like) {
  const bool tokens_first = like.size(1) > 1 && like.size(2) > 1 && like.stride(1) < like.stride(2);
  at::Tensor t = tokens_first ? fresh(like, {like.size(0), like.size(2), like.size(1), like.size(3)}, like.scalar_type()).transpose(1, 2)
                              : fresh(like);
  return operand_of(t);
}

struct Attention {
  const at::Tensor *q, *k, *v, *lens;
  csw_attention_shape s;
};
// (q, k, v, causal, kv_lens, scale) from six arguments in a row
bool attention_of(PyObject* const* a, Attention* at) {
  int type;
  if (!(at->q = as_tensor(a[0], "q")) || !(at->k = as_tensor(a[1], "k")) || !(at->v = as_tensor(a[2], "v")) ||
      !optional_tensor(a[4], "kv_lens", &at->lens))
    return false;
  const at::Tensor &q = *at->q, &k = *at->k, &v = *at->v;
  if (!require_values(q, "q", &type)) return false;
  if (type == CSW_TYPE_F32) return value_error("%s must be float16 or bfloat16", "q");
  for (const at::Tensor* t : {at->k, at->v}) {
    const char* name = t == at->k ? "k" : "v";
    if (!same_device(*t, q, name)) return false;
    if (t->scalar_type() != q.scalar_type()) return value_error("%s has another type than q", name);
  }
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) return value_error("q, k and v must be [batch, heads, tokens, dim]");
  if (!k.sizes().equals(v.sizes())) return value_error("k and v have different shapes");
  if (k.size(0) != q.size(0) || k.size(3) != q.size(3)) return value_error("q and k differ in batch or dim");
  if (q.size(3) % 8 || q.size(3) < 8 || q.size(3) > 128) return value_error("dim must be a multiple of 8 up to 128");
  if (k.size(1) < 1 || q.size(1) < 1 || q.size(1) % k.size(1))
    return value_error("the heads of q must be a multiple of those of k");
  const int causal = PyObject_IsTrue(a[3]);
  if (causal < 0) return false;
  if (at->lens) {
    const at::Tensor& l = *at->lens;
    if (!l.is_cuda() || l.scalar_type() != at::kInt || l.dim() != 1 || l.numel() != q.size(0) || !l.is_contiguous())
      return value_error("kv_lens must be a contiguous int32 CUDA tensor with one length for each batch entry");
    if (!same_device(l, q, "kv_lens")) return false;
  }
  double scale;
  if (a[5] == Py_None) {
    scale = 1.0 / std::sqrt((double)q.size(3));
  } else {
    scale = PyFloat_AsDouble(a[5]);
    if (scale == -1.0 && PyErr_Occurred()) return false;
    if (!std::isfinite((float)scale)) return value_error("scale must be finite");
  }
  at->s = {type, causal, (size_t)q.size(0), (size_t)q.size(1), (size_t)k.size(1), (size_t)q.size(2), (size_t)k.size(2),
           (size_t)q.size(3), (float)scale, at->lens ? static_cast<const int32_t*>(ptr(*at->lens)) : nullptr};
  return true;
}

// attention_forward(q, k, v, causal, kv_lens, scale) -> (o, lse)
PyObject* attention_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Attention f;
    if (!arg_count(n, 6) || !attention_of(a, &f)) return nullptr;
    const c10::cuda::CUDAGuard on(f.q->device());
    const Operand q = operand_of(*f.q), k = operand_of(*f.k), v = operand_of(*f.v), o = new_operand(*f.q);
    at::Tensor lse = fresh(*f.q, {f.q->size(0), f.q->size(1), f.q->size(2)}, at::kFloat);
    float* l = static_cast<float*>(out(lse));
    if (!launch(*f.q, "csw_attention_forward", [&](csw_stream_t s) {
          return csw_attention_forward(&f.s, &q.o, &k.o, &v.o, &o.o, l, s);
        }))
      return nullptr;
    return tuple_of({o.t, lse});
  });
}

// attention_backward(do, q, k, v, causal, kv_lens, scale, o, lse) -> (dq, dk, dv)
PyObject* attention_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Attention f;
    if (!arg_count(n, 9) || !attention_of(a + 1, &f)) return nullptr;
    const at::Tensor* dout = as_tensor(a[0], "do");
    const at::Tensor* given = dout ? as_tensor(a[7], "o") : nullptr;
    const at::Tensor* lse = given ? as_tensor(a[8], "lse") : nullptr;
    if (!lse || !require_f32(*lse, *f.q, f.q->size(0) * f.q->size(1) * f.q->size(2), "lse")) return nullptr;
    for (const at::Tensor* t : {dout, given}) {
      const char* name = t == dout ? "do" : "o";
      if (!same_device(*t, *f.q, name)) return nullptr;
      if (t->scalar_type() != f.q->scalar_type() || !t->sizes().equals(f.q->sizes())) {
        value_error("%s has another type or shape than q", name);
        return nullptr;
      }
    }
    const c10::cuda::CUDAGuard on(f.q->device());
    size_t need;
    if (!status_ok(csw_attention_workspace(&f.s, &need), "csw_attention_workspace")) return nullptr;
    const Operand q = operand_of(*f.q), k = operand_of(*f.k), v = operand_of(*f.v), o = operand_of(*given),
                  d = operand_of(*dout), dq = new_operand(*f.q), dk = new_operand(*f.k), dv = new_operand(*f.v);
    at::Tensor space = fresh(*f.q, {(int64_t)need}, at::kByte);
    const float* l = static_cast<const float*>(ptr(*lse));
    void* ws = out(space);
    if (!launch(*f.q, "csw_attention_backward", [&](csw_stream_t s) {
          return csw_attention_backward(&f.s, &q.o, &k.o, &v.o, &o.o, l, &d.o, &dq.o, &dk.o, &dv.o, ws, need, s);
        }))
      return nullptr;
    return tuple_of({dq.t, dk.t, dv.t});
  });
}

// The gradient accumulator of the leaf that a tensor is, or is a view, a copy or another function of alone; null where there
// is none, or where the tensor depends on more than one.
std::shared_ptr<torch::autograd::Node> accumulator_of(const at::Tensor& t) {
  if (t.is_leaf()) return torch::autograd::impl::try_get_grad_accumulator(t);
  std::shared_ptr<torch::autograd::Node> node = t.grad_fn();
  while (node && !node->next_edges().empty()) {
    std::shared_ptr<torch::autograd::Node> next;
    for (const torch::autograd::Edge& e : node->next_edges()) {
      if (!e.is_valid()) continue;
      if (next) return nullptr;
      next = e.function;
    }
    node = std::move(next);
  }
  return node && dynamic_cast<torch::autograd::AccumulateGrad*>(node.get()) ? node : nullptr;
}

// check_capture(tensors): capture_allows
PyObject* check_capture(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    for (Py_ssize_t i = 0; i < n; ++i)
      if (THPVariable_Check(a[i]) && !capture_allows(THPVariable_Unpack(a[i]))) return nullptr;
    Py_RETURN_NONE;
  });
}

}  // namespace

PyMethodDef cswap_ops_methods[] = {
    CSW_METHOD(q8_compress, "(t, out) -> packed"),
    CSW_METHOD(q8_decompress, "(packed, numel, dtype, out) -> tensor"),
    CSW_METHOD(gelu_forward, "(x) -> (y, packed)"),
    CSW_METHOD(gelu_backward, "(dy, packed, recompute) -> dx or (dx, y)"),
    CSW_METHOD(layer_norm_forward, "(x, weight, bias, eps, residual) -> (y, sum, mean, rstd)"),
    CSW_METHOD(layer_norm_backward, "(dy, x, mean, rstd, weight, sums) -> (dx, dweight, dbias)"),
    CSW_METHOD(attention_forward, "(q, k, v, causal, kv_lens, scale) -> (o, lse)"),
    CSW_METHOD(attention_backward, "(do, q, k, v, causal, kv_lens, scale, o, lse) -> (dq, dk, dv)"),
    CSW_METHOD(check_capture, "(*tensors) -> None"),
    {nullptr, nullptr, 0, nullptr}};
