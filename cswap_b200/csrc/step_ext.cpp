// Tensor-level front end of the 8-bit floating-point matrices and the optimizer's step (the wrappers in fp8.py and optim.py
// keep the documented signatures; these functions take every argument by position).
#include "ext_util.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <utility>
#include <vector>

using namespace cswext;

namespace {

int64_t blocks_of(int64_t n) { return n / 128 + (n % 128 != 0); }
int64_t padded(int64_t n) { return (n + 15) / 16 * 16; }

// ---- matrices in 8-bit floating point ------------------------------------------------------------------------------
// Whether codes lie as the kernels read them: rows `stride` bytes apart, which begin on 16 bytes and have their padding to
// a multiple of 16 behind them, the last one, too.
bool lies_padded(const at::Tensor& c, int64_t* stride) {
  const int64_t rows = c.size(0), cols = c.size(1);
  *stride = rows > 1 ? c.stride(0) : padded(cols);
  if (rows == 0 || cols == 0) return true;
  const int64_t held = (int64_t)c.storage().nbytes() - c.storage_offset();
  return (cols == 1 || c.stride(1) == 1) && *stride % 16 == 0 && *stride >= cols && held >= rows * *stride &&
         reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0;
}
// codes and scales as fp8_quantize gives them
bool matrix_of(PyObject* codes, PyObject* scales, const char* name, const char* scales_name, const at::Tensor** t,
               csw_fp8_matrix* m) {
  const at::Tensor* c = as_tensor(codes, name);
  const at::Tensor* s = c ? as_tensor(scales, scales_name) : nullptr;
  if (!s) return false;
  if (!c->is_cuda()) return value_error("%s must be a CUDA tensor (this path has no CPU implementation)", name);
  if (c->scalar_type() != at::kFloat8_e4m3fn || c->dim() != 2)
    return value_error("%s must be a matrix of float8_e4m3fn codes", name);
  const int64_t rows = c->size(0), cols = c->size(1);
  int64_t stride;
  if (!lies_padded(*c, &stride))
    return value_error("%s must have rows that begin on 16 bytes and are padded to a multiple of them", name);
  if (!same_device(*s, *c, scales_name)) return false;
  if (s->scalar_type() != at::kFloat8_e8m0fnu || s->dim() != 2 || s->size(0) != blocks_of(rows) || s->size(1) != blocks_of(cols))
    return value_error("%s must be float8_e8m0fnu, one for each block of 128 x 128 codes", scales_name);
  if (!require_flat(*s, scales_name)) return false;
  *t = c;
  *m = {ptr(*c), ptr(*s), (size_t)rows, (size_t)cols, (size_t)stride, 0};
  return true;
}

bool dtype_of(PyObject* o, at::ScalarType* kind, int* type) {
  if (!THPDtype_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "dtype must be a torch.dtype");
    return false;
  }
  *kind = reinterpret_cast<THPDtype*>(o)->scalar_type;
  *type = type_code(*kind);
  return *type >= 0 || value_error("%s must be float32, float16 or bfloat16", "dtype");
}

struct Quantized {
  at::Tensor codes, scales, sums;
};
// A matrix of rows that lie `stride` values apart.  The values are checked; what the call itself finds wrong is thrown.
Quantized quantized(const at::Tensor& x, int type, int64_t rows, int64_t cols, int64_t stride, bool sums,
                    at::ScalarType sums_kind) {
  const c10::cuda::CUDAGuard on(x.device());
  size_t need;
  require_ok(csw_fp8_quantize_workspace(rows, cols, &need), "csw_fp8_quantize_workspace");
  const int64_t code_stride = padded(cols);
  Quantized q{fresh(x, {rows, code_stride}, at::kFloat8_e4m3fn), fresh(x, {blocks_of(rows), blocks_of(cols)}, at::kFloat8_e8m0fnu), {}};
  at::Tensor space;
  void* ws = nullptr;
  void* totals = nullptr;
  if (sums) {
    q.sums = fresh(x, {cols}, sums_kind);
    totals = out(q.sums);
    if (need) {
      space = fresh(x, {(int64_t)need}, at::kByte);
      ws = out(space);
    }
  }
  require_ok(csw_fp8_quantize(ptr(x), type, rows, cols, stride, out(q.codes), code_stride, out(q.scales), totals,
                              type_code(sums_kind), ws, need,
                              c10::cuda::getCurrentCUDAStream(x.device().index()).stream()),
             "csw_fp8_quantize");
  if (code_stride != cols) q.codes = q.codes.as_strided({rows, cols}, {code_stride, 1});
  return q;
}
// whether t is a matrix whose rows lie apart by some distance, or one behind the other
bool lies_in_rows(const at::Tensor& t) {
  return t.is_contiguous() ||
         (t.dim() == 2 && t.size(0) > 1 && (t.size(1) == 1 || t.stride(1) == 1) && t.stride(0) >= t.size(1));
}
Quantized quantized(const at::Tensor& x, int type, bool sums, at::ScalarType sums_kind = at::kFloat) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  const int64_t cols = x.size(-1);
  return quantized(x, type, rows, cols, x.is_contiguous() ? cols : x.stride(0), sums, sums_kind);
}
// of codes that lie padded
csw_fp8_matrix matrix_of(const at::Tensor& codes, const at::Tensor& scales, bool transposed) {
  int64_t stride;
  lies_padded(codes, &stride);
  return {ptr(codes), ptr(scales), (size_t)codes.size(0), (size_t)codes.size(1), (size_t)stride, transposed};
}
// A matrix that autograd has kept, as the kernels read it.  It has been through the program's saved-tensor hooks: a copy that
// went through the host's memory lies densely, its rows without their padding, which is put back here.
void as_kept(at::Tensor* codes, at::Tensor* scales, int64_t rows, int64_t cols, const at::Device& on) {
  auto is = [&](const at::Tensor& t, at::ScalarType kind, int64_t r, int64_t c) {
    return t.defined() && t.device() == on && t.layout() == at::kStrided && t.scalar_type() == kind && t.dim() == 2 && t.size(0) == r &&
           t.size(1) == c;
  };
  TORCH_CHECK(is(*codes, at::kFloat8_e4m3fn, rows, cols) && is(*scales, at::kFloat8_e8m0fnu, blocks_of(rows), blocks_of(cols)),
              "fp8_linear: a saved-tensor hook gave back a tensor of another type, shape or device than the one it was given");
  int64_t stride;
  if (!lies_padded(*codes, &stride)) {
    const at::Tensor room = fresh(*codes, {rows, padded(cols)}, at::kByte).narrow(1, 0, cols);
    room.copy_(codes->view(at::kByte));
    *codes = room.view(at::kFloat8_e4m3fn);
  }
  if (!scales->is_contiguous()) *scales = scales->view(at::kByte).contiguous().view(at::kFloat8_e8m0fnu);
}
at::Tensor product(const csw_fp8_matrix& a, const csw_fp8_matrix& b, const at::Tensor* bias, const at::Tensor& like,
                   at::ScalarType kind, at::IntArrayRef sizes) {
  const c10::cuda::CUDAGuard on(like.device());
  at::Tensor dst = fresh(like, sizes, kind);
  require_ok(csw_fp8_matmul(&a, &b, bias ? ptr(*bias) : nullptr, bias ? type_code(bias->scalar_type()) : 0, out(dst),
                            type_code(kind), c10::cuda::getCurrentCUDAStream(like.device().index()).stream()),
             "csw_fp8_matmul");
  return dst;
}

// fp8_quantize(x, sums) -> (codes, scales), or with their columns' sums
PyObject* fp8_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int type;
    if (!arg_count(n, 2)) return nullptr;
    const at::Tensor* x = as_tensor(a[0], "x");
    if (!x || !require_values(*x, "x", &type)) return nullptr;
    const int wanted = PyObject_IsTrue(a[1]);
    if (wanted < 0) return nullptr;
    if (x->dim() < 1) {
      value_error("x needs one axis at least");
      return nullptr;
    }
    if (!lies_in_rows(*x)) {
      value_error("%s must be contiguous", "x");
      return nullptr;
    }
    const Quantized q = quantized(*x, type, wanted);
    return wanted ? tuple_of({q.codes, q.scales, q.sums}) : tuple_of({q.codes, q.scales});
  });
}

// fp8_dequantize(codes, scales, dtype) -> tensor
PyObject* fp8_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* codes;
    csw_fp8_matrix m;
    at::ScalarType kind;
    int type;
    if (!arg_count(n, 3) || !matrix_of(a[0], a[1], "codes", "scales", &codes, &m) || !dtype_of(a[2], &kind, &type))
      return nullptr;
    at::Tensor dst = fresh(*codes, codes->sizes(), kind);
    void* to = out(dst);
    if (!launch(*codes, "csw_fp8_dequantize", [&](csw_stream_t s) {
          return csw_fp8_dequantize(m.codes, m.code_stride, m.scales, m.rows, m.cols, to, type, s);
        }))
      return nullptr;
    return THPVariable_Wrap(dst);
  });
}

// fp8_matmul(a, a_scales, b, b_scales, transpose_a, transpose_b, bias, dtype) -> tensor
PyObject* fp8_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *l, *r, *bias;
    csw_fp8_matrix left, right;
    at::ScalarType kind;
    int type, bias_type = 0;
    if (!arg_count(n, 8) || !matrix_of(a[0], a[1], "a", "a_scales", &l, &left) ||
        !matrix_of(a[2], a[3], "b", "b_scales", &r, &right) || !same_device(*r, *l, "b") ||
        !optional_tensor(a[6], "bias", &bias) || !dtype_of(a[7], &kind, &type))
      return nullptr;
    left.transposed = PyObject_IsTrue(a[4]), right.transposed = PyObject_IsTrue(a[5]);
    if (left.transposed < 0 || right.transposed < 0) return nullptr;
    const size_t rows = left.transposed ? left.cols : left.rows, inner = left.transposed ? left.rows : left.cols;
    const size_t cols = right.transposed ? right.rows : right.cols;
    if (inner != (right.transposed ? right.cols : right.rows)) {
      value_error("a and b do not fit: the columns of the one must be the rows of the other");
      return nullptr;
    }
    if (bias) {
      if (!require_values(*bias, "bias", &bias_type) || !same_device(*bias, *l, "bias") || !require_flat(*bias, "bias"))
        return nullptr;
      if (bias->dim() != 1 || (size_t)bias->numel() != cols) {
        value_error("%s must hold one value for each column of the product", "bias");
        return nullptr;
      }
    }
    at::Tensor dst = fresh(*l, {(int64_t)rows, (int64_t)cols}, kind);
    void* to = out(dst);
    const void* more = bias ? ptr(*bias) : nullptr;
    if (!launch(*l, "csw_fp8_matmul", [&](csw_stream_t s) {
          return csw_fp8_matmul(&left, &right, more, bias_type, to, type, s);
        }))
      return nullptr;
    return THPVariable_Wrap(dst);
  });
}

// The linear layer as a node of autograd's, without Python in its backward pass: a layer of a few hundred rows takes less time
// than a function of Python's there.
struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
  using Context = torch::autograd::AutogradContext;
  static at::Tensor forward(Context* ctx, const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& bias) {
    const Quantized held = quantized(x, type_code(x.scalar_type()), false);
    const Quantized w = quantized(weight, type_code(weight.scalar_type()), false);
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = weight.size(0);
    // what a gradient that is not asked for would need is not kept
    const bool keep_x = weight.requires_grad(), keep_w = x.requires_grad();
    ctx->save_for_backward({keep_x ? held.codes : at::Tensor(), keep_x ? held.scales : at::Tensor(),
                            keep_w ? w.codes : at::Tensor(), keep_w ? w.scales : at::Tensor()});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)weight.scalar_type(),
                                                    bias ? (int64_t)bias->scalar_type() : -1};
    return product(matrix_of(held.codes, held.scales, false), matrix_of(w.codes, w.scales, true), bias ? &*bias : nullptr, x,
                   x.scalar_type(), sizes);
  }
  static torch::autograd::variable_list backward(Context* ctx, const torch::autograd::variable_list& grads) {
    const bool again = at::GradMode::is_enabled();
    torch::autograd::variable_list r(3);
    if (!grads[0].defined()) return r;
    {
      at::NoGradGuard none;
      auto saved = ctx->get_saved_variables();
      const auto shape = ctx->saved_data["shape"].toIntVector(), types = ctx->saved_data["types"].toIntVector();
      const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = types[2] >= 0 && ctx->needs_input_grad(2);
      const at::Tensor rows = grads[0].dim() == 2 ? grads[0] : grads[0].flatten(0, -2);
      const at::Tensor dy = lies_in_rows(rows) ? rows : rows.contiguous();
      const Quantized g = quantized(dy, type_code(dy.scalar_type()), want_b, want_b ? (at::ScalarType)types[2] : at::kFloat);
      const csw_fp8_matrix along = matrix_of(g.codes, g.scales, false), across = matrix_of(g.codes, g.scales, true);
      const int64_t cols = shape.back();
      if (want_x) {
        as_kept(&saved[2], &saved[3], dy.size(1), cols, dy.device());
        r[0] = product(along, matrix_of(saved[2], saved[3], false), nullptr, dy, (at::ScalarType)types[0], shape);
      }
      if (want_w) {
        as_kept(&saved[0], &saved[1], dy.size(0), cols, dy.device());
        r[1] = product(across, matrix_of(saved[0], saved[1], false), nullptr, dy, (at::ScalarType)types[1], {dy.size(1), cols});
      }
      if (want_b) r[2] = g.sums;
    }
    if (again) {  // a gradient of these gradients is an error, where one is asked for
      for (at::Tensor& t : r)
        if (t.defined()) t.requires_grad_(true);
      r = (*std::make_shared<torch::autograd::DelayedError>("fp8_linear is differentiable once", (int64_t)r.size()))(std::move(r));
    }
    return r;
  }
};

bool layer_of(const at::Tensor* x, const at::Tensor* bias, int64_t in, int64_t outs, const at::Tensor& on) {
  int type;
  if (!require_values(*x, "x", &type) || !same_device(on, *x, "weight")) return false;
  if (x->dim() < 2 || x->size(-1) != in)
    return value_error("x needs two axes at least, and a weight of [out, in] for its last one");
  if (!bias) return true;
  if (!require_values(*bias, "bias", &type) || !same_device(*bias, *x, "bias")) return false;
  return (bias->dim() == 1 && bias->numel() == outs) || value_error("%s must hold one value for each row of the weight", "bias");
}
at::Tensor in_rows(const at::Tensor& t) { return lies_in_rows(t) ? t : t.contiguous(); }

// fp8_linear(x, weight, bias) -> y
PyObject* fp8_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* bias;
    int type;
    if (!arg_count(n, 3)) return nullptr;
    const at::Tensor* x = as_tensor(a[0], "x");
    const at::Tensor* w = x ? as_tensor(a[1], "weight") : nullptr;
    if (!w || !optional_tensor(a[2], "bias", &bias) || !require_values(*w, "weight", &type)) return nullptr;
    if (w->dim() != 2) {
      value_error("weight must be [out, in]");
      return nullptr;
    }
    if (!layer_of(x, bias, w->size(1), w->size(0), *w)) return nullptr;
    for (const at::Tensor* t : {x, w, bias})
      if (t && !capture_allows(*t)) return nullptr;
    at::Tensor y;
    {
      pybind11::gil_scoped_release free;
      y = Fp8Linear::apply(in_rows(*x), in_rows(*w), bias ? std::optional<at::Tensor>(bias->contiguous()) : std::nullopt);
    }
    return THPVariable_Wrap(y);
  });
}

// fp8_linear_held(x, codes, scales, bias) -> y
PyObject* fp8_linear_held(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *codes, *bias;
    csw_fp8_matrix m;
    if (!arg_count(n, 4)) return nullptr;
    const at::Tensor* x = as_tensor(a[0], "x");
    if (!x || !optional_tensor(a[3], "bias", &bias) || !matrix_of(a[1], a[2], "weight", "scales", &codes, &m) ||
        !layer_of(x, bias, codes->size(1), codes->size(0), *codes))
      return nullptr;
    if (at::GradMode::is_enabled() && (x->requires_grad() || (bias && bias->requires_grad()))) {
      value_error("no gradient passes through a weight that was quantized before: call under torch.no_grad()");
      return nullptr;
    }
    at::Tensor y;
    {
      pybind11::gil_scoped_release free;
      const at::Tensor rows = in_rows(*x), b = bias ? bias->contiguous() : at::Tensor();
      const c10::cuda::CUDAGuard on(rows.device());
      std::vector<int64_t> sizes = x->sizes().vec();
      sizes.back() = codes->size(0);
      int64_t count = 1;
      for (size_t i = 0; i + 1 < sizes.size(); ++i) count *= sizes[i];
      size_t need;
      require_ok(csw_fp8_linear_workspace(count, m.cols, m.rows, &need), "csw_fp8_linear_workspace");
      at::Tensor space = need ? fresh(rows, {(int64_t)need}, at::kByte) : at::Tensor();
      y = fresh(rows, sizes, rows.scalar_type());
      const int type = type_code(rows.scalar_type());
      require_ok(csw_fp8_linear(ptr(rows), type, count, rows.is_contiguous() ? m.cols : rows.stride(0), &m,
                                bias ? ptr(b) : nullptr, bias ? type_code(b.scalar_type()) : 0, out(y), type,
                                need ? out(space) : nullptr, need, c10::cuda::getCurrentCUDAStream(rows.device().index()).stream()),
                 "csw_fp8_linear");
    }
    return THPVariable_Wrap(y);
  });
}

// ---- the optimizer's step ------------------------------------------------------------------------------------------
// The tensors of a list, a tuple or anything else that can be gone through, once: it lives until the launch, since what it was
// made of may hold its tensors no longer.  What they are checked for is their caller's.
struct List {
  THPObjectPtr fast;
  Py_ssize_t size = 0;
  bool of(PyObject* o) {
    fast = PySequence_Fast(o, "a list of tensors is wanted");
    if (!fast) return false;
    size = PySequence_Fast_GET_SIZE(fast.get());
    return true;
  }
  PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(fast.get(), i); }
};
bool same_size(const List& l, Py_ssize_t n, const char* name) {
  return l.size == n || value_error("%s must have an entry for each parameter", name);
}

// What is written by a call, apart: a range for each tensor, by its role.  And what is read, which may lie where nothing is
// written, or be the very tensor that its own entry of the lists writes: a value is read by the thread that writes it, before.
struct Written {
  struct Range {
    const char *begin, *end;
    size_t entry;
    bool operator<(const Range& o) const { return begin < o.begin; }
  };
  static constexpr size_t kMost = 7;  // roles, what is read among them
  struct Role {
    Range* first;
    size_t size;
  };
  std::unique_ptr<Range[]> space;
  Role roles[kMost];
  size_t count;  // of those that are written; the one behind them is read
  explicit Written(size_t written) : count(written) {}
  // for lists of so many entries, each of which reads `reads` tensors
  void room_for(size_t entries, size_t reads) {
    space.reset(new Range[(count + reads) * entries]);
    for (size_t i = 0; i <= count; ++i) roles[i] = {space.get() + i * entries, 0};
  }
  void add(size_t role, const void* p, size_t bytes, size_t entry) {
    const char* begin = static_cast<const char*>(p);
    if (bytes) roles[role].first[roles[role].size++] = {begin, begin + bytes, entry};
  }
  void add_read(const void* p, size_t bytes, size_t entry) { add(count, p, bytes, entry); }
  static bool ascend(const Range* r, size_t n) {
    for (size_t i = 1; i < n; ++i)
      if (r[i].begin < r[i - 1].end) return false;
    return true;
  }
  // Most programs' tensors of one role ascend in memory, apart from those of the others: no need to sort them then.
  bool apart() {
    Range hulls[kMost];
    size_t n = 0;
    bool plain = true;
    for (size_t i = 0; i < count; ++i) {
      const Role& r = roles[i];
      plain = plain && ascend(r.first, r.size);
      if (r.size) hulls[n++] = {r.first[0].begin, r.first[r.size - 1].end, 0};
    }
    const Role& read = roles[count];
    if (read.size) {
      Range& hull = hulls[n++] = read.first[0];
      for (size_t i = 1; i < read.size; ++i)
        hull.begin = std::min(hull.begin, read.first[i].begin), hull.end = std::max(hull.end, read.first[i].end);
    }
    std::sort(hulls, hulls + n);
    if (plain && ascend(hulls, n)) return true;
    std::vector<Range> all;
    for (size_t i = 0; i < count; ++i) all.insert(all.end(), roles[i].first, roles[i].first + roles[i].size);
    std::sort(all.begin(), all.end());
    if (!ascend(all.data(), all.size())) return value_error("the tensors that the step writes overlap");
    for (size_t i = 0; i < read.size; ++i) {
      const Range& r = read.first[i];
      auto w = std::partition_point(all.begin(), all.end(), [&](const Range& o) { return o.end <= r.begin; });
      for (; w != all.end() && w->begin < r.end; ++w)
        if (w->begin != r.begin || w->end != r.end || w->entry != r.entry)
          return value_error("a tensor that the step reads overlaps one that it writes");
    }
    return true;
  }
};
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// a tensor that lies as `as` does: the same shape and order in memory
bool lies_like(const at::Tensor& t, const at::Tensor& as, const char* name) {
  if (!same_device(t, as, name)) return false;
  if (!t.sizes().equals(as.sizes())) return value_error("%s has another shape than its parameter", name);
  if (t.is_contiguous() && as.is_contiguous()) return true;
  return t.strides().equals(as.strides()) || value_error("%s lies in another order than its parameter", name);
}
bool require_dense(const at::Tensor& t, const char* name) {
  return t.is_contiguous() || t.is_non_overlapping_and_dense() || value_error("%s must lie densely", name);
}
// codes (n) or scales (one for 128) of a state
bool bytes_of(const at::Tensor& t, const at::Tensor& on, int64_t n, const char* name) {
  if (!same_device(t, on, name)) return false;
  if (t.scalar_type() != at::kByte || t.numel() != n) return value_error("%s has another type or size than its parameter asks for", name);
  return require_flat(t, name);
}
// a state, whose tensors are written in four roles from `role` on, or read
bool eight_of(PyObject* o, const at::Tensor& on, csw_adamw_tensor* t, Written* written, bool write, size_t role, size_t entry,
              std::vector<List>* kept) {
  List l;
  if (!l.of(o)) return false;
  if (l.size != 4) return value_error("a state is (exp_avg, exp_avg_sq, their scales)");
  void** const to[4] = {&t->exp_avg, &t->exp_avg_sq, &t->exp_avg_scale, &t->exp_avg_sq_scale};
  const int64_t n = on.numel();
  for (int i = 0; i < 4; ++i) {
    const at::Tensor* s = as_tensor(l[i], "a state");
    if (!s || !bytes_of(*s, on, i < 2 ? n : blocks_of(n), "a state")) return false;
    *to[i] = ptr(*s);
    const size_t bytes = i < 2 ? n : blocks_of(n);
    if (write) {
      written->add(role + i, *to[i], bytes, entry);
      changed(*s);
    } else {
      written->add_read(*to[i], bytes, entry);
    }
  }
  if (l.fast.get() != o) kept->push_back(std::move(l));
  return true;
}
bool floats_of(PyObject* o, const at::Tensor& as, const char* name, const at::Tensor** t) {
  *t = as_tensor(o, name);
  if (!*t || !lies_like(**t, as, name)) return false;
  return (*t)->scalar_type() == at::kFloat || value_error("%s must be float32", name);
}
bool number(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  return !(*v == -1.0 && PyErr_Occurred());
}
// a number on the device that takes the place of one of the host's
bool on_device(const at::Tensor& t, const at::Tensor& on, at::ScalarType kind, const char* name, const void** p) {
  if (!same_device(t, on, name)) return false;
  if (t.scalar_type() != kind || t.numel() != 1)
    return value_error(kind == at::kLong ? "%s must be a number or one int64 on the device" : "%s must be a number or one float32 on the device", name);
  *p = t.const_data_ptr();
  return true;
}

// The tail of both steps' arguments: step, lr, beta1, beta2, eps, weight_decay, norm, max_norm
bool options_of(PyObject* const* a, const at::Tensor* on, csw_adamw_options* o) {
  double v[5];
  const void* p;
  if (THPVariable_Check(a[0])) {
    if (on && !on_device(THPVariable_Unpack(a[0]), *on, at::kLong, "step", &p)) return false;
    o->d_step = on ? static_cast<const int64_t*>(p) : nullptr;
    o->step = 1;
  } else {
    o->step = PyLong_AsLongLong(a[0]);
    if (o->step == -1 && PyErr_Occurred()) return false;
    if (o->step < 1) return value_error("step counts from 1");
  }
  if (THPVariable_Check(a[1])) {
    if (on && !on_device(THPVariable_Unpack(a[1]), *on, at::kFloat, "lr", &p)) return false;
    o->d_lr = on ? static_cast<const float*>(p) : nullptr;
    o->lr = 0.0;
  } else if (!number(a[1], &o->lr)) {
    return false;
  }
  for (int i = 0; i < 4; ++i)
    if (!number(a[2 + i], &v[i])) return false;
  o->beta1 = v[0], o->beta2 = v[1], o->eps = v[2], o->weight_decay = v[3];
  auto fine = [](double x) { return x >= 0.0 && x <= 3.4e38; };
  if (!fine(o->lr)) return value_error("lr must not be negative");
  for (int i = 0; i < 2; ++i)
    if (!(v[i] >= 0.0 && v[i] < 1.0)) return value_error("betas must be at least 0 and below 1");
  if (!fine(v[2])) return value_error("eps must not be negative");
  if (!fine(v[3])) return value_error("weight_decay must not be negative");
  o->max_norm = 0.0;
  if (a[6] != Py_None) {
    const at::Tensor* t = as_tensor(a[6], "norm");
    if (!t || !number(a[7], &o->max_norm)) return false;
    if (on && !on_device(*t, *on, at::kFloat, "norm", &p)) return false;
    o->d_norm = on ? static_cast<const float*>(p) : nullptr;
    if (!fine(o->max_norm)) return value_error("max_norm must not be negative");
  }
  return true;
}

// params, grads and copies (an empty list where there are none) of a call; the first parameter in *on
bool tensors_of(const List& params, PyObject* grads, PyObject* copies, List* grads_list, List* copies_list,
                std::vector<csw_adamw_tensor>* to, Written* written, const at::Tensor** on) {
  List &g = *grads_list, &c = *copies_list;
  if (!g.of(grads) || !same_size(g, params.size, "grads")) return false;
  const bool with_copies = copies != Py_None;
  if (with_copies && (!c.of(copies) || !same_size(c, params.size, "copies"))) return false;
  to->resize(params.size);
  written->room_for(params.size, 1);
  *on = nullptr;
  for (Py_ssize_t i = 0; i < params.size; ++i) {
    csw_adamw_tensor& t = (*to)[i];
    const at::Tensor* p = as_tensor(params[i], "a parameter");
    const at::Tensor* d = p ? as_tensor(g[i], "a gradient") : nullptr;
    if (!d || !require_values(*p, "a parameter", &t.param_type) || !require_dense(*p, "a parameter") ||
        !require_values(*d, "a gradient", &t.grad_type) || !lies_like(*d, *p, "a gradient"))
      return false;
    if (!*on) *on = p;
    if (!same_device(*p, **on, "a parameter")) return false;
    t.param = ptr(*p), t.grad = ptr(*d), t.numel = (size_t)p->numel();
    written->add(0, t.param, t.numel * p->element_size(), i);
    written->add_read(t.grad, t.numel * d->element_size(), i);
    if (with_copies && c[i] != Py_None) {
      const at::Tensor* k = as_tensor(c[i], "a copy");
      if (!k || !require_values(*k, "a copy", &t.copy_type) || !lies_like(*k, *p, "a copy")) return false;
      t.copy = ptr(*k);
      written->add(1, t.copy, t.numel * k->element_size(), i);
    }
  }
  return true;
}
void all_changed(const List& params, const List& copies) {
  for (Py_ssize_t i = 0; i < params.size; ++i) changed(THPVariable_Unpack(params[i]));
  for (Py_ssize_t i = 0; i < copies.size; ++i)
    if (THPVariable_Check(copies[i])) changed(THPVariable_Unpack(copies[i]));
}

bool step_of(const std::vector<csw_adamw_tensor>& tensors, const csw_adamw_options& o, const at::Tensor* on) {
  return !on || launch(*on, "csw_adamw_step",
                       [&](csw_stream_t s) { return csw_adamw_step(tensors.data(), tensors.size(), &o, s); });
}

// adamw_step(params, grads, exp_avgs, exp_avg_sqs, copies, step, lr, beta1, beta2, eps, weight_decay, norm, max_norm) -> None
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    List params, g, c, m, v;
    std::vector<csw_adamw_tensor> tensors;
    Written written(4);
    const at::Tensor *on, *t;
    csw_adamw_options o{};
    o.bits = 32;
    if (!arg_count(n, 13) || !params.of(a[0]) || !tensors_of(params, a[1], a[4], &g, &c, &tensors, &written, &on) ||
        !m.of(a[2]) || !v.of(a[3]) || !same_size(m, params.size, "exp_avgs") ||
        !same_size(v, params.size, "exp_avg_sqs") || !options_of(a + 5, on, &o))
      return nullptr;
    for (Py_ssize_t i = 0; i < params.size; ++i) {
      const at::Tensor& p = THPVariable_Unpack(params[i]);
      if (!floats_of(m[i], p, "exp_avg", &t)) return nullptr;
      tensors[i].exp_avg = ptr(*t);
      written.add(2, tensors[i].exp_avg, 4 * tensors[i].numel, i);
      if (!floats_of(v[i], p, "exp_avg_sq", &t)) return nullptr;
      tensors[i].exp_avg_sq = ptr(*t);
      written.add(3, tensors[i].exp_avg_sq, 4 * tensors[i].numel, i);
    }
    if (!written.apart() || !step_of(tensors, o, on)) return nullptr;
    all_changed(params, c);
    for (Py_ssize_t i = 0; i < params.size; ++i) changed(THPVariable_Unpack(m[i])), changed(THPVariable_Unpack(v[i]));
    Py_RETURN_NONE;
  });
}

// adamw8_step(params, grads, states, copies, step, lr, beta1, beta2, eps, weight_decay, norm, max_norm, seed) -> None
PyObject* adamw8_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    List params, g, c, states;
    std::vector<List> kept;
    std::vector<csw_adamw_tensor> tensors;
    Written written(6);
    const at::Tensor* on;
    csw_adamw_options o{};
    o.bits = 8;
    if (!arg_count(n, 13) || !params.of(a[0]) || !tensors_of(params, a[1], a[3], &g, &c, &tensors, &written, &on) ||
        !states.of(a[2]) || !same_size(states, params.size, "states") || !options_of(a + 4, on, &o))
      return nullptr;
    const unsigned long long seed = PyLong_AsUnsignedLongLong(a[12]);
    if (PyErr_Occurred()) return nullptr;
    if (seed >> 32) {
      value_error("seed must be below 2^32");
      return nullptr;
    }
    o.seed = (uint32_t)seed;
    for (Py_ssize_t i = 0; i < params.size; ++i)
      if (!eight_of(states[i], THPVariable_Unpack(params[i]), &tensors[i], &written, true, 2, i, &kept)) return nullptr;
    if (!written.apart() || !step_of(tensors, o, on)) return nullptr;
    all_changed(params, c);
    Py_RETURN_NONE;
  });
}

// adamw8_convert(states, exp_avgs, exp_avg_sqs, pack) -> None
PyObject* adamw8_convert(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    List states, m, v;
    std::vector<List> kept;
    if (!arg_count(n, 4) || !states.of(a[0]) || !m.of(a[1]) || !v.of(a[2]) ||
        !same_size(m, states.size, "exp_avgs") || !same_size(v, states.size, "exp_avg_sqs"))
      return nullptr;
    const int pack = PyObject_IsTrue(a[3]);
    if (pack < 0) return nullptr;
    std::vector<csw_adamw_tensor> tensors(states.size);
    Written written(4);
    written.room_for(states.size, 4);
    const at::Tensor* on = nullptr;
    for (Py_ssize_t i = 0; i < states.size; ++i) {
      csw_adamw_tensor& t = tensors[i];
      const at::Tensor* first = as_tensor(m[i], "exp_avg");
      const at::Tensor* second;
      int type;
      if (!first || !require_values(*first, "exp_avg", &type) || !require_dense(*first, "exp_avg") ||
          !floats_of(m[i], *first, "exp_avg", &first) || !floats_of(v[i], *first, "exp_avg_sq", &second))
        return nullptr;
      if (!on) on = first;
      if (!same_device(*first, *on, "exp_avg") || !eight_of(states[i], *first, &t, &written, pack, 0, i, &kept))
        return nullptr;
      t.param = ptr(*first), t.copy = ptr(*second), t.numel = (size_t)first->numel();
      if (pack) {
        written.add_read(t.param, 4 * t.numel, i), written.add_read(t.copy, 4 * t.numel, i);
      } else {
        written.add(0, t.param, 4 * t.numel, i), written.add(1, t.copy, 4 * t.numel, i);
        changed(*first), changed(*second);
      }
    }
    if (!written.apart()) return nullptr;
    if (on && !launch(*on, pack ? "csw_adamw8_pack" : "csw_adamw8_unpack", [&](csw_stream_t s) {
          return pack ? csw_adamw8_pack(tensors.data(), tensors.size(), s) : csw_adamw8_unpack(tensors.data(), tensors.size(), s);
        }))
      return nullptr;
    Py_RETURN_NONE;
  });
}

// gradient_norm(tensors) -> float32
PyObject* gradient_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    List grads;
    if (!arg_count(n, 1) || !grads.of(a[0])) return nullptr;
    if (grads.size == 0) {
      value_error("a norm needs a tensor at least");
      return nullptr;
    }
    std::vector<csw_adamw_tensor> tensors(grads.size);
    const at::Tensor* on = nullptr;
    for (Py_ssize_t i = 0; i < grads.size; ++i) {
      csw_adamw_tensor& t = tensors[i];
      const at::Tensor* g = as_tensor(grads[i], "a gradient");
      if (!g || !require_values(*g, "a gradient", &t.grad_type) || !require_dense(*g, "a gradient")) return nullptr;
      if (!on) on = g;
      if (!same_device(*g, *on, "a gradient")) return nullptr;
      t.grad = ptr(*g), t.numel = (size_t)g->numel();
    }
    const c10::cuda::CUDAGuard guard(on->device());  // the size goes by the device's SMs
    size_t need;
    if (!status_ok(csw_gradient_norm_workspace(tensors.data(), tensors.size(), &need), "csw_gradient_norm_workspace"))
      return nullptr;
    at::Tensor norm = fresh(*on, {}, at::kFloat), space = fresh(*on, {(int64_t)need}, at::kByte);
    float* to = static_cast<float*>(out(norm));
    void* ws = out(space);
    if (!launch(*on, "csw_gradient_norm",
                [&](csw_stream_t s) { return csw_gradient_norm(tensors.data(), tensors.size(), to, ws, need, s); }))
      return nullptr;
    return THPVariable_Wrap(norm);
  });
}

}  // namespace

PyMethodDef cswap_step_methods[] = {
    CSW_METHOD(fp8_quantize, "(x, sums) -> (codes, scales) or (codes, scales, sums)"),
    CSW_METHOD(fp8_dequantize, "(codes, scales, dtype) -> tensor"),
    CSW_METHOD(fp8_matmul, "(a, a_scales, b, b_scales, transpose_a, transpose_b, bias, dtype) -> tensor"),
    CSW_METHOD(fp8_linear, "(x, weight, bias) -> tensor"),
    CSW_METHOD(fp8_linear_held, "(x, codes, scales, bias) -> tensor"),
    CSW_METHOD(adamw_step, "(params, grads, exp_avgs, exp_avg_sqs, copies, step, lr, beta1, beta2, eps, weight_decay, norm, "
                           "max_norm) -> None"),
    CSW_METHOD(adamw8_step, "(params, grads, states, copies, step, lr, beta1, beta2, eps, weight_decay, norm, max_norm, seed) "
                            "-> None"),
    CSW_METHOD(adamw8_convert, "(states, exp_avgs, exp_avg_sqs, pack) -> None"),
    CSW_METHOD(gradient_norm, "(tensors) -> float32"),
    {nullptr, nullptr, 0, nullptr}};
