// C ABI of the training operators: argument checking.  Declarations: include/cswap_b200.h, sections 7 to 9.
#include <cuda_runtime.h>

#include "../../include/cswap_b200.h"
#include "attention_kernels.h"
#include "fp8_kernels.h"
#include "internal.h"
#include "norm_kernels.h"
#include "optim_kernels.h"
#include "pdl.cuh"
#include "q8_kernels.h"
#include "waits.h"

using namespace csw;

namespace {

constexpr size_t kMostValues = (size_t)1 << 42;  // grids of 2^31 - 1 blocks are far off, sizes in bytes do not wrap
constexpr size_t kMostRows = ((size_t)1 << 31) - 1;

csw_status done(cudaError_t e) { return e == cudaSuccess ? CSW_OK : cuda_fail(e); }
bool known_type(int t) { return t == CSW_TYPE_F32 || t == CSW_TYPE_F16 || t == CSW_TYPE_BF16; }
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
size_t size_of(int t) { return t == CSW_TYPE_F32 ? 4 : 2; }
// a value's address is a multiple of its size
bool good(const void* p, int type) { return p && aligned(p, size_of(type)); }

csw_status packed_fits(const void* packed, size_t bytes, size_t n) {
  size_t need;
  if (csw_q8_bytes(n, &need) != CSW_OK) return CSW_ERR_ARG;
  if (n && (!packed || !aligned(packed, 16))) return CSW_ERR_ARG;
  return bytes < need ? CSW_ERR_SIZE : CSW_OK;
}

bool norm_args(int type, int param_type, size_t rows, size_t cols) {
  return known_type(type) && (param_type == type || param_type == CSW_TYPE_F32) && rows <= kMostRows && cols > 0 &&
         cols <= kMostRows && (rows == 0 || cols <= kMostValues / rows);
}

// whether the operand can be addressed and, if its rows are copied as tiles, lies as a tile copy needs it
bool operand(const csw_attention_operand* o, const csw_attention_shape* s, size_t heads, size_t tokens) {
  if (!o) return false;
  if (s->batch == 0 || tokens == 0) return true;
  // the stride of an axis of one step is not used
  auto strides = [](ptrdiff_t stride, size_t n) { return n < 2 || (stride > 0 && stride % 8 == 0); };
  return o->data && aligned(o->data, 16) && strides(o->batch_stride, s->batch) && strides(o->head_stride, heads) &&
         strides(o->token_stride, tokens);
}
bool attention_args(const csw_attention_shape* s) {
  if (!s || (s->type != CSW_TYPE_F16 && s->type != CSW_TYPE_BF16)) return false;
  constexpr size_t kMost = (size_t)1 << 29;  // sums of positions stay below 2^31
  if (s->batch > 65535 || s->heads > 65535 || s->q_len > kMost || s->k_len > kMost) return false;
  if (s->dim == 0 || s->dim > 128 || s->dim % 8) return false;
  if (s->kv_heads == 0 || s->heads % s->kv_heads) return false;
  if (s->heads == 0) return false;
  const size_t rows = s->batch * s->heads;  // below 2^32
  if (rows && ((s->q_len + 127) / 128 > kMostRows / rows || (s->k_len + 127) / 128 > kMostRows / rows)) return false;
  return s->kv_lens == nullptr || aligned(s->kv_lens, 4);
}
// An earlier call's kernel that gave up on a wait is told here, to a call that has something to launch.
csw_status before_waits() {
  int gave_up = 0;
  const csw_status st = done(take_status(&gave_up));
  return st != CSW_OK ? st : gave_up ? CSW_ERR_TIMEOUT : CSW_OK;
}

// codes and scales of a matrix, as the kernels can address them
bool matrix(const void* codes, const void* scales, size_t rows, size_t cols, size_t stride) {
  if (rows > kMostRows || cols > kMostRows) return false;
  if (rows == 0 || cols == 0) return true;
  if (fp8_blocks(rows) > kMostRows / fp8_blocks(cols)) return false;
  return codes && scales && aligned(codes, 16) && stride % 16 == 0 && stride >= cols && stride <= ((size_t)1 << 39) && stride <= kMostValues / rows;
}

constexpr size_t kMostOfTensor = (size_t)1 << 41, kMostTensors = (size_t)1 << 24;
bool adamw_list(const csw_adamw_tensor* t, size_t count) {
  if (count > kMostTensors || (count && !t)) return false;
  for (size_t i = 0; i < count; ++i)
    if (t[i].numel > kMostOfTensor) return false;
  return true;
}
// the state of a tensor in so many bits
bool adamw_state(const csw_adamw_tensor& t, int bits) {
  if (bits == 8) return t.exp_avg && t.exp_avg_sq && t.exp_avg_scale && t.exp_avg_sq_scale;
  return good(t.exp_avg, CSW_TYPE_F32) && good(t.exp_avg_sq, CSW_TYPE_F32) && !t.exp_avg_scale && !t.exp_avg_sq_scale;
}
csw_status adamw8_convert(const csw_adamw_tensor* t, size_t count, bool pack, csw_stream_t stream) {
  if (!adamw_list(t, count)) return CSW_ERR_ARG;
  for (size_t i = 0; i < count; ++i)
    if (t[i].numel && (!adamw_state(t[i], 8) || t[i].param_type != CSW_TYPE_F32 || t[i].copy_type != CSW_TYPE_F32 ||
                       !good(t[i].param, CSW_TYPE_F32) || !good(t[i].copy, CSW_TYPE_F32)))
      return CSW_ERR_ARG;
  return done(adamw8_convert_launch(t, count, pack, stream));
}
bool gradients(const csw_adamw_tensor* t, size_t count) {
  if (!adamw_list(t, count)) return false;
  for (size_t i = 0; i < count; ++i)
    if (t[i].numel && (!known_type(t[i].grad_type) || !good(t[i].grad, t[i].grad_type))) return false;
  return true;
}
// the rate, decay or epsilon of an optimizer; also not a NaN
bool rate(double v) { return v >= 0.0 && v <= 3.4e38; }

}  // namespace

extern "C" {

csw_status csw_q8_bytes(size_t n, size_t* bytes) {
  if (!bytes || n > kMostValues) return CSW_ERR_ARG;
  *bytes = q8_scales_at(n) + 4 * q8_groups(n);
  return CSW_OK;
}

csw_status csw_q8_compress(const void* d_in, int type, size_t n, void* d_out, size_t cap, csw_stream_t stream) {
  if (!known_type(type) || (n && !good(d_in, type))) return CSW_ERR_ARG;
  const csw_status st = packed_fits(d_out, cap, n);
  return st != CSW_OK ? st : done(q8_compress_launch(d_in, type, n, d_out, stream));
}

csw_status csw_q8_decompress(const void* d_in, size_t bytes, size_t n, void* d_out, int type, csw_stream_t stream) {
  if (!known_type(type) || (n && !good(d_out, type))) return CSW_ERR_ARG;
  const csw_status st = packed_fits(d_in, bytes, n);
  return st != CSW_OK ? st : done(q8_decompress_launch(d_in, n, d_out, type, stream));
}

csw_status csw_gelu_forward(const void* d_x, int type, size_t n, void* d_y, void* d_packed, size_t cap,
                            csw_stream_t stream) {
  if (!known_type(type) || (n && (!good(d_x, type) || !good(d_y, type)))) return CSW_ERR_ARG;
  const csw_status st = packed_fits(d_packed, cap, n);
  return st != CSW_OK ? st : done(gelu_forward_launch(d_x, type, n, d_y, d_packed, stream));
}

csw_status csw_gelu_backward(const void* d_dy, int type, const void* d_packed, size_t bytes, size_t n, void* d_dx,
                             void* d_y, csw_stream_t stream) {
  if (!known_type(type) || (n && (!good(d_dy, type) || !good(d_dx, type)))) return CSW_ERR_ARG;
  if (d_y && !good(d_y, type)) return CSW_ERR_ARG;
  const csw_status st = packed_fits(d_packed, bytes, n);
  return st != CSW_OK ? st : done(gelu_backward_launch(d_dy, type, d_packed, n, d_dx, d_y, stream));
}

csw_status csw_layer_norm_forward(const void* d_x, const void* d_residual, const void* d_weight, const void* d_bias,
                                  int type, int param_type, size_t rows, size_t cols, float eps, void* d_y, void* d_sum,
                                  float* d_mean, float* d_rstd, csw_stream_t stream) {
  if (!norm_args(type, param_type, rows, cols)) return CSW_ERR_ARG;
  if (rows == 0) return CSW_OK;
  if (!good(d_x, type) || !good(d_y, type) || !good(d_mean, CSW_TYPE_F32) || !good(d_rstd, CSW_TYPE_F32))
    return CSW_ERR_ARG;
  if (d_residual && (!good(d_residual, type) || !good(d_sum, type))) return CSW_ERR_ARG;
  if (!aligned(d_weight, size_of(param_type)) || !aligned(d_bias, size_of(param_type))) return CSW_ERR_ARG;
  return done(norm_forward_launch({d_x, d_residual, d_weight, d_bias, d_y, d_residual ? d_sum : nullptr, d_mean, d_rstd,
                                   type, param_type, rows, cols, eps},
                                  stream));
}

csw_status csw_layer_norm_workspace(size_t rows, size_t cols, size_t* bytes) {
  if (!bytes || !norm_args(CSW_TYPE_F32, CSW_TYPE_F32, rows, cols)) return CSW_ERR_ARG;
  *bytes = norm_backward_partials(rows, cols) * 2 * cols * sizeof(float);
  return CSW_OK;
}

csw_status csw_layer_norm_backward(const void* d_dy, const void* d_x, const float* d_mean, const float* d_rstd,
                                   const void* d_weight, int type, int param_type, size_t rows, size_t cols, void* d_dx,
                                   void* d_dweight, void* d_dbias, void* d_workspace, size_t workspace_bytes,
                                   csw_stream_t stream) {
  size_t need;
  if (!norm_args(type, param_type, rows, cols) || csw_layer_norm_workspace(rows, cols, &need) != CSW_OK)
    return CSW_ERR_ARG;
  if (rows && (!good(d_dy, type) || !good(d_x, type) || !good(d_dx, type) || !good(d_mean, CSW_TYPE_F32) ||
               !good(d_rstd, CSW_TYPE_F32)))
    return CSW_ERR_ARG;
  for (const void* p : {d_weight, (const void*)d_dweight, (const void*)d_dbias})
    if (!aligned(p, size_of(param_type))) return CSW_ERR_ARG;
  const bool sums = d_dweight || d_dbias;
  if (sums && need && !good(d_workspace, CSW_TYPE_F32)) return CSW_ERR_ARG;
  if (sums && workspace_bytes < need) return CSW_ERR_SIZE;
  return done(norm_backward_launch({d_dy, d_x, d_mean, d_rstd, d_weight, d_dx, d_dweight, d_dbias, (float*)d_workspace,
                                    type, param_type, rows, cols},
                                   stream));
}

csw_status csw_attention_forward(const csw_attention_shape* shape, const csw_attention_operand* q,
                                 const csw_attention_operand* k, const csw_attention_operand* v,
                                 const csw_attention_operand* o, float* d_lse, csw_stream_t stream) {
  if (!attention_args(shape)) return CSW_ERR_ARG;
  const csw_attention_shape& s = *shape;
  if (!operand(q, shape, s.heads, s.q_len) || !operand(k, shape, s.kv_heads, s.k_len) ||
      !operand(v, shape, s.kv_heads, s.k_len) || !operand(o, shape, s.heads, s.q_len))
    return CSW_ERR_ARG;
  if (s.batch * s.q_len != 0 && !good(d_lse, CSW_TYPE_F32)) return CSW_ERR_ARG;
  const csw_status st = s.batch && s.q_len ? before_waits() : CSW_OK;
  return st != CSW_OK ? st : done(attention_forward_launch(s, *q, *k, *v, *o, d_lse, stream));
}

csw_status csw_attention_wait_limit(int64_t clocks) {
  if (clocks == INT64_MIN) return CSW_ERR_ARG;
  set_wait_limit(clocks);
  return CSW_OK;
}

csw_status csw_attention_workspace(const csw_attention_shape* shape, size_t* bytes) {
  if (!bytes || !attention_args(shape)) return CSW_ERR_ARG;
  *bytes = attention_workspace_values(*shape) * sizeof(float);
  return CSW_OK;
}

csw_status csw_attention_backward(const csw_attention_shape* shape, const csw_attention_operand* q,
                                  const csw_attention_operand* k, const csw_attention_operand* v,
                                  const csw_attention_operand* o, const float* d_lse, const csw_attention_operand* dout,
                                  const csw_attention_operand* dq, const csw_attention_operand* dk,
                                  const csw_attention_operand* dv, void* d_workspace, size_t workspace_bytes,
                                  csw_stream_t stream) {
  size_t need;
  if (csw_attention_workspace(shape, &need) != CSW_OK) return CSW_ERR_ARG;
  const csw_attention_shape& s = *shape;
  for (const csw_attention_operand* p : {q, o, dout, dq})
    if (!operand(p, shape, s.heads, s.q_len)) return CSW_ERR_ARG;
  for (const csw_attention_operand* p : {k, v, dk, dv})
    if (!operand(p, shape, s.kv_heads, s.k_len)) return CSW_ERR_ARG;
  if (need && (!good(d_lse, CSW_TYPE_F32) || !d_workspace || !aligned(d_workspace, 16))) return CSW_ERR_ARG;
  if (workspace_bytes < need) return CSW_ERR_SIZE;
  const csw_status st = s.batch && (s.q_len || s.k_len) ? before_waits() : CSW_OK;
  if (st != CSW_OK) return st;
  return done(attention_backward_launch(s, {*q, *k, *v, *o, *dout, *dq, *dk, *dv, d_lse, (float*)d_workspace}, stream));
}

csw_status csw_fp8_quantize_workspace(size_t rows, size_t cols, size_t* bytes) {
  if (!bytes || rows > kMostRows || cols > kMostRows || (rows && cols > kMostValues / rows)) return CSW_ERR_ARG;
  *bytes = rows > kFp8Block ? fp8_blocks(rows) * cols * sizeof(float) : 0;
  return CSW_OK;
}

csw_status csw_fp8_quantize(const void* d_x, int type, size_t rows, size_t cols, size_t x_stride, void* d_codes,
                            size_t code_stride, void* d_scales, void* d_sums, int sums_type, void* d_workspace,
                            size_t workspace_bytes, csw_stream_t stream) {
  size_t need;
  if (!known_type(type) || !matrix(d_codes, d_scales, rows, cols, code_stride) ||
      csw_fp8_quantize_workspace(rows, cols, &need) != CSW_OK)
    return CSW_ERR_ARG;
  if (rows && cols && (!good(d_x, type) || x_stride < cols || x_stride > kMostValues / rows)) return CSW_ERR_ARG;
  if (d_sums && (!known_type(sums_type) || !good(d_sums, sums_type))) return CSW_ERR_ARG;
  if (d_sums && need && !good(d_workspace, CSW_TYPE_F32)) return CSW_ERR_ARG;
  if (d_sums && workspace_bytes < need) return CSW_ERR_SIZE;
  return done(fp8_quantize_launch({d_x, type, rows, cols, x_stride, d_codes, code_stride, static_cast<uint8_t*>(d_scales),
                                   d_sums, sums_type, static_cast<float*>(d_workspace)},
                                  stream));
}

csw_status csw_fp8_dequantize(const void* d_codes, size_t code_stride, const void* d_scales, size_t rows, size_t cols,
                              void* d_out, int type, csw_stream_t stream) {
  if (!known_type(type) || !matrix(d_codes, d_scales, rows, cols, code_stride)) return CSW_ERR_ARG;
  if (rows && cols && !good(d_out, type)) return CSW_ERR_ARG;
  return done(fp8_dequantize_launch(d_codes, code_stride, static_cast<const uint8_t*>(d_scales), rows, cols, d_out, type,
                                    stream));
}

csw_status csw_fp8_matmul(const csw_fp8_matrix* a, const csw_fp8_matrix* b, const void* d_bias, int bias_type, void* d_out,
                          int type, csw_stream_t stream) {
  if (!a || !b || !known_type(type)) return CSW_ERR_ARG;
  for (const csw_fp8_matrix* m : {a, b})
    if (!matrix(m->codes, m->scales, m->rows, m->cols, m->code_stride)) return CSW_ERR_ARG;
  const size_t m = a->transposed ? a->cols : a->rows, k = a->transposed ? a->rows : a->cols;
  const size_t n = b->transposed ? b->rows : b->cols;
  if (k != (b->transposed ? b->cols : b->rows)) return CSW_ERR_ARG;
  if (m == 0 || n == 0) return CSW_OK;
  constexpr size_t kMost = kMostRows - 128;  // a tile's last row stays below 2^31
  if (m > kMost || n > kMost || fp8_blocks(m) > kMostRows / 32 / ((n + 31) / 32)) return CSW_ERR_ARG;
  if (!good(d_out, type)) return CSW_ERR_ARG;
  if (d_bias && (!known_type(bias_type) || !good(d_bias, bias_type))) return CSW_ERR_ARG;
  const csw_status st = before_waits();
  if (st != CSW_OK) return st;
  auto of = [](const csw_fp8_matrix& x) {
    return Fp8Matrix{x.codes, static_cast<const uint8_t*>(x.scales), x.rows, x.cols, x.code_stride, x.transposed != 0};
  };
  return done(fp8_matmul_launch(of(*a), of(*b), d_bias, bias_type, d_out, type, stream));
}

csw_status csw_fp8_linear_workspace(size_t rows, size_t cols, size_t outs, size_t* bytes) {
  if (!bytes || rows > kMostRows || cols > kMostRows || outs > kMostRows) return CSW_ERR_ARG;
  if (rows && (cols + 15 > kMostValues / rows || fp8_blocks(rows) > kMostRows / (fp8_blocks(cols) + 1))) return CSW_ERR_ARG;
  *bytes = rows == 0 || fp8_linear_at_once(rows, cols, outs) ? 0 : (cols + 15) / 16 * 16 * rows + fp8_blocks(rows) * fp8_blocks(cols);
  return CSW_OK;
}

csw_status csw_fp8_linear(const void* d_x, int type, size_t rows, size_t x_stride, const csw_fp8_matrix* weight,
                          const void* d_bias, int bias_type, void* d_out, int out_type, void* d_workspace,
                          size_t workspace_bytes, csw_stream_t stream) {
  if (!weight || !known_type(type) || !known_type(out_type) || weight->transposed) return CSW_ERR_ARG;
  const size_t outs = weight->rows, cols = weight->cols;
  size_t need;
  if (!matrix(weight->codes, weight->scales, outs, cols, weight->code_stride) ||
      csw_fp8_linear_workspace(rows, cols, outs, &need) != CSW_OK)
    return CSW_ERR_ARG;
  if (rows == 0 || outs == 0) return CSW_OK;
  constexpr size_t kMost = kMostRows - 128;
  if (rows > kMost || outs > kMost || fp8_blocks(rows) > kMostRows / 32 / ((outs + 31) / 32)) return CSW_ERR_ARG;
  if (cols && (!good(d_x, type) || x_stride < cols || x_stride > kMostValues / rows)) return CSW_ERR_ARG;
  if (!good(d_out, out_type) || (d_bias && (!known_type(bias_type) || !good(d_bias, bias_type)))) return CSW_ERR_ARG;
  if (need && (!d_workspace || !aligned(d_workspace, 16))) return CSW_ERR_ARG;
  if (workspace_bytes < need) return CSW_ERR_SIZE;
  const csw_status st = before_waits();
  if (st != CSW_OK) return st;
  const size_t stride = (cols + 15) / 16 * 16;
  return done(fp8_linear_launch({d_x, type, rows, cols, x_stride, d_workspace, stride,
                                 static_cast<uint8_t*>(d_workspace) + stride * rows, nullptr, 0, nullptr},
                                {weight->codes, static_cast<const uint8_t*>(weight->scales), outs, cols, weight->code_stride, true},
                                d_bias, bias_type, d_out, out_type, stream));
}

csw_status csw_adamw_step(const csw_adamw_tensor* tensors, size_t count, const csw_adamw_options* options,
                          csw_stream_t stream) {
  if (!options || (options->bits != 8 && options->bits != 32) || !gradients(tensors, count)) return CSW_ERR_ARG;
  const csw_adamw_options& o = *options;
  if (!rate(o.lr) || !rate(o.eps) || !rate(o.weight_decay) || !(o.beta1 >= 0.0 && o.beta1 < 1.0) ||
      !(o.beta2 >= 0.0 && o.beta2 < 1.0))
    return CSW_ERR_ARG;
  if (!o.d_step && o.step < 1) return CSW_ERR_ARG;
  if (!aligned(o.d_step, 8) || !aligned(o.d_lr, 4) || !aligned(o.d_norm, 4)) return CSW_ERR_ARG;
  if (o.d_norm && !rate(o.max_norm)) return CSW_ERR_ARG;
  for (size_t i = 0; i < count; ++i) {
    const csw_adamw_tensor& t = tensors[i];
    if (t.numel == 0) continue;
    if (!known_type(t.param_type) || !good(t.param, t.param_type) || !adamw_state(t, o.bits)) return CSW_ERR_ARG;
    if (t.copy && (!known_type(t.copy_type) || !good(t.copy, t.copy_type))) return CSW_ERR_ARG;
  }
  return done(adamw_launch(tensors, count, o, stream));
}

csw_status csw_adamw8_pack(const csw_adamw_tensor* tensors, size_t count, csw_stream_t stream) {
  return adamw8_convert(tensors, count, true, stream);
}
csw_status csw_adamw8_unpack(const csw_adamw_tensor* tensors, size_t count, csw_stream_t stream) {
  return adamw8_convert(tensors, count, false, stream);
}

csw_status csw_gradient_norm_workspace(const csw_adamw_tensor* tensors, size_t count, size_t* bytes) {
  if (!bytes || !adamw_list(tensors, count)) return CSW_ERR_ARG;
  *bytes = gradient_norm_partials(tensors, count) * sizeof(double);
  return CSW_OK;
}
csw_status csw_gradient_norm(const csw_adamw_tensor* tensors, size_t count, float* d_norm, void* d_workspace,
                             size_t workspace_bytes, csw_stream_t stream) {
  size_t need;
  if (!gradients(tensors, count) || !good(d_norm, CSW_TYPE_F32) ||
      csw_gradient_norm_workspace(tensors, count, &need) != CSW_OK)
    return CSW_ERR_ARG;
  if (need && (!d_workspace || !aligned(d_workspace, 8))) return CSW_ERR_ARG;
  if (workspace_bytes < need) return CSW_ERR_SIZE;
  return done(gradient_norm_launch(tensors, count, d_norm, static_cast<double*>(d_workspace), stream));
}

}  // extern "C"
