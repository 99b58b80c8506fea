// C ABI of the training operators: argument checking.  Declarations: include/cswap_b200.h, section 7.
#include <cuda_runtime.h>

#include "../../include/cswap_b200.h"
#include "attention_kernels.h"
#include "internal.h"
#include "norm_kernels.h"
#include "pdl.cuh"
#include "q8_kernels.h"

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
csw_status before_attention() {
  int gave_up = 0;
  const csw_status st = done(attention_take_status(&gave_up));
  return st != CSW_OK ? st : gave_up ? CSW_ERR_TIMEOUT : CSW_OK;
}

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
  const csw_status st = s.batch && s.q_len ? before_attention() : CSW_OK;
  return st != CSW_OK ? st : done(attention_forward_launch(s, *q, *k, *v, *o, d_lse, stream));
}

csw_status csw_attention_wait_limit(int64_t clocks) {
  if (clocks == INT64_MIN) return CSW_ERR_ARG;
  attention_wait_limit(clocks);
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
  const csw_status st = s.batch && (s.q_len || s.k_len) ? before_attention() : CSW_OK;
  if (st != CSW_OK) return st;
  return done(attention_backward_launch(s, {*q, *k, *v, *o, *dout, *dq, *dk, *dv, d_lse, (float*)d_workspace}, stream));
}

}  // extern "C"
