// Attention, forward and backward.  With a query row q_i, the keys j it may see, and scale c:
//
//   s_j = c q_i.k_j,  L_i = log sum exp s_j,  p_j = exp(s_j - L_i),  o_i = sum p_j v_j
//   D_i = do_i.o_i,  ds_j = p_j (do_i.v_j - D_i)
//   dq_i = c sum ds_j k_j,  dk_j = c sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// Only L is kept for backward, which forms the probabilities again.  A row that sees no key has o = 0, L = -inf and
// takes part in no gradient.
//
// One warp a row, lanes along the head's dimension.
#include <cuda_runtime.h>

#include "attention_kernels.h"
#include "pdl.cuh"
#include "values.cuh"

namespace csw {
namespace {

constexpr int kWarps = 8;
constexpr int kPer = 4;  // values of a head of up to 128 that a lane holds

struct View {
  void* p;
  int64_t b, h, t;
  template <class T>
  __device__ T* row(uint64_t batch, uint64_t head, uint64_t token) const {
    return static_cast<T*>(p) + (int64_t)batch * b + (int64_t)head * h + (int64_t)token * t;
  }
};
View view_of(const csw_attention_operand& o) { return {o.data, o.batch_stride, o.head_stride, o.token_stride}; }

struct Shape {
  uint32_t batch, heads, kv_heads, q_len, k_len, dim;
  int causal;
  float scale;
  const int32_t* lens;
  __device__ uint32_t keys(uint32_t b) const {
    return lens ? (uint32_t)min(max(lens[b], 0), (int)k_len) : k_len;
  }
};
Shape shape_of(const csw_attention_shape& s) {
  return {(uint32_t)s.batch, (uint32_t)s.heads, (uint32_t)s.kv_heads, (uint32_t)s.q_len, (uint32_t)s.k_len,
          (uint32_t)s.dim,   s.causal,          s.scale,               s.kv_lens};
}

template <class T>
__device__ __forceinline__ void load_row(const T* p, uint32_t dim, uint32_t lane, float (&f)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) f[i] = lane + 32 * i < dim ? widen(p[lane + 32 * i]) : 0.0f;
}
template <class T>
__device__ __forceinline__ void store_row(T* p, uint32_t dim, uint32_t lane, const float (&f)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 32 * i < dim) p[lane + 32 * i] = narrow<T>(f[i]);
}
__device__ __forceinline__ float dot(const float (&a)[kPer], const float (&b)[kPer]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) s += a[i] * b[i];
#pragma unroll
  for (int d = 16; d; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
  return s;
}

template <class T>
__global__ void __launch_bounds__(32 * kWarps) attention_forward_kernel(Shape s, View q, View k, View v, View o, float* lse) {
  pdl_wait();
  const uint64_t r = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const uint32_t lane = threadIdx.x % 32;
  if (r >= (uint64_t)s.batch * s.heads * s.q_len) return;
  const uint32_t i = r % s.q_len, h = r / s.q_len % s.heads, b = r / s.q_len / s.heads, g = h / (s.heads / s.kv_heads);
  int64_t n = s.keys(b);
  if (s.causal) n = min(n, (int64_t)i + s.k_len - s.q_len + 1);
  float a[kPer], acc[kPer] = {}, top = -INFINITY, sum = 0.0f;
  load_row(q.row<T>(b, h, i), s.dim, lane, a);
  for (int64_t j = 0; j < n; ++j) {
    float kk[kPer], vv[kPer];
    load_row(k.row<T>(b, g, j), s.dim, lane, kk);
    load_row(v.row<T>(b, g, j), s.dim, lane, vv);
    const float x = dot(a, kk) * s.scale;
    const float m = fmaxf(top, x);
    const float f = top == m ? 1.0f : expf(top - m), p = x == m ? 1.0f : expf(x - m);
    top = m;
    sum = sum * f + p;
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] = acc[c] * f + p * vv[c];
  }
#pragma unroll
  for (int c = 0; c < kPer; ++c) acc[c] = n > 0 ? acc[c] / sum : 0.0f;
  store_row(o.row<T>(b, h, i), s.dim, lane, acc);
  if (lane == 0) lse[r] = n > 0 ? top + logf(sum) : -INFINITY;
}

// dq, and D for the other kernel
template <class T>
__global__ void __launch_bounds__(32 * kWarps)
    attention_dq_kernel(Shape s, View q, View k, View v, View o, View dout, const float* lse, View dq, float* delta) {
  pdl_wait();
  const uint64_t r = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const uint32_t lane = threadIdx.x % 32;
  if (r >= (uint64_t)s.batch * s.heads * s.q_len) return;
  const uint32_t i = r % s.q_len, h = r / s.q_len % s.heads, b = r / s.q_len / s.heads, g = h / (s.heads / s.kv_heads);
  int64_t n = s.keys(b);
  if (s.causal) n = min(n, (int64_t)i + s.k_len - s.q_len + 1);
  float a[kPer], out[kPer], d[kPer], acc[kPer] = {};
  load_row(q.row<T>(b, h, i), s.dim, lane, a);
  load_row(o.row<T>(b, h, i), s.dim, lane, out);
  load_row(dout.row<T>(b, h, i), s.dim, lane, d);
  const float D = dot(out, d), L = lse[r];
  if (lane == 0) delta[r] = D;
  for (int64_t j = 0; j < n; ++j) {
    float kk[kPer], vv[kPer];
    load_row(k.row<T>(b, g, j), s.dim, lane, kk);
    load_row(v.row<T>(b, g, j), s.dim, lane, vv);
    const float p = expf(dot(a, kk) * s.scale - L);
    const float ds = p * (dot(d, vv) - D) * s.scale;
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] += ds * kk[c];
  }
  store_row(dq.row<T>(b, h, i), s.dim, lane, acc);
}

template <class T>
__global__ void __launch_bounds__(32 * kWarps) attention_dkv_kernel(Shape s, View q, View k, View v, View dout,
                                                                    const float* lse, const float* delta, View dk,
                                                                    View dv) {
  pdl_wait();
  const uint64_t r = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const uint32_t lane = threadIdx.x % 32;
  if (r >= (uint64_t)s.batch * s.kv_heads * s.k_len) return;
  const uint32_t j = r % s.k_len, g = r / s.k_len % s.kv_heads, b = r / s.k_len / s.kv_heads;
  const uint32_t share = s.heads / s.kv_heads;
  float kk[kPer], vv[kPer], ak[kPer] = {}, av[kPer] = {};
  load_row(k.row<T>(b, g, j), s.dim, lane, kk);
  load_row(v.row<T>(b, g, j), s.dim, lane, vv);
  int64_t first = j < s.keys(b) ? 0 : s.q_len;
  if (s.causal) first = max(first, (int64_t)j - s.k_len + s.q_len);
  for (uint32_t h = g * share; h < (g + 1) * share; ++h) {
    for (int64_t i = first; i < s.q_len; ++i) {
      float a[kPer], d[kPer];
      load_row(q.row<T>(b, h, i), s.dim, lane, a);
      load_row(dout.row<T>(b, h, i), s.dim, lane, d);
      const uint64_t at = ((uint64_t)b * s.heads + h) * s.q_len + i;
      const float p = expf(dot(a, kk) * s.scale - lse[at]);
      const float ds = p * (dot(d, vv) - delta[at]) * s.scale;
#pragma unroll
      for (int c = 0; c < kPer; ++c) ak[c] += ds * a[c], av[c] += p * d[c];
    }
  }
  store_row(dk.row<T>(b, g, j), s.dim, lane, ak);
  store_row(dv.row<T>(b, g, j), s.dim, lane, av);
}

unsigned blocks_for(uint64_t rows) { return (unsigned)((rows + kWarps - 1) / kWarps); }

}  // namespace

cudaError_t attention_forward_launch(const csw_attention_shape& s, const csw_attention_operand& q,
                                     const csw_attention_operand& k, const csw_attention_operand& v,
                                     const csw_attention_operand& o, float* lse, cudaStream_t stream) {
  const uint64_t rows = (uint64_t)s.batch * s.heads * s.q_len;
  if (rows == 0) return cudaSuccess;
  const auto kernel = s.type == CSW_TYPE_F16 ? attention_forward_kernel<__half> : attention_forward_kernel<__nv_bfloat16>;
  return pdl_launch(kernel, blocks_for(rows), 32 * kWarps, 0, stream, shape_of(s), view_of(q), view_of(k), view_of(v),
                    view_of(o), lse);
}

cudaError_t attention_backward_launch(const csw_attention_shape& s, const AttentionBackward& a, cudaStream_t stream) {
  const uint64_t q_rows = (uint64_t)s.batch * s.heads * s.q_len, k_rows = (uint64_t)s.batch * s.kv_heads * s.k_len;
  cudaError_t e = cudaSuccess;
  const bool half = s.type == CSW_TYPE_F16;
  if (q_rows)
    e = pdl_launch(half ? attention_dq_kernel<__half> : attention_dq_kernel<__nv_bfloat16>, blocks_for(q_rows),
                   32 * kWarps, 0, stream, shape_of(s), view_of(a.q), view_of(a.k), view_of(a.v), view_of(a.o),
                   view_of(a.dout), a.lse, view_of(a.dq), a.delta);
  if (e == cudaSuccess && k_rows)
    e = pdl_launch(half ? attention_dkv_kernel<__half> : attention_dkv_kernel<__nv_bfloat16>, blocks_for(k_rows),
                   32 * kWarps, 0, stream, shape_of(s), view_of(a.q), view_of(a.k), view_of(a.v), view_of(a.dout),
                   a.lse, (const float*)a.delta, view_of(a.dk), view_of(a.dv));
  return e;
}

}  // namespace csw
