// 8-bit checkpoints of activations, and GELU with its input kept as one.
//
// The format: groups of 128 consecutive values (the last one may be shorter).  With m the group's largest magnitude,
// s = m / 127 and r = 127 / m, a value x is held as the integer q = rint(x * r), ties to even, and stands for q * s;
// every step is one correctly rounded float32 operation, so that any implementation of these lines gives the same
// codes.  A group whose m is below 2^-120, where 127 / m would overflow, is held as zeros (s = 0); a group with a NaN
// or an infinity has a NaN for its scale and stands for NaNs, so that a step that has diverged shows.
//
// What bounds these kernels: HBM.  A warp holds a group, four values a lane, so that the largest magnitude is one
// redux.sync over the bit patterns (whose order is that of the magnitudes, infinities and NaN above all numbers), and a
// warp's codes are one 128-byte line.  50331648 float32 values, cold: compressed in 47 us (5.3 TB/s of the 253 MB read and
// written), back in 39 (6.5); GELU with the checkpoint 76 us (6.0), its backward pass with the activation again 113 (5.8);
// 6.5 TB/s is what a plain copy reaches.
#include <cuda_runtime.h>

#include "../../include/cswap_b200.h"
#include "pdl.cuh"
#include "q8_kernels.h"
#include "values.cuh"

namespace csw {
namespace {

constexpr int kWarps = 8;

struct Group {
  float scale;
  char4 code;
};

__device__ __forceinline__ Group q8_encode(const float (&x)[4]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  const float m = __uint_as_float(top);
  Group g;
  float r = 0.0f;
  if (top >= 0x7f800000u) {
    g.scale = __uint_as_float(0x7fffffffu);
  } else if (m < 0x1p-120f) {
    g.scale = 0.0f;
  } else {
    g.scale = __fdiv_rn(m, 127.0f);
    r = __fdiv_rn(127.0f, m);
  }
  // an infinity or NaN times 0 converts to the code 0; |x * r| <= 127 (1 + 2^-23), which rounds to 127
  g.code = make_char4((signed char)__float2int_rn(__fmul_rn(x[0], r)), (signed char)__float2int_rn(__fmul_rn(x[1], r)),
                      (signed char)__float2int_rn(__fmul_rn(x[2], r)), (signed char)__float2int_rn(__fmul_rn(x[3], r)));
  return g;
}

__device__ __forceinline__ void q8_decode(char4 c, float s, float (&x)[4]) {
  x[0] = __fmul_rn((float)c.x, s), x[1] = __fmul_rn((float)c.y, s);
  x[2] = __fmul_rn((float)c.z, s), x[3] = __fmul_rn((float)c.w, s);
}

// four values from i on, of which those at n and behind read as zero
template <class T>
__device__ __forceinline__ void load4(const T* p, uint64_t i, uint64_t n, bool vec, float (&x)[4]) {
  if (vec && i + 4 <= n) {
    load_pack(p + i, x);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j < n ? widen(p[i + j]) : 0.0f;
  }
}
template <class T>
__device__ __forceinline__ void store4(T* p, uint64_t i, uint64_t n, bool vec, const float (&x)[4]) {
  if (vec && i + 4 <= n) {
    store_pack(p + i, x);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = narrow<T>(x[j]);
  }
}
__device__ __forceinline__ void store_codes(char4* codes, uint64_t i, uint64_t n, char4 c) {
  if (i + 4 <= n) {
    codes[i / 4] = c;
  } else {
    signed char* p = reinterpret_cast<signed char*>(codes);
    if (i < n) p[i] = c.x;
    if (i + 1 < n) p[i + 1] = c.y;
    if (i + 2 < n) p[i + 2] = c.z;
  }
}
__device__ __forceinline__ char4 load_codes(const char4* codes, uint64_t i, uint64_t n) {
  if (i + 4 <= n) return codes[i / 4];
  const signed char* p = reinterpret_cast<const signed char*>(codes);
  return make_char4(i < n ? p[i] : 0, i + 1 < n ? p[i + 1] : 0, i + 2 < n ? p[i + 2] : 0, 0);
}

// Phi, the distribution function of the normal distribution, and exp(-x^2 / 2), which its density is 1 / sqrt(2 pi) of.
// Phi(-z) = exp(-z^2 / 2) (c1 t + ... + c7 t^7) with t = 1 / (1 + 0.32 z), z >= 0: the form of Abramowitz and Stegun's
// 7.1.26, with two terms more and coefficients fitted for the least absolute error (6 10^-9; 2 10^-7 at most as float32
// rounds it).  The one exponential serves Phi and the density: some 20 instructions a value, where the library's
// function made a pass over 50331648 float32 values 133 us there and 165 back, bound by instructions.
struct Normal {
  float sum, bell;
};
__device__ __forceinline__ Normal normal(float x) {
  const float z = fabsf(x);
  float t, bell;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(z, 0.32f, 1.0f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(bell) : "f"(z * z * -0.72134752044f));
  float p = fmaf(0.04195379838347435f, t, -0.22253216803073883f);
  p = fmaf(p, t, 0.372079998254776f);
  p = fmaf(p, t, -0.12819476425647736f);
  p = fmaf(p, t, 0.19610773026943207f);
  p = fmaf(p, t, 0.11168046295642853f);
  p = fmaf(p, t, 0.12890493869781494f);
  const float below = p * t * bell;
  return {x > 0.0f ? 1.0f - below : below, bell};
}
constexpr float kDensity = 0.3989422804014327f;  // 1 / sqrt(2 pi)

// U groups a warp.  kGelu: y = x Phi(x) is written as well.
template <class T, int U, bool kGelu>
__global__ void __launch_bounds__(32 * kWarps) q8_encode_kernel(const T* __restrict__ x, uint64_t n, bool vec,
                                                                T* __restrict__ y, char4* __restrict__ codes,
                                                                float* __restrict__ scales) {
  pdl_wait(x);
  const uint64_t groups = (n + kQ8Group - 1) / kQ8Group;
  const uint64_t g0 = ((uint64_t)blockIdx.x * kWarps + threadIdx.x / 32) * U;
  const uint32_t lane = threadIdx.x % 32;
  float v[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) load4(x, (g0 + u) * kQ8Group + 4 * lane, n, vec, v[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = (g0 + u) * kQ8Group + 4 * lane;
    const Group g = q8_encode(v[u]);
    store_codes(codes, i, n, g.code);
    if (lane == 0 && g0 + u < groups) scales[g0 + u] = g.scale;
    if (kGelu) {
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = v[u][j] * normal(v[u][j]).sum;
      store4(y, i, n, vec, o);
    }
  }
}

// The codes of U groups a warp and, for kGelu, the gradient behind: without kGelu `out` receives the values; with it
// dx = dy (Phi(x) + x phi(x)) and, where `again` is given, x Phi(x).
template <class T, int U, bool kGelu>
__global__ void __launch_bounds__(32 * kWarps)
    q8_decode_kernel(const char4* __restrict__ codes, const float* __restrict__ scales, uint64_t n, bool vec,
                     const T* __restrict__ dy, T* __restrict__ out, T* __restrict__ again) {
  pdl_wait(codes);
  pdl_behind(scales, dy);
  const uint64_t groups = (n + kQ8Group - 1) / kQ8Group;
  const uint64_t g0 = ((uint64_t)blockIdx.x * kWarps + threadIdx.x / 32) * U;
  const uint32_t lane = threadIdx.x % 32;
  char4 c[U];
  float s[U], d[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = (g0 + u) * kQ8Group + 4 * lane;
    c[u] = load_codes(codes, i, n);
    s[u] = g0 + u < groups ? scales[g0 + u] : 0.0f;
    if (kGelu) load4(dy, i, n, vec, d[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = (g0 + u) * kQ8Group + 4 * lane;
    float x[4];
    q8_decode(c[u], s[u], x);
    if (!kGelu) {
      store4(out, i, n, vec, x);
    } else {
      float o[4], a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Normal f = normal(x[j]);
        a[j] = x[j] * f.sum;
        o[j] = d[u][j] * fmaf(x[j] * kDensity, f.bell, f.sum);
      }
      store4(out, i, n, vec, o);
      if (again) store4(again, i, n, vec, a);
    }
  }
}

template <class T>
bool aligned4(const void* p) {
  return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0;
}
unsigned blocks_for(uint64_t n, int per_warp) {
  return (unsigned)((q8_groups(n) + kWarps * per_warp - 1) / (kWarps * per_warp));
}
float* scales_of(void* packed, uint64_t n) { return reinterpret_cast<float*>((char*)packed + q8_scales_at(n)); }

// Four groups a warp keep four loads in flight; below that many values a warp takes one, to spread over the SMs
// (59136 bfloat16 values: 462 warps, where four groups a warp would leave 33 of 148 SMs with any).
constexpr uint64_t kSpread = 1 << 20;

template <class T, bool kGelu>
cudaError_t encode(const void* x, uint64_t n, void* y, void* packed, cudaStream_t stream) {
  const bool vec = aligned4<T>(x) && (!kGelu || aligned4<T>(y));
  const bool wide = n >= kSpread;
  return pdl_launch(wide ? q8_encode_kernel<T, 4, kGelu> : q8_encode_kernel<T, 1, kGelu>, blocks_for(n, wide ? 4 : 1),
                    32 * kWarps, 0, stream, (const T*)x, n, vec, (T*)y, (char4*)packed, scales_of(packed, n));
}
template <class T, bool kGelu>
cudaError_t decode(const void* packed, uint64_t n, const void* dy, void* out, void* again, cudaStream_t stream) {
  const bool vec = aligned4<T>(out) && (!dy || aligned4<T>(dy)) && (!again || aligned4<T>(again));
  const bool wide = n >= kSpread;
  return pdl_launch(wide ? q8_decode_kernel<T, 4, kGelu> : q8_decode_kernel<T, 1, kGelu>, blocks_for(n, wide ? 4 : 1),
                    32 * kWarps, 0, stream, (const char4*)packed, (const float*)scales_of((void*)packed, n), n, vec,
                    (const T*)dy, (T*)out, (T*)again);
}

}  // namespace

cudaError_t q8_compress_launch(const void* x, int type, uint64_t n, void* packed, cudaStream_t stream) {
  cudaError_t e = cudaErrorInvalidValue;
  if (n == 0) return cudaSuccess;
  with_type(type, [&](auto t) { e = encode<decltype(t), false>(x, n, nullptr, packed, stream); });
  return e;
}
cudaError_t q8_decompress_launch(const void* packed, uint64_t n, void* out, int type, cudaStream_t stream) {
  cudaError_t e = cudaErrorInvalidValue;
  if (n == 0) return cudaSuccess;
  with_type(type, [&](auto t) { e = decode<decltype(t), false>(packed, n, nullptr, out, nullptr, stream); });
  return e;
}
cudaError_t gelu_forward_launch(const void* x, int type, uint64_t n, void* y, void* packed, cudaStream_t stream) {
  cudaError_t e = cudaErrorInvalidValue;
  if (n == 0) return cudaSuccess;
  with_type(type, [&](auto t) { e = encode<decltype(t), true>(x, n, y, packed, stream); });
  return e;
}
cudaError_t gelu_backward_launch(const void* dy, int type, const void* packed, uint64_t n, void* dx, void* again,
                                 cudaStream_t stream) {
  cudaError_t e = cudaErrorInvalidValue;
  if (n == 0) return cudaSuccess;
  with_type(type, [&](auto t) { e = decode<decltype(t), true>(packed, n, dy, dx, again, stream); });
  return e;
}

}  // namespace csw
