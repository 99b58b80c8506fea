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
// warp's codes are one 128-byte line.  Numbers become codes and back by adding powers of two, and a group's two divisions
// are made by one lane for all.  50331648 values, back to back: float32 compressed in 39 us (6.5 TB/s of what is read and
// written; a plain copy reaches as much), back in 40, GELU with the checkpoint 69, its backward pass with the activation
// again 98 (6.7); bfloat16 35, 27, 57 and 57 us (4.3 to 6.1 TB/s, bound by instructions and the loads in flight).
#include <cuda_runtime.h>

#include "../../include/cswap_b200.h"
#include "pdl.cuh"
#include "q8_kernels.h"
#include "values.cuh"

namespace csw {
namespace {

constexpr int kWarps = 8;

// 1.5 2^23: a number of up to 2^22 that it is added to is rounded to a whole one, ties to even, whose low byte is the
// sum's.  (The instructions that convert numbers share the unit of the exponentials, 16 a clock and SM.)
constexpr float kMagic = 12582912.0f;

// The largest magnitude's bits of a group that a warp holds.
__device__ __forceinline__ uint32_t q8_top(const float (&x)[4]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  return __reduce_max_sync(0xffffffffu, top);
}
// scale and 127 / m from it
__device__ __forceinline__ float2 q8_scales(uint32_t top) {
  const float m = __uint_as_float(top);
  if (top >= 0x7f800000u) return make_float2(__uint_as_float(0x7fffffffu), 0.0f);
  if (m < 0x1p-120f) return make_float2(0.0f, 0.0f);
  return make_float2(__fdiv_rn(m, 127.0f), __fdiv_rn(127.0f, m));
}
// |x r| <= 127 (1 + 2^-23), which rounds to 127
__device__ __forceinline__ uint32_t q8_encode(const float (&x)[4], uint32_t top, float r) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], r), kMagic));
  const uint32_t codes = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  return top >= 0x7f800000u ? 0 : codes;  // an infinity or NaN times 0 is no number
}
__device__ __forceinline__ void q8_decode(uint32_t codes, float s, float (&x)[4]) {
  const uint32_t b = codes ^ 0x80808080u;  // a code and 128, which 2^23 takes up exactly
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = __fmul_rn(__fadd_rn(__uint_as_float(__byte_perm(b, 0x4b000000u, 0x7440 + i)), -8388736.0f), s);
}

// Four values from i on, of which those at n and behind are zero, as they lie in memory.
template <class T>
__device__ __forceinline__ Packed<T, 4> load4(const T* p, uint64_t i, uint64_t n, bool vec) {
  Packed<T, 4> k;
  if (vec && i + 4 <= n) {
    k.all = *reinterpret_cast<const typename Words<sizeof(T) * 4>::type*>(p + i);
  } else {
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j < n ? widen(p[i + j]) : 0.0f;
    store_pack(reinterpret_cast<T*>(&k), x);
  }
  return k;
}
template <class T>
__device__ __forceinline__ void widen4(const Packed<T, 4>& k, float (&x)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = value_of<T>(k.word, j);
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
__device__ __forceinline__ void store_codes(uint32_t* codes, uint64_t i, uint64_t n, uint32_t c) {
  if (i + 4 <= n) {
    codes[i / 4] = c;
  } else {
    unsigned char* p = reinterpret_cast<unsigned char*>(codes);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (i + j < n) p[i + j] = (unsigned char)(c >> (8 * j));
  }
}
__device__ __forceinline__ uint32_t load_codes(const uint32_t* codes, uint64_t i, uint64_t n) {
  if (i + 4 <= n) return codes[i / 4];
  const unsigned char* p = reinterpret_cast<const unsigned char*>(codes);
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (i + j < n) c |= (uint32_t)p[i + j] << (8 * j);
  return c;
}

// Phi, the distribution function of the normal distribution, and exp(-x^2 / 2), which its density is 1 / sqrt(2 pi) of.
// Phi(-z) = exp(-z^2 / 2) (c1 t + ... + c7 t^7) with t = 1 / (1 + 0.32 z), z >= 0: the form of Abramowitz and Stegun's
// 7.1.26, with two terms more and coefficients fitted for the least absolute error (6 10^-9; 2 10^-7 at most as float32
// rounds it).  The one exponential serves Phi and the density: some 20 instructions a value, where the library's
// function made a pass over 50331648 float32 values 133 us there and 165 back (69 and 98 now), bound by instructions.
// Two values at a time, in instructions for both where there are any: sixteen-bit values leave a pass half the time that
// float32 ones do.
struct Normal {
  Pair sum, bell;
};
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_of(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ Normal normal(Pair x) {
  const Pair z = {fabsf(x.x), fabsf(x.y)};
  const Pair d = fma2(z, both(0.32f), both(1.0f)), e = mul2(mul2(z, z), both(-0.72134752044f));
  const Pair t = {reciprocal(d.x), reciprocal(d.y)}, bell = {exp2_of(e.x), exp2_of(e.y)};
  Pair p = fma2(both(0.04195379838347435f), t, both(-0.22253216803073883f));
  p = fma2(p, t, both(0.372079998254776f));
  p = fma2(p, t, both(-0.12819476425647736f));
  p = fma2(p, t, both(0.19610773026943207f));
  p = fma2(p, t, both(0.11168046295642853f));
  p = fma2(p, t, both(0.12890493869781494f));
  const Pair below = mul2(mul2(p, t), bell), above = fma2(below, both(-1.0f), both(1.0f));
  return {{x.x > 0.0f ? above.x : below.x, x.y > 0.0f ? above.y : below.y}, bell};
}
constexpr float kDensity = 0.3989422804014327f;  // 1 / sqrt(2 pi)

// U groups a warp.  kGelu: y = x Phi(x) is written as well.
template <class T, int U, bool kGelu>
__global__ void __launch_bounds__(32 * kWarps) q8_encode_kernel(const T* __restrict__ x, uint64_t n, bool vec,
                                                                T* __restrict__ y, uint32_t* __restrict__ codes,
                                                                float* __restrict__ scales) {
  pdl_wait(x);
  const uint64_t groups = (n + kQ8Group - 1) / kQ8Group;
  const uint64_t g0 = ((uint64_t)blockIdx.x * kWarps + threadIdx.x / 32) * U;
  const uint32_t lane = threadIdx.x % 32;
  Packed<T, 4> held[U];  // widened when they are used: more of them are on their way at once
#pragma unroll
  for (int u = 0; u < U; ++u) held[u] = load4(x, (g0 + u) * kQ8Group + 4 * lane, n, vec);
  // the two divisions of a group take longer than the rest of its values: a lane does those of one group, for all
  uint32_t top[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[4];
    widen4<T>(held[u], v);
    top[u] = q8_top(v);
  }
  uint32_t mine = top[0];
#pragma unroll
  for (int u = 1; u < U; ++u) mine = lane % U == u ? top[u] : mine;
  const float2 of_mine = q8_scales(mine);
  if (lane < U && g0 + lane < groups) scales[g0 + lane] = of_mine.x;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = (g0 + u) * kQ8Group + 4 * lane;
    float v[4];
    widen4<T>(held[u], v);
    store_codes(codes, i, n, q8_encode(v, top[u], __shfl_sync(0xffffffffu, of_mine.y, u)));
    if (kGelu) {
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const Pair x = {v[j], v[j + 1]}, r = mul2(x, normal(x).sum);
        o[j] = r.x, o[j + 1] = r.y;
      }
      store4(y, i, n, vec, o);
    }
  }
}

// The codes of U groups a warp and, for kGelu, the gradient behind: without kGelu `out` receives the values; with it
// dx = dy (Phi(x) + x phi(x)) and, where `again` is given, x Phi(x).
template <class T, int U, bool kGelu>
__global__ void __launch_bounds__(32 * kWarps)
    q8_decode_kernel(const uint32_t* __restrict__ codes, const float* __restrict__ scales, uint64_t n, bool vec,
                     const T* __restrict__ dy, T* __restrict__ out, T* __restrict__ again) {
  pdl_wait(codes);
  pdl_behind(scales, dy);
  const uint64_t groups = (n + kQ8Group - 1) / kQ8Group;
  const uint64_t g0 = ((uint64_t)blockIdx.x * kWarps + threadIdx.x / 32) * U;
  const uint32_t lane = threadIdx.x % 32;
  uint32_t c[U];
  float s[U];
  Packed<T, 4> d[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = (g0 + u) * kQ8Group + 4 * lane;
    c[u] = load_codes(codes, i, n);
    s[u] = g0 + u < groups ? scales[g0 + u] : 0.0f;
    if (kGelu) d[u] = load4(dy, i, n, vec);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = (g0 + u) * kQ8Group + 4 * lane;
    float x[4];
    q8_decode(c[u], s[u], x);
    if (!kGelu) {
      store4(out, i, n, vec, x);
    } else {
      float o[4], a[4], dv[4];
      widen4<T>(d[u], dv);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const Pair y = {x[j], x[j + 1]};
        const Normal f = normal(y);
        const Pair v = mul2(y, f.sum), g = mul2({dv[j], dv[j + 1]}, fma2(mul2(y, both(kDensity)), f.bell, f.sum));
        a[j] = v.x, a[j + 1] = v.y, o[j] = g.x, o[j + 1] = g.y;
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

// Groups a warp, each a load in flight: four, eight of sixteen-bit values, whose loads are half as wide (four: compressed in
// 57 us, eight: 35); below that many values a warp takes one, to spread over the SMs
// (59136 bfloat16 values: 462 warps, where four groups a warp would leave 33 of 148 SMs with any).
constexpr uint64_t kSpread = 1 << 20;
template <class T, bool kGelu>
cudaError_t encode(const void* x, uint64_t n, void* y, void* packed, cudaStream_t stream) {
  const bool vec = aligned4<T>(x) && (!kGelu || aligned4<T>(y));
  const bool wide = n >= kSpread;
  constexpr int kWide = sizeof(T) == 2 ? 8 : 4;
  return pdl_launch(wide ? q8_encode_kernel<T, kWide, kGelu> : q8_encode_kernel<T, 1, kGelu>, blocks_for(n, wide ? kWide : 1),
                    32 * kWarps, 0, stream, (const T*)x, n, vec, (T*)y, (uint32_t*)packed, scales_of(packed, n));
}
template <class T, bool kGelu>
cudaError_t decode(const void* packed, uint64_t n, const void* dy, void* out, void* again, cudaStream_t stream) {
  const bool vec = aligned4<T>(out) && (!dy || aligned4<T>(dy)) && (!again || aligned4<T>(again));
  const bool wide = n >= kSpread;
  constexpr int kWide = sizeof(T) == 2 ? 8 : 4;
  return pdl_launch(wide ? q8_decode_kernel<T, kWide, kGelu> : q8_decode_kernel<T, 1, kGelu>, blocks_for(n, wide ? kWide : 1),
                    32 * kWarps, 0, stream, (const uint32_t*)packed, (const float*)scales_of((void*)packed, n), n, vec,
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
