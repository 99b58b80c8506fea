// The value types of the training operators (float32, float16, bfloat16): conversion, and loads and stores of a few
// values at once.  Everything is computed in float32; a value is rounded to its type once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace csw {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N values that lie aligned to their whole size (at most 16 bytes): one load or store
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};
template <class T, int N>
__device__ __forceinline__ void load_pack(const T* p, float (&f)[N]) {
  const Pack<T, N> k = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = widen(k.v[i]);
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T* p, const float (&f)[N]) {
  Pack<T, N> k;
#pragma unroll
  for (int i = 0; i < N; ++i) k.v[i] = narrow<T>(f[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = k;
}

// Calls f(T()) for the type that a CSW_TYPE_* code names; false for a code that names none.
template <class F>
inline bool with_type(int type, F&& f) {
  switch (type) {
    case 0: f(float()); return true;
    case 1: f(__half()); return true;
    case 2: f(__nv_bfloat16()); return true;
    default: return false;
  }
}

}  // namespace csw
