// The value types of the training operators (float32, float16, bfloat16): conversion, and loads and stores of a few
// values at once.  Everything is computed in float32; a value is rounded to its type once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

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

// N values that lie aligned to their whole size (at most 16 bytes): one load or store, as words
template <int BYTES>
struct Words;
template <>
struct Words<2> {
  using type = unsigned short;
};
template <>
struct Words<4> {
  using type = uint32_t;
};
template <>
struct Words<8> {
  using type = uint2;
};
template <>
struct Words<16> {
  using type = uint4;
};
template <class T, int N>
union Packed {
  typename Words<sizeof(T) * N>::type all;
  uint32_t word[sizeof(T) * N < 4 ? 1 : sizeof(T) * N / 4];
  unsigned short half;
};
// value j of a pack's words
template <class T>
__device__ __forceinline__ float value_of(const uint32_t* w, int j) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
  const uint32_t bits = w[j / 2];
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(j % 2 ? bits & 0xffff0000u : bits << 16);
  return __half2float(__ushort_as_half((unsigned short)(j % 2 ? bits >> 16 : bits & 0xffff)));
}
template <class T, int N>
__device__ __forceinline__ void load_pack(const T* p, float (&f)[N]) {
  Packed<T, N> k;
  k.word[0] = 0;
  k.all = *reinterpret_cast<const typename Words<sizeof(T) * N>::type*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = value_of<T>(k.word, i);
}
template <class T>
__device__ __forceinline__ uint32_t word_of(float a, float b);
template <>
__device__ __forceinline__ uint32_t word_of<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t word_of<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T* p, const float (&f)[N]) {
  if constexpr (N == 1) {
    *p = narrow<T>(f[0]);
  } else {
    Packed<T, N> k;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) k.word[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) k.word[i / 2] = word_of<T>(f[i], f[i + 1]);
    }
    *reinterpret_cast<typename Words<sizeof(T) * N>::type*>(p) = k.all;
  }
}

// two float32 operations in one instruction
struct Pair {
  float x, y;
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("{\n\t.reg .b64 a, b, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 r, a, b, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 r, a, b;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 r, a, b;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ Pair both(float v) { return {v, v}; }

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
