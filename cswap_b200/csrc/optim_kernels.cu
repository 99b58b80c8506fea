// AdamW over many tensors at once, its state in 32 bits or in 8, and the norm of all gradients.
//
//   g' = c g,  c = min(1, max_norm / (norm + 1e-6)) where a norm is given
//   m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// State in 8 bits.  Groups of 128 consecutive values of a tensor share a scale 2^E, held as the byte E + 127: E is the least
// for which the group's largest magnitude is at most 1.75 2^E, but -126 at least; 0 stands for a group of zeros, 255 for one
// with a value that is no number or beyond 1.75 2^126.  A code of m is a sign, 4 bits of exponent and 3 of mantissa, of v 5
// and 3, the greatest exponent that of 2^E, with gradual underflow.  So the code is a float32 number's bits from the 20th on,
// once the number is scaled to the foot of the type's range, where underflow comes by itself.
//
// Rounding.  v changes by a thousandth a step, half a code's step is 3 to 6 %: rounded to the nearest, v would stay where it
// once was.  So the 20 bits that are cut off round up as often as they say, by random bits from the seed, the step, the tensor's
// place in the call and the value's index: the averages are right in the mean, and the same call gives the same bits.  v is
// not rounded to zero in a group that has anything: m's smallest step is 2^-17 of its group's scale, the root of v's smallest
// 2^-16.5, so that m / sqrt(v) stays of the size that it has for the group's largest.
//
// What bounds it.  In 32 bits HBM: 28 bytes a value, 447 us for the 110 M float32 parameters of a BERT-base-shaped encoder, 6.8
// TB/s.  In 8 bits the instructions, some 70 a value (8 of them for its random bits, 20 for both codes): as many with 16-bit
// gradients and copies 337 us, 1.25 times what its bytes take; 40 registers a thread, so that six CTAs an SM cover one another's
// loads (64 registers, four CTAs: a tenth longer).
//
// Every 32-bit operation that a code depends on is rounded by itself (no fused multiply-add), so that the codes follow from
// the definition whatever a compiler does.
//
// One launch takes hundreds of tensors: where they lie travels in the kernel's parameters, so that nothing is copied to the
// device and a captured call holds all that it needs.
#include "optim_kernels.h"

#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "internal.h"
#include "pdl.cuh"
#include "values.cuh"

namespace csw {
namespace {

// A piece of a tensor is 2048 values, 8 a thread: a group of 128 belongs to half a warp, whose lanes have four neighbours of its
// first half and four of its second, so that loads and stores of any type are runs of whole lines.
constexpr int kThreads = 256, kGroup = 128;
constexpr uint32_t kPiece = kThreads * 8;
// a thread's first value in a piece; the second four are kNext further on
__device__ __forceinline__ uint32_t first_value() { return threadIdx.x / 16 * kGroup + threadIdx.x % 16 * 4; }
constexpr uint32_t kNext = kGroup / 2;

struct Entry {
  const void* grad;
  void *param, *copy, *m, *v;
  uint8_t *m_scale, *v_scale;
  uint64_t numel;
  uint8_t param_type, grad_type, copy_type;  // CSW_TYPE_*
  // Whether four values are one load in all of the tensors, a piece beginning `shift` values before the first: tensors that lie
  // one behind the other in flat buffers have none of them on a boundary, but all the same way off it.
  bool packs;
  uint8_t shift;
};
template <int N>
struct Table {
  static constexpr int kSize = N;
  Entry tensor[N];
  uint32_t first[N + 1];  // pieces before each tensor
  int count;
  uint32_t place;  // of the first tensor in the call
};

struct Step {
  float b1, rest1, b2, rest2, eps;
  float decay, size, root;  // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  const float* norm;
  float max_norm;
  uint32_t call;  // random bits of the call
  // in place of the above where the program keeps them on the device
  const int64_t* step;
  const float* lr;
  double wide_b1, wide_b2, wide_lr, wide_decay;
  uint32_t seed;
  int64_t host_step;
};

// Tensors of a table: as many as 4 KB of a kernel's parameters hold beside the step, for lists of that many, or 380 (parameters are
// 32764 bytes at most), since the host pays for a table's bytes whatever stands in them.  A call's time on the host and on the
// device, tensors of 500 values, state in 32 bits: 20 tensors 3.6 us and 3.6 with the small table, 6.7 and 3.7 with the large
// one; 52 tensors 4.1 and 3.8, 7.1 and 4.1; 100 tensors, which the small one would take two launches for, 7.5 and 4.1.
constexpr int kFew = (4096 - sizeof(Step) - 16) / (sizeof(Entry) + 4), kMany = 380;
static_assert(sizeof(Table<kFew>) + sizeof(Step) <= 4096 && sizeof(Table<kMany>) + sizeof(Step) <= 32764, "kernel parameters");

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9e3779b1u;
  x ^= x >> 15;
  x *= 0x85ebca77u;
  return x ^ x >> 16;
}
__host__ __device__ __forceinline__ uint32_t random_of(uint32_t from, uint32_t place) { return mix(from + place * 0x9e3779b9u); }

// What depends on the step and the learning rate, in 64 bits.
__host__ __device__ inline void settle(Step& s, int64_t t, double lr) {
  const double n = (double)(t > 1 ? t : 1);
  s.decay = (float)(1.0 - lr * s.wide_decay);
  s.size = (float)(lr / -expm1(n * log(s.wide_b1)));
  s.root = (float)(1.0 / sqrt(-expm1(n * log(s.wide_b2))));
  s.call = random_of(s.seed, (uint32_t)t);
}

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, uint32_t piece) {
  int lo = 0, hi = t.count;  // first[lo] <= piece < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= piece) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Eight values of a thread, from index i and i + kNext on.  WHOLE: all of a tensor that lies in packs; else those from 0 up to
// n, and zeros for the others.
template <class T, bool WHOLE>
__device__ __forceinline__ void load_of(const void* from, int64_t i, int64_t n, bool packs, float (&f)[8]) {
  const T* p = static_cast<const T*>(from) + i;
#pragma unroll
  for (int q = 0; q < 2; ++q, p += kNext, i += kNext) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (WHOLE || (packs && i >= 0 && i + 4 <= n)) {
      load_pack(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j >= 0 && i + j < n) v[j] = widen(p[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) f[4 * q + j] = v[j];
  }
}
template <class T, bool WHOLE>
__device__ __forceinline__ void store_of(void* to, int64_t i, int64_t n, bool packs, const float (&f)[8]) {
  T* p = static_cast<T*>(to) + i;
#pragma unroll
  for (int q = 0; q < 2; ++q, p += kNext, i += kNext) {
    const float v[4] = {f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]};
    if (WHOLE || (packs && i >= 0 && i + 4 <= n)) {
      store_pack(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j >= 0 && i + j < n) p[j] = narrow<T>(v[j]);
    }
  }
}
template <bool WHOLE>
__device__ __forceinline__ void load_any(const void* from, int type, int64_t i, int64_t n, bool packs, float (&f)[8]) {
  if (type == CSW_TYPE_F32) load_of<float, WHOLE>(from, i, n, packs, f);
  else if (type == CSW_TYPE_F16) load_of<__half, WHOLE>(from, i, n, packs, f);
  else load_of<__nv_bfloat16, WHOLE>(from, i, n, packs, f);
}
template <bool WHOLE>
__device__ __forceinline__ void store_any(void* to, int type, int64_t i, int64_t n, bool packs, const float (&f)[8]) {
  if (type == CSW_TYPE_F32) store_of<float, WHOLE>(to, i, n, packs, f);
  else if (type == CSW_TYPE_F16) store_of<__half, WHOLE>(to, i, n, packs, f);
  else store_of<__nv_bfloat16, WHOLE>(to, i, n, packs, f);
}

// ---- 8-bit codes ------------------------------------------------------------------------------------------------------
template <bool WHOLE>
__device__ __forceinline__ uint2 load_codes(const void* from, int64_t i, int64_t n, bool packs) {
  const uint8_t* p = static_cast<const uint8_t*>(from) + i;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int q = 0; q < 2; ++q, p += kNext, i += kNext) {
    if (WHOLE || (packs && i + 4 <= n)) {
      w[q] = *reinterpret_cast<const uint32_t*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n) w[q] |= (uint32_t)p[j] << 8 * j;
    }
  }
  return make_uint2(w[0], w[1]);
}
template <bool WHOLE>
__device__ __forceinline__ void store_codes(void* to, int64_t i, int64_t n, bool packs, uint2 codes) {
  uint8_t* p = static_cast<uint8_t*>(to) + i;
#pragma unroll
  for (int q = 0; q < 2; ++q, p += kNext, i += kNext) {
    const uint32_t w = q ? codes.y : codes.x;
    if (WHOLE || (packs && i + 4 <= n)) {
      *reinterpret_cast<uint32_t*>(p) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n) p[j] = (uint8_t)(w >> 8 * j);
    }
  }
}
// SIGNED: m, else v.  The exponent of the foot of float32's range, seen from a group's scale.
template <bool SIGNED>
constexpr int kFoot = SIGNED ? 112 : 96;
__device__ __forceinline__ float power_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Both ways a value is multiplied with a power of two that may be beyond float32: in one step where it is not (averages from
// 2^-118 to 2^15 and 2^31, for all of a warp), else in two, of which the first is exact or what it leaves ends as zero in
// either way; and with what stands for no scale.
template <bool SIGNED>
__device__ __forceinline__ void values_of(uint2 codes, uint32_t scale, float (&f)[8]) {
  constexpr int kOnce = SIGNED ? -8 : kFoot<SIGNED>;  // from a scale's exponent to that of the one factor
  if (SIGNED) {  // these codes are e4m3 numbers with the exponent's bias 8 lower (and never that format's NaN)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const __half2_raw h =
          __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 4 ? codes.x : codes.y) >> (j % 4 * 8)), __NV_E4M3);
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
      f[j] = v.x, f[j + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f[j] = __uint_as_float(__byte_perm(j < 4 ? codes.x : codes.y, 0, 0x0444u | (uint32_t)(j % 4) << 12) >> 4);
  }
  const int e = (int)scale - 127 + kOnce;
  float power;
  if (__all_sync(0xffffffffu, scale - 1 < 254 && e >= -126 && e <= 127)) {
    power = power_of(e);
  } else {
    const float exact = scale == 0 ? 0.0f : scale == 255 ? __uint_as_float(0x7fc00000u) : power_of((int)scale - 127);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(f[j], power_of(kOnce));
    power = exact;
  }
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const Pair v = mul2({f[j], f[j + 1]}, both(power));
    f[j] = v.x, f[j + 1] = v.y;
  }
}
// The largest magnitude of a group's 16 threads, as bits; a NaN's are above all others.
__device__ __forceinline__ uint32_t top_of(const float (&f)[8]) {
  float top = f[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) asm("max.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(top) : "f"(f[j]));
  uint32_t bits = __float_as_uint(top) & 0x7fffffffu;
#pragma unroll
  for (int d = 1; d < 16; d *= 2) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
  return bits;
}
// Codes of a group whose largest magnitude is top, and its scale; cut(j): what is added to the 20 bits that are cut off, four
// bits further up.
template <bool SIGNED, class F>
__device__ __forceinline__ uint2 codes_of(const float (&f)[8], uint32_t top, F&& cut, uint32_t* scale) {
  const int e = max((int)(top >> 23) - 127 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
  *scale = top == 0 ? 0 : e > 126 ? 255 : (uint32_t)(e + 127);
  const bool none = *scale == 0 || *scale == 255;
  float size[8];
  if (__all_sync(0xffffffffu, !none && e + kFoot<SIGNED> <= 126)) {
    const float power = power_of(-e - kFoot<SIGNED>);
#pragma unroll
    for (int j = 0; j < 8; ++j) size[j] = __fmul_rn(fabsf(f[j]), power);
  } else {
    const float power = none ? 0.0f : power_of(-e);
#pragma unroll
    for (int j = 0; j < 8; ++j) size[j] = __fmul_rn(__fmul_rn(fabsf(f[j]), power), power_of(-kFoot<SIGNED>));
  }
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w[j] = __float_as_uint(size[j]) * 16u + cut(j);  // the code on top
    if (SIGNED) w[j] |= __float_as_uint(f[j]) & 0x80000000u;
    else w[j] = max(w[j], 1u << 24);
  }
  auto four = [](const uint32_t* v) {
    return __byte_perm(__byte_perm(v[0], v[1], 0x0073u), __byte_perm(v[2], v[3], 0x0073u), 0x5410u);
  };
  return none ? make_uint2(0, 0) : make_uint2(four(w), four(w + 4));
}

// ---- the step -----------------------------------------------------------------------------------------------------------
// The unit's square root and reciprocal, off by 2^-23 at most: a parameter's move is added to something much larger.  They take
// what is below 2^-126 for zero, which an epsilon from 2^-40 on does not notice; below that the exact ones are taken.
__device__ __forceinline__ float root_of(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A CTA's pieces, one behind the other: f(tensor, its index in the table, this thread's first value in it, whole), whole as
// std::true_type for a piece that has nothing but values in packs: there is then nothing to ask for each of them.
template <int N, class F>
__device__ __forceinline__ void over_pieces(const Table<N>& table, uint32_t run, F&& f) {
  uint32_t piece = blockIdx.x * run;
  const uint32_t end = min(piece + run, table.first[table.count]);
  int at = tensor_of(table, piece);
  for (; piece < end; ++piece) {
    while (piece >= table.first[at + 1]) ++at;
    const Entry& t = table.tensor[at];
    const int64_t begin = (int64_t)(piece - table.first[at]) * kPiece - t.shift, i = begin + first_value();
    if (t.packs && begin >= 0 && begin + (int64_t)kPiece <= (int64_t)t.numel) f(t, at, i, std::true_type());
    else f(t, at, i, std::false_type());
  }
}

// What a CTA knows of the step.
struct Now {
  float b1, rest1, b2, rest2, eps, decay, size, root, factor;
  uint32_t call;
};
template <bool EIGHT, bool WHOLE>
__device__ __forceinline__ void adamw_piece(const Entry& t, uint32_t place, int64_t i, const Now& now) {
  const int64_t n = (int64_t)t.numel;
  const uint64_t group = (uint64_t)i / kGroup;  // of an 8-bit state, whose pieces are not shifted
  const bool some = WHOLE || group * kGroup < t.numel;
  float g[8], p[8], m[8], v[8];
  uint2 mc, vc;
  uint32_t m_scale = 0, v_scale = 0;
  if constexpr (EIGHT) {
    mc = load_codes<WHOLE>(t.m, i, n, t.packs), vc = load_codes<WHOLE>(t.v, i, n, t.packs);
    if (some) m_scale = t.m_scale[group], v_scale = t.v_scale[group];
  } else {
    load_of<float, WHOLE>(t.m, i, n, t.packs, m);
    load_of<float, WHOLE>(t.v, i, n, t.packs, v);
  }
  load_any<WHOLE>(t.grad, t.grad_type, i, n, t.packs, g);
  load_any<WHOLE>(t.param, t.param_type, i, n, t.packs, p);
  if constexpr (EIGHT) {
    values_of<true>(mc, m_scale, m);
    values_of<false>(vc, v_scale, v);
  }
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    // Two at a time only where no sum follows: a product and a sum of pairs become one operation, whatever their rounding says.
    const Pair s = mul2({g[j], g[j + 1]}, both(now.factor)), r = mul2(s, both(now.rest2));
    m[j] = __fadd_rn(__fmul_rn(m[j], now.b1), __fmul_rn(s.x, now.rest1));
    m[j + 1] = __fadd_rn(__fmul_rn(m[j + 1], now.b1), __fmul_rn(s.y, now.rest1));
    v[j] = __fadd_rn(__fmul_rn(v[j], now.b2), __fmul_rn(r.x, s.x));
    v[j + 1] = __fadd_rn(__fmul_rn(v[j + 1], now.b2), __fmul_rn(r.y, s.y));
  }
  if (now.eps >= 0x1p-40f) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const Pair below = fma2({root_of(v[j]), root_of(v[j + 1])}, both(now.root), both(now.eps));
      const Pair move = mul2({m[j], m[j + 1]}, {inverse_of(below.x), inverse_of(below.y)});
      const Pair r = fma2(both(-now.size), move, mul2({p[j], p[j + 1]}, both(now.decay)));
      p[j] = r.x, p[j + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      p[j] = fmaf(-now.size, m[j] / fmaf(sqrtf(v[j]), now.root, now.eps), p[j] * now.decay);
  }
  store_any<WHOLE>(t.param, t.param_type, i, n, t.packs, p);
  if (t.copy) store_any<WHOLE>(t.copy, t.copy_type, i, n, t.packs, p);
  if constexpr (EIGHT) {
    if (!WHOLE) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j / 4 * kNext + j % 4 >= n) m[j] = v[j] = 0.0f;
    }
    const uint32_t key = random_of(now.call, place) + (uint32_t)i;
    uint32_t r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = mix(key + j / 4 * kNext + j % 4);
    // 16 random bits over 0x80, at the place of the bits that are cut off
    mc = codes_of<true>(m, top_of(m), [&](int j) { return __byte_perm(r[j], 0x80u, 0x5324u); }, &m_scale);
    vc = codes_of<false>(v, top_of(v), [&](int j) { return __byte_perm(r[j], 0x80u, 0x5104u); }, &v_scale);
    store_codes<WHOLE>(t.m, i, n, t.packs, mc);
    store_codes<WHOLE>(t.v, i, n, t.packs, vc);
    if (some && threadIdx.x % 16 == 0) t.m_scale[group] = (uint8_t)m_scale, t.v_scale[group] = (uint8_t)v_scale;
  } else {
    store_of<float, WHOLE>(t.m, i, n, t.packs, m);
    store_of<float, WHOLE>(t.v, i, n, t.packs, v);
  }
}

template <int N, bool EIGHT>
__global__ void __launch_bounds__(kThreads, 6) adamw_kernel(const __grid_constant__ Table<N> table,
                                                         const __grid_constant__ Step given) {
  __shared__ Step computed;
  pdl_trigger_if_few();
  pdl_wait();
  Now now{given.b1, given.rest1, given.b2, given.rest2, given.eps, given.decay, given.size, given.root, 1.0f, given.call};
  if (given.step || given.lr) {
    // Every CTA works them out for itself, which HBM's share of the time hides in 32 bits (444 us either way for the 110 M
    // parameters above) and the instructions' does not in 8 (373 us in place of 337).
    if (threadIdx.x == 0) {
      computed = given;
      settle(computed, given.step ? *given.step : given.host_step, given.lr ? (double)*given.lr : given.wide_lr);
    }
    __syncthreads();
    now.decay = computed.decay, now.size = computed.size, now.root = computed.root, now.call = computed.call;
  }
  if (given.norm) {
    const float q = __fdiv_rn(given.max_norm, __fadd_rn(*given.norm, 1e-6f));
    now.factor = q >= 1.0f ? 1.0f : q;  // NaN of a norm that is none
  }
  over_pieces(table, 1, [&](const Entry& t, int at, int64_t i, auto whole) {
    adamw_piece<EIGHT, decltype(whole)::value>(t, table.place + at, i, now);
  });
}

// The state in 8 bits from and to averages in 32, which stand in the places of param and copy; rounded to the nearest.
template <int N, bool PACK>
__global__ void __launch_bounds__(kThreads) adamw8_convert_kernel(const __grid_constant__ Table<N> table) {
  pdl_trigger_if_few();
  pdl_wait();
  over_pieces(table, 1, [&](const Entry& t, int, int64_t i, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    const int64_t n = (int64_t)t.numel;
    const uint64_t group = (uint64_t)i / kGroup;
    const bool some = kWhole || group * kGroup < t.numel;
    float m[8], v[8];
    uint32_t m_scale = 0, v_scale = 0;
    if constexpr (PACK) {
      load_of<float, kWhole>(t.param, i, n, t.packs, m);
      load_of<float, kWhole>(t.copy, i, n, t.packs, v);
      auto half = [](int) { return 1u << 23; };
      store_codes<kWhole>(t.m, i, n, t.packs, codes_of<true>(m, top_of(m), half, &m_scale));
      store_codes<kWhole>(t.v, i, n, t.packs, codes_of<false>(v, top_of(v), half, &v_scale));
      if (some && threadIdx.x % 16 == 0) t.m_scale[group] = (uint8_t)m_scale, t.v_scale[group] = (uint8_t)v_scale;
    } else {
      const uint2 mc = load_codes<kWhole>(t.m, i, n, t.packs), vc = load_codes<kWhole>(t.v, i, n, t.packs);
      if (some) m_scale = t.m_scale[group], v_scale = t.v_scale[group];
      values_of<true>(mc, m_scale, m);
      values_of<false>(vc, v_scale, v);
      store_of<float, kWhole>(t.param, i, n, t.packs, m);
      store_of<float, kWhole>(t.copy, i, n, t.packs, v);
    }
  });
}

// ---- the norm -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ double sum_of_threads(double s) {
  __shared__ double warps[kThreads / 32];
#pragma unroll
  for (int d = 16; d; d /= 2) s += __shfl_down_sync(0xffffffffu, s, d);
  if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < kThreads / 32; ++w) s += warps[w];
  return s;
}
// Squares are summed in 64 bits: a norm that goes into every value must not depend on the order of its sum.
template <int N>
__global__ void __launch_bounds__(kThreads) norm_parts_kernel(const __grid_constant__ Table<N> table, uint32_t run,
                                                              double* parts) {
  pdl_trigger_if_few();
  pdl_wait();
  double s[4] = {0.0, 0.0, 0.0, 0.0};  // sums of their own, so that one need not wait for the other
  over_pieces(table, run, [&](const Entry& t, int, int64_t i, auto whole) {
    float g[8];
    load_any<decltype(whole)::value>(t.grad, t.grad_type, i, (int64_t)t.numel, t.packs, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j % 4] = fma((double)g[j], (double)g[j], s[j % 4]);
  });
  const double sum = sum_of_threads((s[0] + s[1]) + (s[2] + s[3]));
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}
__global__ void __launch_bounds__(kThreads) norm_sum_kernel(const double* __restrict__ parts, uint32_t count, float* norm) {
  pdl_trigger();
  pdl_wait(parts);
  double s = 0.0;
  for (uint32_t i = threadIdx.x; i < count; i += kThreads) s += parts[i];
  s = sum_of_threads(s);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
// Calls launch(table, pieces) for as many tensors at a time as a table holds; empty tensors keep their place.
template <int N, class F>
cudaError_t in_tables(const csw_adamw_tensor* tensors, size_t count, F&& launch) {
  static thread_local Table<N> table;
  for (size_t at = 0; at < count;) {
    table.place = (uint32_t)at;
    uint64_t pieces = 0;
    int n = 0;
    for (; n < N && at < count; ++at, ++n) {
      const csw_adamw_tensor& t = tensors[at];
      // how many values each tensor lies behind a boundary of four of them
      auto off = [](const void* p, size_t size) { return (int)(reinterpret_cast<uintptr_t>(p) / size % 4); };
      auto size_of = [](int type) { return type == CSW_TYPE_F32 ? (size_t)4 : (size_t)2; };
      const bool eight = t.exp_avg_scale;
      const void* const first = t.param ? t.param : t.grad;
      const int shift = off(first, size_of(t.param ? t.param_type : t.grad_type));
      bool packs = !eight || shift == 0;
      auto same = [&](const void* p, size_t size) { packs = packs && (!p || off(p, size) == shift); };
      same(t.grad, size_of(t.grad_type)), same(t.copy, size_of(t.copy_type));
      same(t.exp_avg, eight ? 1 : 4), same(t.exp_avg_sq, eight ? 1 : 4);
      const uint64_t reach = t.numel + (packs ? shift : 0), more = reach / kPiece + (reach % kPiece != 0);
      if (n && pieces + more > 0x7fffffffu) break;
      table.tensor[n] = {t.grad, t.param, t.copy, t.exp_avg, t.exp_avg_sq, static_cast<uint8_t*>(t.exp_avg_scale),
                         static_cast<uint8_t*>(t.exp_avg_sq_scale), t.numel, (uint8_t)t.param_type, (uint8_t)t.grad_type,
                         (uint8_t)t.copy_type, packs, (uint8_t)(packs ? shift : 0)};
      table.first[n] = (uint32_t)pieces;
      pieces += more;
    }
    table.first[n] = (uint32_t)pieces;
    table.count = n;
    if (pieces == 0) continue;
    if (const cudaError_t e = launch(table, (uint32_t)pieces)) return e;
  }
  return cudaSuccess;
}
template <class F>
cudaError_t in_any_tables(const csw_adamw_tensor* tensors, size_t count, F&& launch) {
  return count <= kFew ? in_tables<kFew>(tensors, count, launch) : in_tables<kMany>(tensors, count, launch);
}
// Pieces of a CTA of the norm: the search for its tensor and its sum's way out are spread over some, as long as there are CTAs
// for eight an SM.  (92 us for 110 M bfloat16 values with one piece each, 51 with eight.  The step wants one: 470 us with eight,
// 447 with one, since new CTAs load while others compute.)
uint32_t run_of(uint32_t pieces) { return std::min(std::max(pieces / (8u * (uint32_t)sm_count()), 1u), 8u); }
uint32_t grid_of(uint32_t pieces, uint32_t run) { return pieces / run + (pieces % run != 0); }

}  // namespace

cudaError_t adamw_launch(const csw_adamw_tensor* tensors, size_t count, const csw_adamw_options& o, cudaStream_t stream) {
  Step s{};
  s.b1 = (float)o.beta1, s.rest1 = (float)(1.0 - o.beta1), s.b2 = (float)o.beta2, s.rest2 = (float)(1.0 - o.beta2);
  s.eps = (float)o.eps, s.norm = o.d_norm, s.max_norm = (float)o.max_norm, s.step = o.d_step, s.lr = o.d_lr;
  s.wide_b1 = o.beta1, s.wide_b2 = o.beta2, s.wide_lr = o.lr, s.wide_decay = o.weight_decay;
  s.seed = o.seed, s.host_step = o.step;
  settle(s, o.step, o.lr);
  return in_any_tables(tensors, count, [&](const auto& table, uint32_t pieces) {
    constexpr int N = std::decay_t<decltype(table)>::kSize;
    return pdl_launch(o.bits == 8 ? adamw_kernel<N, true> : adamw_kernel<N, false>, pieces, kThreads, 0, stream, table, s);
  });
}

cudaError_t adamw8_convert_launch(const csw_adamw_tensor* tensors, size_t count, bool pack, cudaStream_t stream) {
  return in_any_tables(tensors, count, [&](const auto& table, uint32_t pieces) {
    constexpr int N = std::decay_t<decltype(table)>::kSize;
    return pdl_launch(pack ? adamw8_convert_kernel<N, true> : adamw8_convert_kernel<N, false>, pieces, kThreads, 0, stream,
                      table);
  });
}

uint64_t gradient_norm_partials(const csw_adamw_tensor* tensors, size_t count) {
  uint64_t parts = 0;
  in_any_tables(tensors, count, [&](const auto&, uint32_t pieces) {
    parts += grid_of(pieces, run_of(pieces));
    return cudaSuccess;
  });
  return parts;
}

cudaError_t gradient_norm_launch(const csw_adamw_tensor* tensors, size_t count, float* norm, double* partials,
                                 cudaStream_t stream) {
  uint32_t parts = 0;
  const cudaError_t e = in_any_tables(tensors, count, [&](const auto& table, uint32_t pieces) {
    constexpr int N = std::decay_t<decltype(table)>::kSize;
    const uint32_t run = run_of(pieces), grid = grid_of(pieces, run);
    const cudaError_t e = pdl_launch(norm_parts_kernel<N>, grid, kThreads, 0, stream, table, run, partials + parts);
    parts += grid;
    return e;
  });
  if (e != cudaSuccess) return e;
  return pdl_launch(norm_sum_kernel, 1, kThreads, 0, stream, (const double*)partials, parts, norm);
}

}  // namespace csw
