// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / c,  var = sum (x - mean)^2 / c,  rstd = 1 / sqrt(var + eps),  h = (x - mean) rstd
//   y = h w + b
//   dx = rstd (g - sum g / c - h sum(g h) / c) with g = dy w;  dw = sum over rows of dy h,  db = sum over rows of dy
//
// What bounds it: HBM, and for rows of thousands of values the latency of their sums.  A row is read once and held in
// registers by the threads that share it, eight values each (2 of a warp's threads up to 16 values, 1024 up to 8192), so
// that the variance is summed from the centred values, a second time over registers and not over memory.  With few values
// a thread many rows share an SM, and one's loads run under another's sums (4099 x 1001 bfloat16, both ways: 33 us with
// eight values a thread, 75 with a warp for a whole row; 8 float16 columns 130 us for 67 million values, 2150 with a warp
// a row).  Longer rows are read again, from L1 or L2.
//
// Backward, each thread keeps the sums of dw and db of its own columns over all rows that its CTA takes; they go to
// memory once per CTA, in a fixed order, and a second launch adds them up.  No atomics: the same call gives the same bits.
//
// Cold: 16384 x 768 float32 with its sum forward 36 us (5.5 TB/s), 16384 x 4096 bfloat16 backward 93 us and 5 for the
// sums' last step (4.3 TB/s; 62 us at a copy's rate: a row is two barriers' worth of latency, and two rows at once,
// which is what registers allow, do not hide all of it).
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/cswap_b200.h"
#include "internal.h"
#include "norm_kernels.h"
#include "pdl.cuh"
#include "values.cuh"

namespace csw {
namespace {

// ---- parameters: of their own type, which is the values' or float32 -----------------------------------------------
__device__ __forceinline__ float param_at(const void* p, int type, uint64_t i) {
  if (type == CSW_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == CSW_TYPE_F16) return widen(static_cast<const __half*>(p)[i]);
  return widen(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void param_to(void* p, int type, uint64_t i, float v) {
  if (type == CSW_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == CSW_TYPE_F16) static_cast<__half*>(p)[i] = narrow<__half>(v);
  else static_cast<__nv_bfloat16*>(p)[i] = narrow<__nv_bfloat16>(v);
}
template <int THREADS>
constexpr int kPlaces = THREADS < 32 ? 1 : THREADS / 32;
// Sums over the THREADS threads that share a row (a part of a warp, a warp, or the whole CTA) of N pairs of values; all of them get them.  A
// CTA's sums take turns with two places in shared memory (`turn`), so that one barrier a sum is enough: a place is written
// again two sums later, behind a barrier that all who read it have passed.
template <int THREADS, int N>
__device__ __forceinline__ void row_sums(float2 (&v)[N], float2 (*shared)[kPlaces<THREADS>], int turn) {
#pragma unroll
  for (int d = THREADS < 32 ? THREADS / 2 : 16; d; d /= 2)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n].x += __shfl_xor_sync(0xffffffffu, v[n].x, d);
      v[n].y += __shfl_xor_sync(0xffffffffu, v[n].y, d);
    }
  if (THREADS > 32) {
    float2(*place)[kPlaces<THREADS>] = shared + (turn & 1) * N;
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (threadIdx.x % 32 == 0) place[n][threadIdx.x / 32] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) v[n].x += place[n][i].x, v[n].y += place[n][i].y;
    }
  }
}
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float2 (*shared)[kPlaces<THREADS>], int turn) {
  float2 s[1] = {make_float2(v, 0.0f)};
  row_sums<THREADS>(s, shared, turn);
  return s[0].x;
}

// VEC values as they lie in memory, in words: held so, they take half the registers that single two-byte values would.
template <class T, int VEC>
struct Raw {
  static constexpr int kWords = VEC * sizeof(T) < 4 ? 1 : VEC * sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ float operator[](int j) const { return value_of<T>(w, j); }
  // one value into its place, which holds zeros
  __device__ void put(int j, T v) {
    if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v);
    else w[j / 2] |= (uint32_t) * reinterpret_cast<const unsigned short*>(&v) << (16 * (j % 2));
  }
  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // all of them from p, aligned to 16 bytes where there are as many or more
  __device__ void read(const T* p) {
    if constexpr (VEC == 1) {
      w[0] = 0;
      put(0, *p);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    }
  }
};

// How the threads lie on the rows.  THREADS threads share a row: thread t holds VEC values from the column
// (k THREADS + t) VEC - shift on, for each k < ITER.  Where the number of columns is no multiple of VEC, rows begin at
// any place among the packs of VEC values (16 bytes) that memory is read in; `shift` is that place, and the packs that
// reach over a row's ends are masked (SHIFTED).  The shift repeats every `period` rows, and a CTA takes only rows of one
// shift: then the columns of a thread stay the same, with their weights and their sums in registers.
template <class T, int VEC, int ITER, int THREADS, bool SHIFTED>
struct Rows {
  static constexpr int kBlock = THREADS <= 32 ? 128 : THREADS, kTogether = kBlock / THREADS;
  // CTAs an SM should have room for: 64 registers a thread forward, 80 or more backward
  static constexpr int kForward = 1024 / kBlock, kBackward = kBlock > 768 ? 1 : 768 / kBlock;
  // Rows at once, backward, where a CTA has an SM to itself and the registers for two: a row waits for its sums' way through
  // shuffles and shared memory, which then serves both (16384 x 4096 bfloat16 93 us, 106 one at a time).  CTAs of 768 and
  // 1024 threads have 80 and 64 registers a thread, which two rows do not fit into (67 million bfloat16 values, rows of
  // 6144: 114 us one at a time, 177 two at once; of 8192: 124 and 146).
  static constexpr int kAtOnce = sizeof(T) == 2 && THREADS == 512 ? 2 : 1;
  uint64_t rows, total;  // total: values
  uint32_t cols, period;
  uint64_t row, step;    // the thread's first row, and how far on the next one is
  int first;             // column of its first value, less than 0 for some that are masked
  __device__ Rows(uint64_t rows_, uint64_t cols_, uint32_t period_)
      : rows(rows_), total(rows_ * cols_), cols((uint32_t)cols_), period(period_) {
    const uint32_t kind = blockIdx.x % period;
    row = ((uint64_t)blockIdx.x / period * kTogether + threadIdx.x / THREADS) * period + kind;
    step = (uint64_t)(gridDim.x / period) * kTogether * period;
    first = (int)(threadIdx.x % THREADS) * VEC - (SHIFTED ? (int)(kind * (uint64_t)cols % VEC) : 0);
  }
  // steps of the warp's first row's thread, which has the most
  __device__ uint64_t rounds() const {
    const uint64_t lead = __shfl_sync(0xffffffffu, row, 0);
    return lead < rows ? (rows - lead + step - 1) / step : 0;
  }
  __device__ int column(int k) const { return first + k * THREADS * VEC; }
  __device__ bool any(int c) const { return (!SHIFTED || c > -VEC) && c < (int)cols; }
  __device__ bool has(int c) const { return !SHIFTED || (c >= 0 && c < (int)cols); }
  // the values from column c on of the row that begins at `base`; what is masked is whatever lies there
  __device__ void load(const T* p, uint64_t base, int c, Raw<T, VEC>& v) const {
    if (!SHIFTED || base + c + VEC <= total) {
      v.read(p + base + c);
    } else {
      v.clear();
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (base + c + j < total) v.put(j, p[base + c + j]);
    }
  }
  __device__ void store(T* p, uint64_t base, int c, const float (&f)[VEC]) const {
    if (!SHIFTED || (c >= 0 && c + VEC <= (int)cols)) {
      store_pack(p + base + c, f);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (has(c + j)) p[base + c + j] = narrow<T>(f[j]);
    }
  }
  // the thread's weights or biases, for all its rows
  template <class P>
  __device__ void params(const void* p, float missing, Raw<P, VEC> (&f)[ITER]) const {
    const P* q = static_cast<const P*>(p);
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int c = column(k);
      f[k].clear();
      if (!any(c)) continue;
      if (q && !SHIFTED) {
        f[k].read(q + c);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!q || has(c + j)) f[k].put(j, q ? q[c + j] : narrow<P>(missing));
      }
    }
  }
};

template <class T, class P, int VEC, int ITER, int THREADS, bool SHIFTED>
__global__ void __launch_bounds__(Rows<T, VEC, ITER, THREADS, SHIFTED>::kBlock,
                                  Rows<T, VEC, ITER, THREADS, SHIFTED>::kForward)
    norm_forward_kernel(const NormForward a, uint32_t period) {
  __shared__ float2 shared[2][kPlaces<THREADS>];
  const T* x = static_cast<const T*>(a.x);
  const T* residual = static_cast<const T*>(a.residual);
  pdl_wait(x);
  pdl_behind(residual);
  const Rows<T, VEC, ITER, THREADS, SHIFTED> at(a.rows, a.cols, period);
  T* sum = static_cast<T*>(a.sum);
  T* y = static_cast<T*>(a.y);
  const float inv = 1.0f / (float)at.cols;
  struct Held {
    Raw<T, VEC> x[ITER], r[ITER];
  };
  auto load = [&](uint64_t row, Held& h) {
    const uint64_t base = row * at.cols;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int c = at.column(k);
      if (at.any(c)) {
        at.load(x, base, c, h.x[k]);
        if (residual) at.load(residual, base, c, h.r[k]);
      }
    }
  };
  // The next row's values are on their way while a row is worked on, for sixteen-bit values: 67 million bfloat16 ones, cold,
  // in rows of 64, 768, 4096 and 8192 columns take 72, 82, 102 and 137 us, 78, 105, 115 and 165 without.  Of float32, half as
  // many take 55, 94 and 82 us in rows of 64, 768 and 2048 with it, 53, 66 and 64 without; rows of 4096 and more, which
  // it would help (70 us against 74, at 8192 82 against 107), go without as well.
  constexpr bool kAhead = sizeof(T) == 2;
  Held now, next;
  if (kAhead && at.row < at.rows) load(at.row, next);
  Raw<P, VEC> w[ITER], b[ITER];
  at.params(a.weight, 1.0f, w);
  at.params(a.bias, 0.0f, b);
  int turn = 0;
  // Where parts of a warp have rows of their own, all of them go on until the last is done: its sums need every lane.
  const uint64_t rounds = THREADS < 32 ? at.rounds() : 0;
  uint64_t row = at.row;
#pragma unroll 1
  for (uint64_t i = 0; THREADS < 32 ? i < rounds : row < at.rows; ++i, row += at.step) {
    const bool mine = THREADS >= 32 || row < at.rows;
    const uint64_t base = row * at.cols;
    if (kAhead) now = next;
    else if (mine) load(row, now);
    if (kAhead && row + at.step < at.rows) load(row + at.step, next);
    float v[ITER][VEC], s = 0.0f;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int c = at.column(k);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = 0.0f;
      if (mine && at.any(c)) {
        // what is normed, and what backward reads, is the sum as it is held
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (at.has(c + j)) v[k][j] = residual ? widen(narrow<T>(now.x[k][j] + now.r[k][j])) : now.x[k][j];
        if (residual) at.store(sum, base, c, v[k]);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += v[k][j];
    }
    const float mean = row_sum<THREADS>(s, shared, turn++) * inv;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int c = at.column(k);
      if (mine && at.any(c)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (at.has(c + j)) v[k][j] -= mean;
          s += v[k][j] * v[k][j];
        }
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<THREADS>(s, shared, turn++) * inv + a.eps);
    if (mine && threadIdx.x % THREADS == 0) a.mean[row] = mean, a.rstd[row] = rstd;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int c = at.column(k);
      if (mine && at.any(c)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k][j] = v[k][j] * rstd * w[k][j] + b[k][j];
        at.store(y, base, c, v[k]);
      }
    }
  }
}

// Long rows: read three times, a pack of VEC values a thread and step.
constexpr int kLongThreads = 512;
template <class T, int VEC>
__global__ void __launch_bounds__(kLongThreads) norm_forward_long_kernel(const NormForward a) {
  __shared__ float2 shared[2][kLongThreads / 32];
  pdl_wait();
  const uint64_t base = (uint64_t)blockIdx.x * a.cols;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* residual = a.residual ? static_cast<const T*>(a.residual) + base : nullptr;
  T* sum = residual ? static_cast<T*>(a.sum) + base : nullptr;
  float s = 0.0f;
  for (uint64_t c = threadIdx.x * VEC; c < a.cols; c += kLongThreads * VEC) {
    float v[VEC];
    load_pack(x + c, v);
    if (residual) {
      float r[VEC];
      load_pack(residual + c, r);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = widen(narrow<T>(v[j] + r[j]));
      store_pack(sum + c, v);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += v[j];
  }
  const T* src = residual ? sum : x;  // a thread reads back what it wrote itself
  const float mean = row_sum<kLongThreads>(s, shared, 0) / (float)a.cols;
  s = 0.0f;
  for (uint64_t c = threadIdx.x * VEC; c < a.cols; c += kLongThreads * VEC) {
    float v[VEC];
    load_pack(src + c, v);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += (v[j] - mean) * (v[j] - mean);
  }
  const float rstd = 1.0f / sqrtf(row_sum<kLongThreads>(s, shared, 1) / (float)a.cols + a.eps);
  if (threadIdx.x == 0) a.mean[blockIdx.x] = mean, a.rstd[blockIdx.x] = rstd;
  T* y = static_cast<T*>(a.y) + base;
  for (uint64_t c = threadIdx.x * VEC; c < a.cols; c += kLongThreads * VEC) {
    float v[VEC];
    load_pack(src + c, v);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float w = a.weight ? param_at(a.weight, a.param_type, c + j) : 1.0f;
      const float b = a.bias ? param_at(a.bias, a.param_type, c + j) : 0.0f;
      v[j] = (v[j] - mean) * rstd * w + b;
    }
    store_pack(y + c, v);
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------
// Workspace row blockIdx.x receives the CTA's sums: dw, then db.  A row's values are held as they came, and widened anew
// for each of the two passes over them; the next row's are on their way meanwhile.
template <class T, class P, int VEC, int ITER, int THREADS, bool SHIFTED>
__global__ void __launch_bounds__(Rows<T, VEC, ITER, THREADS, SHIFTED>::kBlock,
                                  Rows<T, VEC, ITER, THREADS, SHIFTED>::kBackward)
    norm_backward_kernel(const NormBackward a, uint32_t period) {
  using R = Rows<T, VEC, ITER, THREADS, SHIFTED>;
  constexpr int N = R::kAtOnce;
  __shared__ float2 shared[2 * N][kPlaces<THREADS>];
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  pdl_wait(x);
  pdl_behind(dy);
  const R at(a.rows, a.cols, period);
  T* dx = static_cast<T*>(a.dx);
  const float inv = 1.0f / (float)at.cols;
  // values go two at a time, in instructions for both
  constexpr int kPairs = (VEC + 1) / 2;
  Pair dw[ITER][kPairs], db[ITER][kPairs];
#pragma unroll
  for (int k = 0; k < ITER; ++k)
#pragma unroll
    for (int j = 0; j < kPairs; ++j) dw[k][j] = db[k][j] = both(0.0f);
  struct Held {
    Raw<T, VEC> x[ITER], dy[ITER];
    float mean, rstd;
  };
  auto load = [&](uint64_t row, Held& h) {
    const uint64_t base = row * at.cols;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int c = at.column(k);
      if (at.any(c)) at.load(x, base, c, h.x[k]), at.load(dy, base, c, h.dy[k]);
    }
    h.mean = a.mean[row], h.rstd = a.rstd[row];
  };
  Held now[N], next[N];
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (at.row + n * at.step < at.rows) load(at.row + n * at.step, next[n]);
  Raw<P, VEC> w[ITER];
  at.params(a.weight, 1.0f, w);
  int turn = 0;
  const uint64_t rounds = THREADS < 32 ? at.rounds() : 0;  // as forward
  uint64_t row = at.row;
#pragma unroll 1
  for (uint64_t i = 0; THREADS < 32 ? i < rounds : row < at.rows; i += N, row += N * at.step) {
    float2 sums[N];
    // normed values and dy of a pair of columns; a masked value is another row's, 0 in its place adds nothing
    auto pair = [&](const auto& raw, int j) { return Pair{raw[j], VEC > 1 ? raw[j + 1] : 0.0f}; };
    auto values = [&](int n, int k, int j, Pair& h, Pair& g) {
      h = mul2(add2(pair(now[n].x[k], j), both(-now[n].mean)), both(now[n].rstd));
      g = pair(now[n].dy[k], j);
      if (SHIFTED) {
        const int c = at.column(k) + j;
        if (!at.has(c)) h.x = g.x = 0.0f;
        if (!at.has(c + 1)) h.y = g.y = 0.0f;
      }
    };
#pragma unroll
    for (int n = 0; n < N; ++n) {
      now[n] = next[n];
      const uint64_t then = row + (N + n) * at.step;
      if (then < at.rows) load(then, next[n]);
      Pair sg = both(0.0f), sgh = both(0.0f);
      if ((THREADS >= 32 && n == 0) || row + n * at.step < at.rows) {
#pragma unroll
        for (int k = 0; k < ITER; ++k) {
          if (at.any(at.column(k))) {
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
              Pair h, g;
              values(n, k, 2 * j, h, g);
              dw[k][j] = fma2(g, h, dw[k][j]);
              db[k][j] = add2(db[k][j], g);
              g = mul2(g, pair(w[k], 2 * j));
              sg = add2(sg, g);
              sgh = fma2(g, h, sgh);
            }
          }
        }
      }
      sums[n] = make_float2(sg.x + sg.y, sgh.x + sgh.y);
    }
    row_sums<THREADS>(sums, shared, turn++);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if ((THREADS < 32 || n > 0) && row + n * at.step >= at.rows) break;
      // (g w - m0 - h m1) rstd
      const float d = now[n].rstd;
      const Pair m0 = both(-sums[n].x * inv * d), m1 = both(-sums[n].y * inv * d);
#pragma unroll
      for (int k = 0; k < ITER; ++k) {
        if (at.any(at.column(k))) {
          float f[VEC];
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            Pair h, g;
            values(n, k, 2 * j, h, g);
            const Pair v = fma2(h, m1, fma2(mul2(g, pair(w[k], 2 * j)), both(d), m0));
            f[2 * j] = v.x;
            if (VEC > 1) f[2 * j + (VEC > 1)] = v.y;
          }
          at.store(dx, (row + n * at.step) * at.cols, at.column(k), f);
        }
      }
    }
  }
  auto one = [](const Pair& p, int j) { return j % 2 ? p.y : p.x; };
  if (!a.dweight && !a.dbias) return;
  float* part = a.workspace + (uint64_t)blockIdx.x * 2 * a.cols;
  if (R::kTogether > 1) {
    // the sums of a warp's rows, then those of the four warps, in their order
#pragma unroll
    for (int d = THREADS < 32 ? THREADS : 32; d < 32; d *= 2)
#pragma unroll
      for (int k = 0; k < ITER; ++k)
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          auto other = [&](const Pair& p) { return Pair{__shfl_xor_sync(~0u, p.x, d), __shfl_xor_sync(~0u, p.y, d)}; };
          dw[k][j] = add2(dw[k][j], other(dw[k][j]));
          db[k][j] = add2(db[k][j], other(db[k][j]));
        }
    constexpr int kLanes = THREADS < 32 ? THREADS : 32, kMany = kLanes * ITER * VEC, kWarps = R::kBlock / 32;
    __shared__ float together[2][R::kTogether > 1 ? kMany : 1];
    for (int w = 0; w < kWarps; ++w) {
      if (threadIdx.x / 32 == w && threadIdx.x % 32 < kLanes) {
#pragma unroll
        for (int k = 0; k < ITER; ++k)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int i = ((k * VEC + j) * kLanes + threadIdx.x % kLanes) % kMany, c = at.column(k) + j;
            const float pw = one(dw[k][j / 2], j) + (w ? together[0][i] : 0.0f);
            const float pb = one(db[k][j / 2], j) + (w ? together[1][i] : 0.0f);
            if (w < kWarps - 1) {
              together[0][i] = pw, together[1][i] = pb;
            } else if (c >= 0 && c < (int)at.cols) {
              part[c] = pw, part[a.cols + c] = pb;
            }
          }
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int k = 0; k < ITER; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = at.column(k) + j;
        if (c >= 0 && c < (int)at.cols) part[c] = one(dw[k][j / 2], j), part[a.cols + c] = one(db[k][j / 2], j);
      }
  }
}

// Long rows: dx of one row a CTA, read twice ...
template <class T, int VEC>
__global__ void __launch_bounds__(kLongThreads) norm_backward_long_kernel(const NormBackward a) {
  __shared__ float2 shared[2][kLongThreads / 32];
  pdl_wait();
  const uint64_t base = (uint64_t)blockIdx.x * a.cols;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* dy = static_cast<const T*>(a.dy) + base;
  const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x], inv = 1.0f / (float)a.cols;
  auto values = [&](uint64_t c, float (&h)[VEC], float (&g)[VEC]) {
    load_pack(x + c, h);
    load_pack(dy + c, g);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      h[j] = (h[j] - mean) * rstd;
      if (a.weight) g[j] *= param_at(a.weight, a.param_type, c + j);
    }
  };
  float sg = 0.0f, sgh = 0.0f;
  for (uint64_t c = threadIdx.x * VEC; c < a.cols; c += kLongThreads * VEC) {
    float h[VEC], g[VEC];
    values(c, h, g);
#pragma unroll
    for (int j = 0; j < VEC; ++j) sg += g[j], sgh += g[j] * h[j];
  }
  float2 sums[1] = {make_float2(sg, sgh)};
  row_sums<kLongThreads>(sums, shared, 0);
  T* dx = static_cast<T*>(a.dx) + base;
  for (uint64_t c = threadIdx.x * VEC; c < a.cols; c += kLongThreads * VEC) {
    float h[VEC], g[VEC];
    values(c, h, g);
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = (g[j] - sums[0].x * inv - h[j] * (sums[0].y * inv)) * rstd;
    store_pack(dx + c, g);
  }
}
// ... and the sums of a thread's columns over every parts-th row
template <class T, int VEC>
__global__ void __launch_bounds__(128) norm_backward_columns_kernel(const NormBackward a) {
  pdl_wait();
  const uint64_t parts = gridDim.x / ((a.cols + 128 * VEC - 1) / (128 * VEC)), part = blockIdx.x % parts;
  const uint64_t c = (blockIdx.x / parts * 128 + threadIdx.x) * VEC;
  if (c >= a.cols) return;
  float dw[VEC] = {}, db[VEC] = {};
#pragma unroll 4
  for (uint64_t row = part; row < a.rows; row += parts) {
    float h[VEC], g[VEC];
    load_pack(static_cast<const T*>(a.x) + row * a.cols + c, h);
    load_pack(static_cast<const T*>(a.dy) + row * a.cols + c, g);
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[j] += g[j] * ((h[j] - mean) * rstd), db[j] += g[j];
  }
  float* out = a.workspace + part * 2 * a.cols;
#pragma unroll
  for (int j = 0; j < VEC; ++j) out[c + j] = dw[j], out[a.cols + c + j] = db[j];
}

// The partial sums of all CTAs, 8 columns (a sector of memory) a block, each thread every 128th row; then the rows of
// threads, a warp for each result.
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* __restrict__ parts, uint64_t n, uint64_t cols,
                                                           void* dweight, void* dbias, int type) {
  constexpr int kCols = 8, kRows = 1024 / kCols;
  __shared__ float shared[2][kCols][kRows + 1];
  pdl_wait(parts);
  const uint32_t lane = threadIdx.x % kCols, r = threadIdx.x / kCols;
  const uint64_t c = (uint64_t)blockIdx.x * kCols + lane;
  float w = 0.0f, b = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (uint64_t i = r; i < n; i += kRows) {
      w += parts[i * 2 * cols + c];
      b += parts[i * 2 * cols + cols + c];
    }
  }
  shared[0][lane][r] = w, shared[1][lane][r] = b;
  __syncthreads();
  const uint32_t warp = threadIdx.x / 32, which = warp / kCols;
  const uint64_t mine = (uint64_t)blockIdx.x * kCols + warp % kCols;
  if (which < 2 && mine < cols) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows / 32; ++i) v += shared[which][warp % kCols][i * 32 + threadIdx.x % 32];
#pragma unroll
    for (int d = 16; d; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    void* out = which == 0 ? dweight : dbias;
    if (out && threadIdx.x % 32 == 0) param_to(out, type, mine, v);
  }
}

// ---- which kernel --------------------------------------------------------------------------------------------------
constexpr uint64_t kLongest = 8192;
constexpr int kHeld = 8;  // values of a row that a thread holds

template <class T>
bool whole_packs(uint64_t cols) {
  return cols * sizeof(T) % 16 == 0;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How a row's packs lie: of 16 bytes where all rows begin on them, shifted where only the first one does.  Else, and in
// rows of a pack or two that have nothing but ends, single values: up to 256 of them by a warp, more as a long row.
enum class Packs { kWhole, kShifted, kSingle, kLong };
Packs packs_of(int type, uint64_t cols, bool aligned) {
  const uint64_t size = type == CSW_TYPE_F32 ? 4 : 2, spare = 16 / size - 1;
  if (cols > kLongest) return Packs::kLong;
  if (aligned && cols * size % 16 == 0) return Packs::kWhole;
  if (aligned && cols * size >= 64 && cols + spare <= kLongest) return Packs::kShifted;
  return cols <= 32 * kHeld ? Packs::kSingle : Packs::kLong;
}
uint32_t period_of(int type, uint64_t cols, Packs packs) {
  if (packs != Packs::kShifted) return 1;
  uint32_t p = type == CSW_TYPE_F32 ? 4 : 8;
  for (uint64_t c = cols; p > 1 && c % 2 == 0; c /= 2) p /= 2;
  return p;
}
// threads of a row, the fewest that hold it with the masked values that a shifted one has more
int threads_of(int type, uint64_t cols, Packs packs) {
  const uint64_t held = cols + (packs == Packs::kShifted ? 16 / (type == CSW_TYPE_F32 ? 4 : 2) - 1 : 0);
  for (int t : {2, 8, 32, 64, 96, 128, 192, 256, 384, 512, 768})
    if (held <= (uint64_t)t * kHeld) return t;
  return 1024;
}

// CTAs that stay for all their rows, so that weights are read and sums written once each: as many as run at once.
unsigned blocks_of(uint64_t rows, int threads, uint32_t period, uint64_t on_sm) {
  const uint64_t block = threads <= 32 ? 128 : threads, together = block / threads;
  const uint64_t want = (rows + together * period - 1) / (together * period);  // CTAs of each shift
  const uint64_t most = std::max<uint64_t>((uint64_t)sm_count() * std::max<uint64_t>(std::min<uint64_t>(on_sm / block, 8), 1) / period, 1);
  return (unsigned)(std::min(want, most) * period);
}
constexpr uint64_t kLongParts = 64;

// f(pack's values, packs a thread, threads, shifted) for rows that are not long
template <class T, class F>
cudaError_t with_kernel(int threads, Packs packs, F&& f) {
  using std::integral_constant;
  constexpr int V = 16 / sizeof(T);
  using Yes = integral_constant<bool, true>;
  using No = integral_constant<bool, false>;
  using Pack16 = integral_constant<int, V>;
  using Iter16 = integral_constant<int, kHeld / V>;
  if (packs == Packs::kSingle) {
    using One = integral_constant<int, 1>;
    using All = integral_constant<int, kHeld>;
    return threads == 2   ? f(One(), All(), integral_constant<int, 2>(), No())
           : threads == 8 ? f(One(), All(), integral_constant<int, 8>(), No())
                          : f(One(), All(), integral_constant<int, 32>(), No());
  }
  switch (threads) {
#define CSW_THREADS(n) \
  case n: return packs == Packs::kWhole ? f(Pack16(), Iter16(), integral_constant<int, n>(), No()) \
                                        : f(Pack16(), Iter16(), integral_constant<int, n>(), Yes());
    CSW_THREADS(2)
    CSW_THREADS(8)
    CSW_THREADS(32)
    CSW_THREADS(64)
    CSW_THREADS(96)
    CSW_THREADS(128)
    CSW_THREADS(192)
    CSW_THREADS(256)
    CSW_THREADS(384)
    CSW_THREADS(512)
    CSW_THREADS(768)
    CSW_THREADS(1024)
#undef CSW_THREADS
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t norm_forward_launch(const NormForward& a, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  cudaError_t e = cudaErrorInvalidValue;
  with_type(a.type, [&](auto t) {
    using T = decltype(t);
    const Packs packs = packs_of(a.type, a.cols, aligned16(a.x) && aligned16(a.y) && aligned16(a.residual) &&
                                                     aligned16(a.sum) && aligned16(a.weight) && aligned16(a.bias));
    if (packs == Packs::kLong) {
      const bool whole = aligned16(a.x) && aligned16(a.y) && aligned16(a.residual) && aligned16(a.sum) && whole_packs<T>(a.cols);
      e = pdl_launch(whole ? norm_forward_long_kernel<T, 16 / sizeof(T)> : norm_forward_long_kernel<T, 1>, (unsigned)a.rows,
                     kLongThreads, 0, stream, a);
      return;
    }
    const uint32_t period = period_of(a.type, a.cols, packs);
    const int wide = threads_of(a.type, a.cols, packs);
    const unsigned grid = blocks_of(a.rows, wide, period, 1024);
    e = with_kernel<T>(wide, packs, [&](auto vec, auto iter, auto threads, auto shifted) {
      using R = Rows<T, vec.value, iter.value, threads.value, shifted.value>;
      return a.param_type == a.type
                 ? pdl_launch(norm_forward_kernel<T, T, vec.value, iter.value, threads.value, shifted.value>, grid,
                              R::kBlock, 0, stream, a, period)
                 : pdl_launch(norm_forward_kernel<T, float, vec.value, iter.value, threads.value, shifted.value>, grid,
                              R::kBlock, 0, stream, a, period);
    });
  });
  return e;
}

namespace {
uint64_t parts_of(int type, uint64_t rows, uint64_t cols, bool aligned) {
  const Packs packs = packs_of(type, cols, aligned);
  if (packs == Packs::kLong) return std::min(rows, kLongParts);
  return blocks_of(rows, threads_of(type, cols, packs), period_of(type, cols, packs), 768);
}
}  // namespace

uint64_t norm_backward_partials(uint64_t rows, uint64_t cols) {
  uint64_t most = 0;  // whichever type and alignment the call has
  for (int type : {CSW_TYPE_F32, CSW_TYPE_BF16})
    for (bool aligned : {false, true}) most = std::max(most, parts_of(type, rows, cols, aligned));
  return most;
}

cudaError_t norm_backward_launch(const NormBackward& a, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  const bool aligned = aligned16(a.x) && aligned16(a.dy) && aligned16(a.dx) && aligned16(a.weight);
  const uint64_t parts = parts_of(a.type, a.rows, a.cols, aligned);
  const bool sums = a.dweight || a.dbias;
  if (a.rows != 0) {
    e = cudaErrorInvalidValue;
    with_type(a.type, [&](auto t) {
      using T = decltype(t);
      const Packs packs = packs_of(a.type, a.cols, aligned);
      if (packs == Packs::kLong) {
        constexpr int V = 16 / sizeof(T);
        const bool whole = aligned && whole_packs<T>(a.cols);
        const uint64_t across = 128 * (whole ? V : 1);  // columns of a CTA
        e = pdl_launch(whole ? norm_backward_long_kernel<T, V> : norm_backward_long_kernel<T, 1>, (unsigned)a.rows,
                       kLongThreads, 0, stream, a);
        if (e == cudaSuccess && sums)
          e = pdl_launch(whole ? norm_backward_columns_kernel<T, V> : norm_backward_columns_kernel<T, 1>,
                         (unsigned)((a.cols + across - 1) / across * parts), 128, 0, stream, a);
        return;
      }
      const uint32_t period = period_of(a.type, a.cols, packs);
      e = with_kernel<T>(threads_of(a.type, a.cols, packs), packs, [&](auto vec, auto iter, auto threads, auto shifted) {
        using R = Rows<T, vec.value, iter.value, threads.value, shifted.value>;
        return a.param_type == a.type
                   ? pdl_launch(norm_backward_kernel<T, T, vec.value, iter.value, threads.value, shifted.value>,
                                (unsigned)parts, R::kBlock, 0, stream, a, period)
                   : pdl_launch(norm_backward_kernel<T, float, vec.value, iter.value, threads.value, shifted.value>,
                                (unsigned)parts, R::kBlock, 0, stream, a, period);
      });
    });
  }
  if (e == cudaSuccess && sums)
    e = pdl_launch(norm_reduce_kernel, (unsigned)((a.cols + 7) / 8), 1024, 0, stream, a.workspace, parts, a.cols,
                   a.dweight, a.dbias, a.param_type);
  return e;
}

}  // namespace csw
