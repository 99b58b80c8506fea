// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / c,  var = sum (x - mean)^2 / c,  rstd = 1 / sqrt(var + eps),  h = (x - mean) rstd
//   y = h w + b
//   dx = rstd (g - sum g / c - h sum(g h) / c) with g = dy w;  dw = sum over rows of dy h,  db = sum over rows of dy
//
// What bounds it: HBM.  A row is read once and held in registers by the threads that share it (a warp up to 1024
// values, a CTA of 128 or 512 threads up to 4096 and 16384), so that the variance is summed from the centred values, a
// second time over registers and not over memory.  Longer rows are read again, from L2.
//
// Backward, each thread keeps the sums of dw and db of its own columns over all rows that its CTA takes; they go to
// memory once per CTA, in a fixed order, and a second launch adds them up.  No atomics: the same call gives the same bits.
#include <cuda_runtime.h>

#include <algorithm>

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
template <int N>
__device__ __forceinline__ void params_at(const void* p, int type, uint64_t i, float (&f)[N]) {
  if (N == 1) {
    f[0] = param_at(p, type, i);
  } else if (type == CSW_TYPE_F32) {
    const float* q = static_cast<const float*>(p) + i;
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 k = *reinterpret_cast<const float4*>(q + j);
      f[j] = k.x, f[j + 1] = k.y, f[j + 2] = k.z, f[j + 3] = k.w;
    }
  } else if (type == CSW_TYPE_F16) {
    load_pack(static_cast<const __half*>(p) + i, f);
  } else {
    load_pack(static_cast<const __nv_bfloat16*>(p) + i, f);
  }
}

// Sum over the THREADS threads that share a row (a warp, or the whole CTA); all of them get it.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* shared) {
#pragma unroll
  for (int d = 16; d; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (THREADS > 32) {
    __syncthreads();  // the last use of `shared` is over
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) v += shared[i];
  }
  return v;
}
template <int THREADS>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* shared) {
#pragma unroll
  for (int d = 16; d; d /= 2) {
    a += __shfl_xor_sync(0xffffffffu, a, d);
    b += __shfl_xor_sync(0xffffffffu, b, d);
  }
  if (THREADS > 32) {
    __syncthreads();
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) a += shared[i].x, b += shared[i].y;
  }
  return make_float2(a, b);
}

template <class T, int VEC, int ITER, int THREADS>
struct Shape {
  static constexpr int kRowThreads = THREADS;
  static constexpr int kBlock = THREADS < 128 ? 128 : THREADS;
  static constexpr int kRowsPerBlock = kBlock / THREADS;
};

// A row in the registers of THREADS threads: thread t holds VEC values from column (k THREADS + t) VEC on, for each k.
template <class T, int VEC, int ITER, int THREADS>
__global__ void __launch_bounds__(Shape<T, VEC, ITER, THREADS>::kBlock) norm_forward_kernel(const NormForward a) {
  using S = Shape<T, VEC, ITER, THREADS>;
  __shared__ float shared[THREADS > 32 ? THREADS / 32 : 1];
  const T* x = static_cast<const T*>(a.x);
  const T* residual = static_cast<const T*>(a.residual);
  pdl_wait(x);
  pdl_behind(residual);
  const uint32_t t = threadIdx.x % THREADS;
  const uint32_t cols = (uint32_t)a.cols;
  const uint64_t row = (uint64_t)blockIdx.x * S::kRowsPerBlock + threadIdx.x / THREADS;
  if (row >= a.rows) return;  // a whole warp, or no thread of the CTA
  const uint64_t base = row * a.cols;
  float v[ITER][VEC];
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const uint32_t c = (k * THREADS + t) * VEC;
    if (c < cols) {
      load_pack(x + base + c, v[k]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = 0.0f;
    }
  }
  if (residual) {
    T* sum = static_cast<T*>(a.sum);
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const uint32_t c = (k * THREADS + t) * VEC;
      if (c < cols) {
        float r[VEC];
        load_pack(residual + base + c, r);
        // what is normed, and what backward reads, is the sum as it is held
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k][j] = widen(narrow<T>(v[k][j] + r[j]));
        store_pack(sum + base + c, v[k]);
      }
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < ITER; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += v[k][j];
  const float mean = row_sum<THREADS>(s, shared) / (float)cols;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const uint32_t c = (k * THREADS + t) * VEC;
    if (c < cols) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[k][j] -= mean;
        s += v[k][j] * v[k][j];
      }
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<THREADS>(s, shared) / (float)cols + a.eps);
  if (t == 0) a.mean[row] = mean, a.rstd[row] = rstd;
  T* y = static_cast<T*>(a.y);
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const uint32_t c = (k * THREADS + t) * VEC;
    if (c < cols) {
      float w[VEC], b[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = 1.0f, b[j] = 0.0f;
      if (a.weight) params_at(a.weight, a.param_type, c, w);
      if (a.bias) params_at(a.bias, a.param_type, c, b);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = v[k][j] * rstd * w[j] + b[j];
      store_pack(y + base + c, v[k]);
    }
  }
}

// Rows beyond 16384 values: read three times, one value a thread and step.
constexpr int kLongThreads = 512;
template <class T>
__global__ void __launch_bounds__(kLongThreads) norm_forward_long_kernel(const NormForward a) {
  __shared__ float shared[kLongThreads / 32];
  pdl_wait();
  const uint64_t base = (uint64_t)blockIdx.x * a.cols;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* residual = a.residual ? static_cast<const T*>(a.residual) + base : nullptr;
  T* sum = residual ? static_cast<T*>(a.sum) + base : nullptr;
  float s = 0.0f;
  for (uint64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    float v = widen(x[c]);
    if (residual) {
      const T held = narrow<T>(v + widen(residual[c]));
      sum[c] = held;
      v = widen(held);
    }
    s += v;
  }
  const T* src = residual ? sum : x;  // a thread reads back what it wrote itself
  const float mean = row_sum<kLongThreads>(s, shared) / (float)a.cols;
  s = 0.0f;
  for (uint64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float v = widen(src[c]) - mean;
    s += v * v;
  }
  const float rstd = 1.0f / sqrtf(row_sum<kLongThreads>(s, shared) / (float)a.cols + a.eps);
  if (threadIdx.x == 0) a.mean[blockIdx.x] = mean, a.rstd[blockIdx.x] = rstd;
  T* y = static_cast<T*>(a.y) + base;
  for (uint64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float w = a.weight ? param_at(a.weight, a.param_type, c) : 1.0f;
    const float b = a.bias ? param_at(a.bias, a.param_type, c) : 0.0f;
    y[c] = narrow<T>((widen(src[c]) - mean) * rstd * w + b);
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------
// One CTA takes rows r, r + gridDim kRowsPerBlock, ...; workspace row blockIdx.x receives its sums: dw, then db.
template <class T, int VEC, int ITER, int THREADS>
__global__ void __launch_bounds__(Shape<T, VEC, ITER, THREADS>::kBlock) norm_backward_kernel(const NormBackward a) {
  using S = Shape<T, VEC, ITER, THREADS>;
  __shared__ float2 shared[THREADS > 32 ? THREADS / 32 : 1];
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  pdl_wait(x);
  pdl_behind(dy);
  const uint32_t t = threadIdx.x % THREADS;
  const uint32_t cols = (uint32_t)a.cols;
  const float inv = 1.0f / (float)cols;
  float dw[ITER][VEC], db[ITER][VEC];
#pragma unroll
  for (int k = 0; k < ITER; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[k][j] = db[k][j] = 0.0f;
  for (uint64_t row = (uint64_t)blockIdx.x * S::kRowsPerBlock + threadIdx.x / THREADS; row < a.rows;
       row += (uint64_t)gridDim.x * S::kRowsPerBlock) {
    const uint64_t base = row * a.cols;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float h[ITER][VEC], g[ITER][VEC];
    float sg = 0.0f, sgh = 0.0f;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const uint32_t c = (k * THREADS + t) * VEC;
      if (c < cols) {
        load_pack(x + base + c, h[k]);
        load_pack(dy + base + c, g[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const uint32_t c = (k * THREADS + t) * VEC;
      if (c < cols) {
        float w[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = 1.0f;
        if (a.weight) params_at(a.weight, a.param_type, c, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          h[k][j] = (h[k][j] - mean) * rstd;
          dw[k][j] += g[k][j] * h[k][j];
          db[k][j] += g[k][j];
          g[k][j] *= w[j];
          sg += g[k][j];
          sgh += g[k][j] * h[k][j];
        }
      }
    }
    const float2 s = row_sum2<THREADS>(sg, sgh, shared);
    const float m0 = s.x * inv, m1 = s.y * inv;
    T* dx = static_cast<T*>(a.dx) + base;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const uint32_t c = (k * THREADS + t) * VEC;
      if (c < cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[k][j] = (g[k][j] - m0 - h[k][j] * m1) * rstd;
        store_pack(dx + c, g[k]);
      }
    }
  }
  if (!a.dweight && !a.dbias) return;
  float* part = a.workspace + (uint64_t)blockIdx.x * 2 * a.cols;
  if (S::kRowsPerBlock > 1) {
    // the warps' sums, added in the order of the warps
    __shared__ float sums[S::kRowsPerBlock > 1 ? 2 * 32 * ITER * VEC : 1];
    for (int w = 0; w < S::kRowsPerBlock; ++w) {
      if (threadIdx.x / THREADS == w) {
#pragma unroll
        for (int k = 0; k < ITER; ++k)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int i = (k * VEC + j) * 32 + t;
            const float pw = dw[k][j] + (w ? sums[i] : 0.0f);
            const float pb = db[k][j] + (w ? sums[i + 32 * ITER * VEC] : 0.0f);
            if (w < S::kRowsPerBlock - 1) {
              sums[i] = pw, sums[i + 32 * ITER * VEC] = pb;
            } else {
              const uint32_t c = (k * THREADS + t) * VEC + j;
              if (c < cols) part[c] = pw, part[a.cols + c] = pb;
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
        const uint32_t c = (k * THREADS + t) * VEC + j;
        if (c < cols) part[c] = dw[k][j], part[a.cols + c] = db[k][j];
      }
  }
}

// Long rows: dx of one row a CTA, read twice ...
template <class T>
__global__ void __launch_bounds__(kLongThreads) norm_backward_long_kernel(const NormBackward a) {
  __shared__ float2 shared[kLongThreads / 32];
  pdl_wait();
  const uint64_t base = (uint64_t)blockIdx.x * a.cols;
  const T* x = static_cast<const T*>(a.x) + base;
  const T* dy = static_cast<const T*>(a.dy) + base;
  const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x], inv = 1.0f / (float)a.cols;
  float sg = 0.0f, sgh = 0.0f;
  for (uint64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float g = widen(dy[c]) * (a.weight ? param_at(a.weight, a.param_type, c) : 1.0f);
    sg += g;
    sgh += g * ((widen(x[c]) - mean) * rstd);
  }
  const float2 s = row_sum2<kLongThreads>(sg, sgh, shared);
  T* dx = static_cast<T*>(a.dx) + base;
  for (uint64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float g = widen(dy[c]) * (a.weight ? param_at(a.weight, a.param_type, c) : 1.0f);
    dx[c] = narrow<T>((g - s.x * inv - (widen(x[c]) - mean) * rstd * (s.y * inv)) * rstd);
  }
}
// ... and the sums of a thread's column over every gridDim.y-th row
template <class T>
__global__ void __launch_bounds__(128) norm_backward_columns_kernel(const NormBackward a) {
  pdl_wait();
  const uint64_t parts = gridDim.x / ((a.cols + 127) / 128), part = blockIdx.x % parts;
  const uint64_t c = blockIdx.x / parts * 128 + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.0f, db = 0.0f;
  for (uint64_t row = part; row < a.rows; row += parts) {
    const float g = widen(static_cast<const T*>(a.dy)[row * a.cols + c]);
    dw += g * ((widen(static_cast<const T*>(a.x)[row * a.cols + c]) - a.mean[row]) * a.rstd[row]);
    db += g;
  }
  float* out = a.workspace + part * 2 * a.cols;
  out[c] = dw, out[a.cols + c] = db;
}

// The partial sums of all CTAs, 32 columns a block, each thread every 8th row; then the 8 rows of threads in order.
__global__ void __launch_bounds__(256) norm_reduce_kernel(const float* __restrict__ parts, uint64_t n, uint64_t cols,
                                                          void* dweight, void* dbias, int type) {
  __shared__ float shared[2][8][32];
  pdl_wait(parts);
  const uint32_t lane = threadIdx.x % 32, r = threadIdx.x / 32;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  float w = 0.0f, b = 0.0f;
  if (c < cols) {
    for (uint64_t i = r; i < n; i += 8) {
      w += parts[i * 2 * cols + c];
      b += parts[i * 2 * cols + cols + c];
    }
  }
  shared[0][r][lane] = w, shared[1][r][lane] = b;
  __syncthreads();
  if (r < 2 && c < cols) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += shared[r][i][lane];
    void* out = r == 0 ? dweight : dbias;
    if (out) param_to(out, type, c, s);
  }
}

// ---- which kernel --------------------------------------------------------------------------------------------------
constexpr uint64_t kLongest = 16384;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
template <class T>
bool whole_packs(uint64_t cols) {
  return cols * sizeof(T) % 16 == 0;
}

// f<values a thread holds, threads of a row> for rows of up to kLongest values
template <class F>
cudaError_t with_shape(uint64_t cols, F&& f) {
  using std::integral_constant;
#define CSW_SHAPE(n, threads) \
  if (cols <= (uint64_t)n * threads) return f(integral_constant<int, n>(), integral_constant<int, threads>())
  CSW_SHAPE(8, 32);
  CSW_SHAPE(16, 32);
  CSW_SHAPE(24, 32);
  CSW_SHAPE(32, 32);
  CSW_SHAPE(16, 128);
  CSW_SHAPE(32, 128);
  CSW_SHAPE(16, 512);
  CSW_SHAPE(32, 512);
#undef CSW_SHAPE
  return cudaErrorInvalidValue;
}
unsigned rows_per_block(uint64_t cols) { return cols <= 1024 ? 4 : 1; }

// CTAs of a backward pass: they stay for all their rows, so that the sums leave them once.
unsigned backward_blocks(uint64_t rows, uint64_t cols) {
  const uint64_t want = (rows + rows_per_block(cols) - 1) / rows_per_block(cols);
  const uint64_t resident = (uint64_t)sm_count() * (cols <= 1024 ? 3 : cols <= 4096 ? 3 : 1);
  return (unsigned)std::min(want, resident);
}
constexpr uint64_t kLongParts = 64;

}  // namespace

cudaError_t norm_forward_launch(const NormForward& a, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  cudaError_t e = cudaErrorInvalidValue;
  with_type(a.type, [&](auto t) {
    using T = decltype(t);
    if (a.cols > kLongest) {
      e = pdl_launch(norm_forward_long_kernel<T>, (unsigned)a.rows, kLongThreads, 0, stream, a);
      return;
    }
    const bool vec = whole_packs<T>(a.cols) && aligned16(a.x) && aligned16(a.y) && aligned16(a.residual) &&
                     aligned16(a.sum) && aligned16(a.weight) && aligned16(a.bias);
    const unsigned grid = (unsigned)((a.rows + rows_per_block(a.cols) - 1) / rows_per_block(a.cols));
    e = with_shape(a.cols, [&](auto held, auto threads) {
      constexpr int V = 16 / sizeof(T), H = held.value, R = threads.value;
      constexpr int B = Shape<T, V, 1, R>::kBlock;
      return vec ? pdl_launch(norm_forward_kernel<T, V, H / V, R>, grid, B, 0, stream, a)
                 : pdl_launch(norm_forward_kernel<T, 1, H, R>, grid, B, 0, stream, a);
    });
  });
  return e;
}

uint64_t norm_backward_partials(uint64_t rows, uint64_t cols) {
  if (cols > kLongest) return std::min(rows, kLongParts);
  return backward_blocks(rows, cols);
}

cudaError_t norm_backward_launch(const NormBackward& a, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  const uint64_t parts = norm_backward_partials(a.rows, a.cols);
  const bool sums = a.dweight || a.dbias;
  if (a.rows != 0) {
    e = cudaErrorInvalidValue;
    with_type(a.type, [&](auto t) {
      using T = decltype(t);
      if (a.cols > kLongest) {
        e = pdl_launch(norm_backward_long_kernel<T>, (unsigned)a.rows, kLongThreads, 0, stream, a);
        if (e == cudaSuccess && sums)
          e = pdl_launch(norm_backward_columns_kernel<T>, (unsigned)((a.cols + 127) / 128 * parts), 128, 0, stream, a);
        return;
      }
      const bool vec = whole_packs<T>(a.cols) && aligned16(a.x) && aligned16(a.dy) && aligned16(a.dx) &&
                       aligned16(a.weight);
      e = with_shape(a.cols, [&](auto held, auto threads) {
        constexpr int V = 16 / sizeof(T), H = held.value, R = threads.value;
        constexpr int B = Shape<T, V, 1, R>::kBlock;
        return vec ? pdl_launch(norm_backward_kernel<T, V, H / V, R>, (unsigned)parts, B, 0, stream, a)
                   : pdl_launch(norm_backward_kernel<T, 1, H, R>, (unsigned)parts, B, 0, stream, a);
      });
    });
  }
  if (e == cudaSuccess && sums)
    e = pdl_launch(norm_reduce_kernel, (unsigned)((a.cols + 31) / 32), 256, 0, stream, a.workspace, parts, a.cols,
                   a.dweight, a.dbias, a.param_type);
  return e;
}

}  // namespace csw
