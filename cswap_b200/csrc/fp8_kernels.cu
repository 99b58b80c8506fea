// Matrices in 8-bit floating point, and their products on the tensor cores.
//
// Format.  A block of 128 x 128 values has a scale 2^E, held as the byte E + 127.  With a the block's largest finite
// magnitude, E is the least for which a <= 448 2^E, but -126 at least; a value's code is the e4m3 number nearest to x 2^-E,
// ties to even, and NaN for a NaN or an infinity.
//
// Why these blocks.  A floating-point code keeps its three bits of mantissa down to 2^-14.8 of the block's largest value, so
// that a block as large as this loses nothing against a row of 128 as long as its values lie within that; a power of two
// scales exactly, and the tensor cores multiply it in themselves (block_scale), so that sums stay in tensor memory over the
// whole reduction.  And a square block is the same block for the product that reads the matrix along its rows and for the one
// that reads it across: forward, the gradient of the input and that of the weight (y = x W^T, dx = dy W, dW = dy^T x) take
// the same codes, and what a layer keeps is what its product read.
#include "fp8_kernels.h"

#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "internal.h"
#include "pdl.cuh"
#include "tensor_core.cuh"
#include "values.cuh"
#include "waits.h"

namespace csw {
namespace {

constexpr int kBlock = (int)kFp8Block;

// ---- quantizing -----------------------------------------------------------------------------------------------------
// A CTA a block, its values in registers as they are stored: 16 threads a row of 8 values each, 16 rows at a time, so that a
// value is read once.  The columns' sums (what a bias's gradient is) leave each block of rows once and are added up in order.
constexpr int kQuantizeThreads = 256, kRowsEach = kBlock * kBlock / 8 / kQuantizeThreads;

// the scale of a block whose largest magnitude has these bits, and what its values are multiplied with
__device__ __forceinline__ int exponent_of(uint32_t top) {
  return max((int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);  // 448 is 1.75 2^8
}
__device__ __forceinline__ float power_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// 8 values of a row, in words; the magnitude of a word's values is compared as whole numbers
template <class T>
struct Eight {
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t w[kWords];
  __device__ __forceinline__ float operator[](int j) const { return value_of<T>(w, j); }
  __device__ __forceinline__ void load(const T* from) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(from) + i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void load(const T* from, int live) {
    using Bits = typename Words<sizeof(T)>::type;
    uint32_t bits[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bits[j] = 0;
      if (j < live) bits[j] = reinterpret_cast<const Bits*>(from)[j];
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = sizeof(T) == 4 ? bits[i] : bits[2 * i] | bits[2 * i + 1] << 16;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // from any place, by the packs of 16 bytes that it lies in
  __device__ __forceinline__ void load_across(const T* from) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(from);
    const uint4* packs = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
    uint32_t v[kWords + 4];
#pragma unroll
    for (int i = 0; i <= kWords / 4; ++i) {
      const uint4 k = packs[i];
      v[4 * i] = k.x, v[4 * i + 1] = k.y, v[4 * i + 2] = k.z, v[4 * i + 3] = k.w;
    }
    if (at & 8) {
#pragma unroll
      for (int i = 0; i < kWords + 2; ++i) v[i] = v[i + 2];
    }
    if (at & 4) {
#pragma unroll
      for (int i = 0; i < kWords + 1; ++i) v[i] = v[i + 1];
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = sizeof(T) == 2 && (at & 2) ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      m = sizeof(T) == 4 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
    return sizeof(T) == 4 ? m : max(m & 0xffffu, m >> 16);
  }
};
// the first magnitude that is no number
template <class T>
constexpr uint32_t kNoNumber = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;

__device__ __forceinline__ void store_as(void* to, int type, uint64_t i, float v) {
  if (type == 0) static_cast<float*>(to)[i] = v;
  else if (type == 1) static_cast<__half*>(to)[i] = narrow<__half>(v);
  else static_cast<__nv_bfloat16*>(to)[i] = narrow<__nv_bfloat16>(v);
}

template <class T, bool SUMS>
__global__ void __launch_bounds__(kQuantizeThreads) fp8_quantize_kernel(const T* __restrict__ x, uint64_t rows, uint64_t cols,
                                                                        uint64_t stride, bool packs, uint8_t* codes,
                                                                        uint64_t code_stride, uint8_t* scales, void* sums,
                                                                        int sums_type) {
  __shared__ uint32_t tops[kQuantizeThreads / 32];
  __shared__ float column[SUMS ? 16 : 1][SUMS ? kBlock : 1];
  pdl_trigger_if_few();
  pdl_wait(x);
  const uint32_t blocks = (uint32_t)((cols + kBlock - 1) / kBlock);
  const uint64_t bi = blockIdx.x / blocks, bj = blockIdx.x % blocks;
  const int t = threadIdx.x, r0 = t / 16, c = t % 16 * 8;
  const uint64_t row = bi * kBlock + r0, col = bj * kBlock + c;
  const T* from = x + row * stride + col;
  Eight<T> v[kRowsEach];
  if (packs && (bi + 1) * kBlock <= rows && (bj + 1) * kBlock <= cols) {
#pragma unroll
    for (int i = 0; i < kRowsEach; ++i) v[i].load(from + 16 * i * stride);
  } else {
    // Rows that begin anywhere, or end in the block: packs that a value lies in are read whole where they are x's.
    const int live = (int)min((int64_t)8, max((int64_t)cols - (int64_t)col, (int64_t)0));  // of this thread's columns
    const int here = row < rows ? (int)min((rows - 1 - row) / 16, (uint64_t)(kRowsEach - 1)) : -1;  // its last row
    const uintptr_t begin = reinterpret_cast<uintptr_t>(x), end = begin + ((rows - 1) * stride + cols) * sizeof(T);
    const uintptr_t first = reinterpret_cast<uintptr_t>(from), last = reinterpret_cast<uintptr_t>(from + 16 * here * (int64_t)stride);
    if (live == 8 && here >= 0 && (first & ~(uintptr_t)15) >= begin && (last & ~(uintptr_t)15) + 8 * sizeof(T) + 16 <= end) {
#pragma unroll
      for (int i = 0; i < kRowsEach; ++i) {
        v[i].load_across(from + 16 * min(i, here) * stride);
        if (i > here) v[i].clear();
      }
    } else {
#pragma unroll
      for (int i = 0; i < kRowsEach; ++i) v[i].load(from + 16 * i * stride, i <= here ? live : 0);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i) top = max(top, v[i].top());
  const bool odd = top >= kNoNumber<T>;
  if (odd) {
    top = 0;
#pragma unroll
    for (int i = 0; i < kRowsEach; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t bits = __float_as_uint(v[i][j]) & 0x7fffffffu;
        top = max(top, bits < 0x7f800000u ? bits : 0u);
      }
  } else if constexpr (sizeof(T) == 2) {
    top = __float_as_uint(value_of<T>(&top, 0));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (t % 32 == 0) tops[t / 32] = top;
  if constexpr (SUMS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = v[0][j];
#pragma unroll
      for (int i = 1; i < kRowsEach; ++i) s += v[i][j];
      column[r0][c + j] = s;
    }
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantizeThreads / 32; ++w) top = max(top, tops[w]);
  const int e = exponent_of(top);
  if (t == 0) scales[blockIdx.x] = (uint8_t)(e + 127);
  if constexpr (SUMS) {
    if (t < kBlock && bj * kBlock + t < cols) {
      float s = column[0][t];
#pragma unroll
      for (int i = 1; i < 16; ++i) s += column[i][t];
      store_as(sums, sums_type, bi * cols + bj * kBlock + t, s);
    }
  }
  if (col >= cols) return;
  const float factor = power_of(-e);
  uint8_t* to = codes + row * code_stride + col;
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i) {
    uint32_t word[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float2 f = {v[i][j] * factor, v[i][j + 1] * factor};
      if (odd) {  // the conversion would make the largest number of an infinity
        if (isinf(f.x)) f.x = NAN;
        if (isinf(f.y)) f.y = NAN;
      }
      word[j / 4] |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (j % 4 * 8);
    }
    // up to 7 bytes behind the last column belong to the row's stride
    if (row + 16 * i < rows) *reinterpret_cast<uint2*>(to + 16 * i * code_stride) = make_uint2(word[0], word[1]);
  }
}

// The sums of the blocks of rows, in their order: 8 threads a column, each a part of the blocks.
__global__ void __launch_bounds__(256) fp8_sums_kernel(const float* __restrict__ partials, uint64_t parts, uint64_t cols,
                                                       void* sums, int type) {
  __shared__ float part[8][32];
  pdl_trigger_if_few();
  pdl_wait(partials);
  const uint64_t col = (uint64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const int p = threadIdx.x / 32;
  float s = 0.0f;
  if (col < cols)
#pragma unroll 8
    for (uint64_t i = p; i < parts; i += 8) s += partials[i * cols + col];
  part[p][threadIdx.x % 32] = s;
  __syncthreads();
  if (p || col >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
  store_as(sums, type, col, s);
}

// The same way back, for four neighbours of a row's first half and four of its second, so that a row's float32 values leave as
// whole lines (eight neighbours a thread: 70 us for 67 million float32 values where these take 53).
template <class T>
__global__ void __launch_bounds__(kQuantizeThreads) fp8_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                          uint64_t code_stride,
                                                                          const uint8_t* __restrict__ scales, uint64_t rows,
                                                                          uint64_t cols, bool packs, T* out) {
  constexpr int kNext = kBlock / 2;
  pdl_trigger_if_few();
  pdl_wait(codes);
  pdl_behind(scales);
  const uint32_t blocks = (uint32_t)((cols + kBlock - 1) / kBlock);
  const uint64_t row = blockIdx.x / blocks * (uint64_t)kBlock + threadIdx.x / 16;
  const uint64_t col = blockIdx.x % blocks * (uint64_t)kBlock + threadIdx.x % 16 * 4;
  const uint32_t byte = scales[blockIdx.x];  // 0 and 255 are no quantizer's, but a format's: 2^-127 and NaN
  const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
  const uint8_t* from = codes + row * code_stride + col;
  uint32_t word[kRowsEach][2];
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i)
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // up to 3 bytes behind the last column belong to the row's stride
      word[i][q] = 0;
      if (row + 16 * i < rows && col + q * kNext < cols)
        word[i][q] = *reinterpret_cast<const uint32_t*>(from + 16 * i * code_stride + q * kNext);
    }
  T* to = out + row * cols + col;
#pragma unroll
  for (int i = 0; i < kRowsEach; ++i, to += 16 * cols) {
    if (row + 16 * i >= rows) return;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word[i][q] >> 8 * j), __NV_E4M3);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
        f[j] = v.x * scale, f[j + 1] = v.y * scale;
      }
      if (packs && col + q * kNext < cols) {
        store_pack(to + q * kNext, f);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + q * kNext + j < cols) to[q * kNext + j] = narrow<T>(f[j]);
      }
    }
  }
}

// ---- products -------------------------------------------------------------------------------------------------------
using namespace tc;

constexpr uint32_t kTileBytes = kBlock * kBlock;
constexpr int kThreads = 256;

// Tiles of 128 x BN of the result, 128 of the reduction at a time.  A stage of the ring: the row operand's tile and the column
// operand's (whole tiles of 128 x 128 where that is read across its rows); behind all stages two batches of scales; behind them,
// what the CTAs of a cluster send.  A batch has the scales of 16 blocks of the reduction: a word has four blocks', of which a
// product names one, and 128 rows or columns have 512 bytes of a word each.  (A batch a block bounded the kernel: the fence
// between writing it and the tensor cores' reading takes 500 clocks, in which products of 128 x 128 take 256.)  Where the
// stages were, in the end, lie the tile's sums: row by row with 16 bytes between them, so that a warp's 32 rows are in different
// banks, or, for a result with the operands exchanged, column by column.
constexpr int kMostStages = 10, kBatch = 16;
template <int BN>
struct Plan {
  static constexpr int kPanels = (BN + kBlock - 1) / kBlock;  // tiles of 128 columns
  static constexpr int kWordColumns = 4 * (1 + kPanels);  // of tensor memory, of a word of scales
  static constexpr uint32_t kWordBytes = 512 * (1 + kPanels), kBatchBytes = kBatch / 4 * kWordBytes;
  static constexpr int kNeeded = BN + 2 * (kBatch / 4) * kWordColumns;  // columns of tensor memory: sums, then two batches
  static constexpr int kColumns = kNeeded > 256 ? 512 : kNeeded > 128 ? 256 : kNeeded > 64 ? 128 : 64;
  static constexpr int kPitch = BN + 4;
  static constexpr uint32_t kSums = kBlock * kPitch * 4;
  __host__ __device__ static constexpr uint32_t stage(bool across) {
    return kTileBytes + (across ? kPanels * kTileBytes : BN * kBlock);
  }
  // As many stages as there is work for, and room: half an SM's shared memory where a CTA is not alone on it.
  static uint32_t stages(bool across, bool alone, bool parts, uint32_t steps) {
    const uint32_t room = (alone ? 224u : 110u) * 1024 - (parts ? kSums : 0) - 2 * kBatchBytes, each = stage(across);
    const uint32_t least = (kSums + stage(across) - 1) / stage(across);  // the sums have to fit
    return std::max(std::min({room / each, steps, (uint32_t)kMostStages}), least);
  }
  static size_t shared(bool across, bool parts, uint32_t stages) {
    return stages * stage(across) + 2 * kBatchBytes + (parts ? kSums : 0) + 1024;
  }
};
// The place in a ring of stages, and the round.
struct Turn {
  uint32_t stages, s = 0, round = 0;
  __device__ __forceinline__ void next() {
    if (++s == stages) s = 0, ++round;
  }
};

struct Operand {
  CUtensorMap map;
  const uint8_t* scales;
  uint32_t scale_step, scale_k_step;  // from one block to the next, along the rows or columns of the result and the reduction
  bool across;                        // stored with the reduction over its rows
};
struct Product {
  Operand r, c;          // whose rows are the tile's rows and columns
  uint32_t m, n, steps;  // rows and columns of tiles together; blocks of the reduction
  uint32_t row_tiles, col_tiles, parts, stages;
  // the result: [m][n], or [n][m] where the operands were exchanged; the bias goes by its last axis
  void* out;
  const void* bias;
  int type, bias_type;
  bool exchanged, packs;  // packs: rows of the result begin on 16 bytes
  // the column operand as values that are yet to be quantized: p.n rows, x_cols of the reduction, x_stride apart
  const void* x;
  uint64_t x_stride;
  uint32_t x_cols;
  bool x_packs;  // four of them lie so that they are one load
  long long patience;
  bool idle;
  uint32_t* status;
};

__device__ __forceinline__ float bias_at(const Product& p, uint32_t i) {
  return p.bias_type == 0   ? static_cast<const float*>(p.bias)[i]
         : p.bias_type == 1 ? widen(static_cast<const __half*>(p.bias)[i])
                            : widen(static_cast<const __nv_bfloat16*>(p.bias)[i]);
}
// four values of a row of the result, `gap` columns from one to the next; neighbours (1) where rows begin on 16 bytes
template <class T>
__device__ __forceinline__ void emit(const Product& p, uint32_t row, uint32_t col, uint32_t gap, const float (&f)[4]) {
  const uint32_t cols = p.exchanged ? p.m : p.n;
  T* out = static_cast<T*>(p.out) + (uint64_t)row * cols + col;
  if (p.packs && col + 4 <= cols) {
    store_pack(out, f);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j * gap < cols) out[j * gap] = narrow<T>(f[j]);
  }
}

// Sums in shared memory on their way out: `parts` copies of rows of the result, `pitch` floats from one to the next, added in
// their order.  Four values a lane, several rows of a warp at once; where rows of the result begin anywhere, the values of a lane
// lie apart, so that a warp's stores of one value each are still one run.
struct Sums {
  const float* at;
  uint32_t parts, rows, pitch, width;
};
template <class T>
__device__ __forceinline__ void emit_rows(const Product& p, const Sums& s, uint32_t row, uint32_t col) {
  constexpr int kAtOnce = 4;
  const uint32_t all = p.exchanged ? p.n : p.m, cols = p.exchanged ? p.m : p.n;
  const uint32_t lanes = min(s.width / 4, 32u), group = 32 / lanes;  // of a row; rows of a warp
  const uint32_t mine = threadIdx.x / 32 * group + threadIdx.x % 32 / lanes, step = blockDim.x / 32 * group;
  const uint32_t gap = p.packs ? 1 : lanes;
  for (uint32_t c = threadIdx.x % lanes * (p.packs ? 4 : 1); c < s.width && col + c < cols; c += lanes * 4) {
    float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + c + j * gap < cols) b[j] = bias_at(p, col + c + j * gap);
    }
    auto four = [&](const float* from) {
      return p.packs ? *reinterpret_cast<const float4*>(from) : make_float4(from[0], from[gap], from[2 * gap], from[3 * gap]);
    };
    for (uint32_t i = mine; i < s.rows && row + i < all; i += kAtOnce * step) {
      float4 f[kAtOnce];
      const float* from[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        from[u] = s.at + min(i + u * step, s.rows - 1) * s.pitch + c;
        f[u] = four(from[u]);
      }
      for (uint32_t q = 1; q < s.parts; ++q)
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const float4 v = four(from[u] + q * s.rows * s.pitch);
          f[u].x += v.x, f[u].y += v.y, f[u].z += v.z, f[u].w += v.w;
        }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const uint32_t r = i + u * step;
        const float v[4] = {f[u].x + b[0], f[u].y + b[1], f[u].z + b[2], f[u].w + b[3]};
        if (r < s.rows && row + r < all) emit<T>(p, row + r, col + c, gap, v);
      }
    }
  }
}

// Tiles are gone through in strips of 8 columns of them, row by row: what runs at the same time shares both operands' tiles in
// L2, also where one of them is larger than that.
struct Place {
  uint32_t row, col;
};
__device__ __forceinline__ Place place_of(uint32_t tile, uint32_t row_tiles, uint32_t col_tiles) {
  const uint32_t strip = tile / (row_tiles * 8), width = min(col_tiles - strip * 8, 8u), in = tile - strip * row_tiles * 8;
  return {in / width, strip * 8 + in % width};
}

#define CSW_WAIT_WARP(bar, parity)                                         \
  if (!__all_sync(0xffffffffu, bar_wait(bar, parity, p.patience))) {       \
    *reinterpret_cast<volatile uint32_t*>(&flag) = 1;                      \
    return;                                                                \
  }

// A warp's batch of scales, one block's to each of its first lanes, of OPERANDS times 128 rows or columns; seen by the tensor
// cores behind an arrival.
template <int OPERANDS>
__device__ __forceinline__ void write_scales(char* to, const uint32_t (&held)[OPERANDS]) {
  uint4* const words = reinterpret_cast<uint4*>(to) + threadIdx.x % 32;
#pragma unroll
  for (int j = 0; j < kBatch / 4 * OPERANDS; ++j) {
    uint32_t w = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) w |= __shfl_sync(0xffffffffu, held[j % OPERANDS], j / OPERANDS * 4 + q) << 8 * q;
    words[32 * j] = make_uint4(w, w, w, w);
  }
  async_fence();
  __syncwarp();
}

// The warp that writes scales and the four that quantize meet once; nothing in front of it can fail.
__device__ __forceinline__ void values_meet() { asm volatile("bar.sync 1, 160;" ::: "memory"); }

// One warp copies tiles, one writes their scales, one issues the products, four take the sums out.  Where there are few
// tiles, a cluster of `parts` CTAs shares one: each takes a part of the reduction, and sends its sums in shares, so that every
// CTA has some rows of the result from all parts, which it adds in their order.  (Loads from the other CTAs' shared memory took
// 460 clocks each, one after the other, copies of whole shares 1500 together.)
//
// What bounds it: the issue of a block's products, some 340 clocks, where BN is 128 or less (products of 128 x 128 take 256); the
// way from L2 into an SM above; and for the smallest ones 2 us from launch to the first block, 2 from the last to the end.
//
// A few rows of values (tokens, in generation) need not be quantized by a launch of their own: with X their type, the warps that
// wait for the sums do it before, every CTA for its part of the reduction.  First the scales of all its blocks, then the codes,
// a warp a block, into the stage that the other operand's tile is copied to.  (One token through 4096 x 4096: 10.6 us in two
// launches, 7.5 in one.)
constexpr int kMostHeld = 512;  // blocks of a CTA's part of the reduction, with X
template <class X>
struct Block {  // four columns of each row
  const Product& p;
  uint32_t col;
  __device__ Block(const Product& q, uint32_t block) : p(q), col(block * kBlock + threadIdx.x % 32 * 4) {}
  __device__ __forceinline__ void load(uint32_t row, float (&f)[4]) const {
    const X* from = static_cast<const X*>(p.x) + row * p.x_stride + col;
    if (p.x_packs && col + 4 <= p.x_cols) {
      load_pack(from, f);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = col + j < p.x_cols ? widen(from[j]) : 0.0f;
    }
  }
  __device__ __forceinline__ int exponent() const {
    uint32_t top = 0;
#pragma unroll 4
    for (uint32_t r = 0; r < p.n; ++r) {
      float f[4];
      load(r, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t bits = __float_as_uint(f[j]) & 0x7fffffffu;
        top = max(top, bits < 0x7f800000u ? bits : 0u);
      }
    }
    return exponent_of(__reduce_max_sync(0xffffffffu, top));
  }
  // to a tile of rows of 128 bytes, swizzled as the tile copies leave them
  __device__ __forceinline__ void write(char* tile, int e) const {
    const float factor = power_of(-e);
    const uint32_t lane = threadIdx.x % 32;
#pragma unroll 4
    for (uint32_t r = 0; r < p.n; ++r) {
      float f[4];
      load(r, f);
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float2 v = {isinf(f[j]) ? NAN : f[j] * factor, isinf(f[j + 1]) ? NAN : f[j + 1] * factor};
        word |= (uint32_t)__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3) << 8 * j;
      }
      *reinterpret_cast<uint32_t*>(tile + r * 128 + ((lane / 4) ^ (r & 7)) * 16 + lane % 4 * 4) = word;
    }
  }
};

template <int BN, class X = void>
__global__ void __launch_bounds__(kThreads, 2) fp8_product_kernel(const __grid_constant__ Product p) {
  using L = Plan<BN>;
  constexpr bool kValues = !std::is_same<X, void>::value;
  extern __shared__ char shared[];
  __shared__ uint64_t bars[2 * kMostStages + 6];
  __shared__ uint8_t held_scales[kValues ? kMostHeld : 1];
  __shared__ uint32_t tmem_at, flag;
  char* const ring = shared + (1024 - smem_at(shared) % 1024) % 1024;
  const uint32_t ring_at = smem_at(ring);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t full = smem_at(bars), empty = full + 8 * kMostStages, done = empty + 8 * kMostStages, received = done + 8;
  const uint32_t scaled = received + 8, unscaled = scaled + 16;
  const uint32_t stage = L::stage(p.c.across), scales_from = p.stages * stage;
  const uint32_t part = blockIdx.x % p.parts, tile = blockIdx.x / p.parts;
  const Place place = place_of(tile, p.row_tiles, p.col_tiles);
  const uint32_t row = place.row * kBlock, col = place.col * BN;
  const uint32_t begin = (uint64_t)p.steps * part / p.parts, count = (uint32_t)((uint64_t)p.steps * (part + 1) / p.parts) - begin;
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < p.stages; ++s) bar_init(full + 8 * s, kValues ? 2 : 1), bar_init(empty + 8 * s, 1);
    for (int b = 0; b < 2; ++b) bar_init(scaled + 8 * b, 1), bar_init(unscaled + 8 * b, 1);
    bar_init(done, 1);
    bar_init(received, 1);
    flag = 0;
    init_visible();
    if (p.steps) prefetch_map(&p.r.map);
    if (p.steps && !kValues) prefetch_map(&p.c.map);
  }
  // Every CTA's barriers are there.  From here to where tensor memory is freed no CTA waits for another one, which might wait
  // for that memory.
  if (p.parts > 1) cluster_meet();
  pdl_trigger_if_few();
  pdl_wait();  // before tensor memory is taken, which a kernel in front may still hold
  if (warp == 3) tmem_alloc<L::kColumns>(smem_at(&tmem_at));
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;
  if (warp == 0) {
    [&] {
      const bool me = elected();
      Turn turn{p.stages};
      for (uint32_t i = 0; i < count; ++i, turn.next()) {
        const uint32_t s = turn.s;
        if (turn.round) CSW_WAIT_WARP(empty + 8 * s, (turn.round - 1) & 1);
        if (p.idle) return;
        const uint32_t bar = full + 8 * s, to = ring_at + s * stage;
        const int k = (int)(begin + i) * kBlock;
        bar_expect_by(me, bar, kValues ? kTileBytes : stage);
        copy_bytes_tile_by(me, to, &p.r.map, bar, p.r.across ? (int)row : k, p.r.across ? k : (int)row);
#pragma unroll
        for (int j = 0; j < L::kPanels && !kValues; ++j)
          copy_bytes_tile_by(me, to + (1 + j) * kTileBytes, &p.c.map, bar, p.c.across ? (int)col + j * kBlock : k,
                             p.c.across ? k : (int)col + j * kBlock);
      }
    }();
  } else if (warp == 2) {
    if (kValues) values_meet();
    [&] {
      for (uint32_t i = 0, n = 0; i < count; i += kBatch, ++n) {
        const uint32_t mine = begin + i + lane % kBatch;  // a block's scales to a lane
        const bool is = i + lane % kBatch < count;
        uint32_t held[1 + L::kPanels];
        held[0] = is ? p.r.scales[(uint64_t)(row / kBlock) * p.r.scale_step + (uint64_t)mine * p.r.scale_k_step] : 0;
#pragma unroll
        for (int j = 0; j < L::kPanels; ++j)
          held[1 + j] = kValues ? (is ? held_scales[mine - begin] : 0)
                        : is && col + j * kBlock < p.n
                            ? p.c.scales[(uint64_t)(col / kBlock + j) * p.c.scale_step + (uint64_t)mine * p.c.scale_k_step]
                            : 0;
        if (n > 1) CSW_WAIT_WARP(unscaled + 8 * (n % 2), (n / 2 - 1) & 1);
        write_scales<1 + L::kPanels>(ring + scales_from + n % 2 * L::kBatchBytes, held);
        if (lane == 0) bar_arrive(scaled + 8 * (n % 2));
      }
    }();
  } else if (warp == 1) {
    [&] {
      const uint32_t desc = scaled_desc(BN, p.r.across, p.c.across);
      const uint32_t r_step = p.r.across ? 4096 / 16 : 32 / 16, c_step = p.c.across ? 4096 / 16 : 32 / 16;
      const bool me = elected();
      Turn turn{p.stages};
      for (uint32_t from = 0, n = 0; from < count; from += kBatch, ++n) {
        const uint32_t b = n % 2, held = tmem + BN + b * (kBatch / 4 * L::kWordColumns);
        const uint32_t steps = min(count - from, (uint32_t)kBatch);
        CSW_WAIT_WARP(scaled + 8 * b, n / 2 & 1);
        fence_after();
        const uint64_t scales = scales_desc(ring_at + scales_from + b * L::kBatchBytes);
        if (me)
          for (uint32_t j = 0; j < (steps + 3) / 4 * (1 + L::kPanels); ++j) copy_scales(held + 4 * j, scales + j * (512 / 16));
        __syncwarp();
        commit_by(me, unscaled + 8 * b);
        for (uint32_t i = 0; i < steps; ++i, turn.next()) {
          const uint32_t s = turn.s;
          CSW_WAIT_WARP(full + 8 * s, turn.round & 1);
          fence_after();
          const uint32_t at = ring_at + s * stage, word = held + i / 4 * L::kWordColumns;
          const uint64_t r = tile_desc(at, kTileBytes), c = tile_desc(at + kTileBytes, kTileBytes);
          const uint32_t which = desc | scales_of(i % 4);
#pragma unroll
          for (int k = 0; k < kBlock / 32; ++k)
            mma_scaled_by(me, tmem, r + k * r_step, c + k * c_step, which, word, word + 4, from + i || k);
          commit_by(me, empty + 8 * s);
          if (from + i + 1 == count) commit_by(me, done);
        }
      }
    }();
  } else if (warp >= 4) {
    if constexpr (kValues) {
      for (uint32_t i = warp - 4; i < count; i += 4) {
        const int e = Block<X>(p, begin + i).exponent();
        if (lane == 0) held_scales[i] = (uint8_t)(e + 127);
      }
      values_meet();
    }
    [&] {
      if constexpr (kValues) {
        for (uint32_t i = warp - 4; i < count; i += 4) {
          const uint32_t round = i / p.stages, s = i - round * p.stages;
          if (round) CSW_WAIT_WARP(empty + 8 * s, (round - 1) & 1);
          Block<X>(p, begin + i).write(ring + s * stage + kTileBytes, (int)held_scales[i] - 127);
          async_fence();
          __syncwarp();
          if (lane == 0) bar_arrive(full + 8 * s);
        }
      }
      if (count) CSW_WAIT_WARP(done, 0);
      fence_after();
      const uint32_t lanes = (uint32_t)(32 * (warp % 4)) << 16, line = 32 * (warp % 4) + lane;
      float* const sums = reinterpret_cast<float*>(ring);
#pragma unroll 1
      for (int j = 0; j < BN; j += 32) {
        uint32_t r[32] = {};
        if (count) {
          load32(tmem + lanes + j, r);
          wait_loads(r);
        }
        if (p.exchanged) {
#pragma unroll
          for (int k = 0; k < 32; ++k) sums[(j + k) * kBlock + line] = __uint_as_float(r[k]);
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<uint4*>(sums + line * L::kPitch + j + k) = make_uint4(r[k], r[k + 1], r[k + 2], r[k + 3]);
        }
      }
    }();
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 3) tmem_free<L::kColumns>(tmem);
  const uint32_t pitch = p.exchanged ? kBlock : L::kPitch, lines = p.exchanged ? BN : kBlock;
  // What waits ran out for is NaN; copies on their way get time to land first.
  auto spoil = [&](float* at, uint32_t n) {
    for (int i = 0; i < 1000; ++i) __nanosleep(10000);
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) at[i] = NAN;
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t*>(p.status) = 1;
      __threadfence_system();
    }
    __syncthreads();
  };
  float* sums = reinterpret_cast<float*>(ring);
  if (*reinterpret_cast<volatile uint32_t*>(&flag)) spoil(sums, lines * pitch);
  const uint32_t rows = lines / p.parts;  // of the result, that this CTA writes
  const uint32_t first_row = p.exchanged ? col : row, all_rows = p.exchanged ? p.n : p.m;
  const uint32_t to_row = first_row + part * rows, to_col = p.exchanged ? row : col;
  if (p.parts > 1) {
    float* const from = reinterpret_cast<float*>(ring + scales_from + 2 * L::kBatchBytes);
    const uint32_t bytes = rows * pitch * 4;
    async_fence();
    __syncthreads();
    if (threadIdx.x == 0) {  // to those whose rows the result has
      if (to_row < all_rows) bar_expect(received, bytes * p.parts);
      for (uint32_t q = 0; q < p.parts && first_row + q * rows < all_rows; ++q)
        send_bytes(peer_at(smem_at(from) + part * bytes, q), ring_at + q * bytes, bytes, peer_at(received, q));
    }
    if (to_row < all_rows && !__syncthreads_and(bar_wait_cluster(received, 0, p.patience))) spoil(from, lines * pitch);
    sums = from;
  }
  const Sums s{sums, p.parts, rows, pitch, p.exchanged ? (uint32_t)kBlock : (uint32_t)BN};
  if (p.type == 0) emit_rows<float>(p, s, to_row, to_col);
  else if (p.type == 1) emit_rows<__half>(p, s, to_row, to_col);
  else emit_rows<__nv_bfloat16>(p, s, to_row, to_col);
  if (p.parts > 1) cluster_meet();  // nobody leaves while what it sends is read
}

// ---- two CTAs on a tile ------------------------------------------------------------------------------------------------
// Tiles of 256 x 256, each on a pair of CTAs, which keep 128 rows and bring 128 of the columns each: a block of the reduction
// then takes 32 KB into an SM for 512 clocks of products, where a CTA on its own takes 48.  A pair goes through tiles until there
// are none left.  Eight warps take a tile's sums into registers, 128 a thread, and tell that the next one's may begin; they are
// rounded, and leave, meanwhile.
//
// What bounds it: the tensor cores, busy 86 % of the time, and in long runs the power limit.  8192 x 8192 x 4096: 195 us, 2.8
// PFLOP/s; products alone would take 165, copies alone 142.
template <class T>
constexpr int kEachOf = 16 / sizeof(T);
constexpr int kPairThreads = 384, kPairStages = 5, kPairTile = 2 * kBlock;
constexpr uint32_t kPairStage = 2 * kTileBytes, kChunk = 32 * 128, kPairChunks = kPairStages * kPairStage;
constexpr uint32_t kWordBytes = 3 * 512;  // four blocks' scales: of 128 rows and of 256 columns
constexpr uint32_t kPairScales = kPairChunks + 8 * kChunk, kBatchBytes = kBatch / 4 * kWordBytes;
constexpr size_t kPairShared = kPairScales + 2 * kBatchBytes + 1024;

template <class T>
__global__ void __launch_bounds__(kPairThreads, 1) fp8_pair_kernel(const __grid_constant__ Product p,
                                                                   const __grid_constant__ CUtensorMap out_map) {
  extern __shared__ char shared[];
  __shared__ uint64_t bars[2 * kPairStages + 6];
  __shared__ uint32_t tmem_at, flag;
  char* const ring = shared + (1024 - smem_at(shared) % 1024) % 1024;
  const uint32_t ring_at = smem_at(ring);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank();
  // full, taken_out and scaled: the first CTA's; empty, done and unscaled: each one's
  const uint32_t full = smem_at(bars), empty = full + 8 * kPairStages, done = empty + 8 * kPairStages, taken_out = done + 8;
  const uint32_t scaled = taken_out + 8, unscaled = scaled + 16;
  const uint32_t tiles = p.row_tiles * p.col_tiles, pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) bar_init(full + 8 * s, 1), bar_init(empty + 8 * s, 1);
    bar_init(done, 1);
    bar_init(taken_out, 16);
    for (int i = 0; i < 2; ++i) bar_init(scaled + 8 * i, 2), bar_init(unscaled + 8 * i, 1);
    flag = 0;
    init_visible();
    prefetch_map(&p.r.map);
    prefetch_map(&p.c.map);
  }
  pdl_wait();
  if (warp == 3) tmem_alloc_pair<512>(smem_at(&tmem_at));
  fence_before();
  __syncthreads();
  cluster_meet();  // both CTAs' barriers are there
  fence_after();
  const uint32_t tmem = tmem_at;
  if (warp == 0) {
    [&] {
      const bool me = elected();
      Turn turn{kPairStages};
      for (uint32_t tile = pair; tile < tiles; tile += pairs) {
        const Place place = place_of(tile, p.row_tiles, p.col_tiles);
        const int row = (int)(place.row * kPairTile + rank * kBlock), col = (int)(place.col * kPairTile + rank * kBlock);
        for (uint32_t k = 0; k < p.steps; ++k, turn.next()) {
          const uint32_t s = turn.s;
          if (turn.round) CSW_WAIT_WARP(empty + 8 * s, (turn.round - 1) & 1);
          if (p.idle) return;
          const uint32_t bar = peer_at(full + 8 * s, 0), to = ring_at + s * kPairStage;
          const int at = (int)k * kBlock;
          bar_expect_by(me && rank == 0, full + 8 * s, 2 * kPairStage);
          copy_bytes_tile_pair_by(me, to, &p.r.map, bar, p.r.across ? row : at, p.r.across ? at : row);
          copy_bytes_tile_pair_by(me, to + kTileBytes, &p.c.map, bar, p.c.across ? col : at, p.c.across ? at : col);
        }
      }
    }();
  } else if (warp == 2) {
    [&] {
      uint32_t n = 0;  // batches
      for (uint32_t tile = pair; tile < tiles; tile += pairs) {
        const Place place = place_of(tile, p.row_tiles, p.col_tiles);
        const uint32_t row = place.row * 2 + rank, col = place.col * 2;  // blocks
        for (uint32_t k = 0; k < p.steps; k += kBatch, ++n) {
          const uint32_t mine = k + lane % kBatch;
          auto scale = [&](const Operand& o, uint32_t block, uint32_t end) {
            return mine < p.steps && block * kBlock < end
                       ? (uint32_t)o.scales[(uint64_t)block * o.scale_step + (uint64_t)mine * o.scale_k_step]
                       : 0u;
          };
          const uint32_t held[3] = {scale(p.r, row, p.m), scale(p.c, col, p.n), scale(p.c, col + 1, p.n)};
          const uint32_t s = n % 2;
          if (n > 1) CSW_WAIT_WARP(unscaled + 8 * s, (n / 2 - 1) & 1);
          write_scales<3>(ring + kPairScales + s * kBatchBytes, held);
          if (lane == 0) peer_arrive(peer_at(scaled + 8 * s, 0));
        }
      }
    }();
  } else if (warp == 1 && rank == 0) {
    [&] {
      const uint32_t desc = scaled_desc(kPairTile, p.r.across, p.c.across) + kPairRows;
      const uint32_t r_step = p.r.across ? 4096 / 16 : 32 / 16, c_step = p.c.across ? 4096 / 16 : 32 / 16;
      const bool me = elected();
      Turn turn{kPairStages};
      uint32_t n = 0, batch = 0;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        const bool there = __all_sync(0xffffffffu, bar_wait_cluster(bar, parity, p.patience));
        if (!there) *reinterpret_cast<volatile uint32_t*>(&flag) = 1;
        return there;
      };
      for (uint32_t tile = pair; tile < tiles; tile += pairs, ++n) {
        if (n && !wait(taken_out, (n - 1) & 1)) return;
        fence_after();
        for (uint32_t from = 0; from < p.steps; from += kBatch, ++batch) {
          const uint32_t b = batch % 2, scales_at = tmem + kPairTile + b * (kBatch / 4 * 12);
          const uint32_t steps = min(p.steps - from, (uint32_t)kBatch);
          if (!wait(scaled + 8 * b, batch / 2 & 1)) return;
          fence_after();
          const uint64_t scales = scales_desc(ring_at + kPairScales + b * kBatchBytes);
          if (me)
            for (uint32_t j = 0; j < (steps + 3) / 4 * 3; ++j) copy_scales_pair(scales_at + 4 * j, scales + j * (512 / 16));
          __syncwarp();
          commit_pair_by(me, unscaled + 8 * b);
          for (uint32_t k = 0; k < steps; ++k, turn.next()) {
            const uint32_t s = turn.s;
            if (!wait(full + 8 * s, turn.round & 1)) return;
            fence_after();
            const uint32_t at = ring_at + s * kPairStage, word = scales_at + k / 4 * 12;
            const uint64_t r = tile_desc(at, kTileBytes), c = tile_desc(at + kTileBytes, kTileBytes);
            const uint32_t which = desc | scales_of(k % 4);
#pragma unroll
            for (int q = 0; q < kBlock / 32; ++q)
              mma_scaled_pair_by(me, tmem, r + q * r_step, c + q * c_step, which, word, word + 4, from + k || q);
            commit_pair_by(me, empty + 8 * s);
            if (from + k + 1 == p.steps) commit_pair_by(me, done);
          }
        }
      }
    }();
  } else if (warp >= 4) {
    [&] {
      const uint32_t lanes = (uint32_t)(32 * (warp % 4)) << 16, half = (warp - 4) / 4 * kBlock;
      char* const chunk = ring + kPairChunks + (warp - 4) * kChunk;
      constexpr int kWide = 128 / sizeof(T);  // columns of a chunk: 32 rows of 128 bytes
      uint32_t n = 0;
      for (uint32_t tile = pair; tile < tiles; tile += pairs, ++n) {
        const Place place = place_of(tile, p.row_tiles, p.col_tiles);
        const uint32_t row = place.row * kPairTile + rank * kBlock + 32 * (warp % 4), col = place.col * kPairTile + half;
        CSW_WAIT_WARP(done, n & 1);
        fence_after();
        uint32_t r[4][32];
#pragma unroll
        for (int j = 0; j < 4; ++j) load32(tmem + lanes + half + 32 * j, r[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) wait_loads(r[j]);
        fence_before();
        __syncwarp();
        if (lane == 0) peer_arrive_near(peer_at(taken_out, 0));
        if (row >= p.m) continue;
#pragma unroll
        for (int at = 0; at < kBlock; at += kWide) {
          if (col + at < p.n) {
            if (lane == 0) stores_read();  // the last copy, from this chunk
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kWide; j += 32) {
              uint32_t(&v)[32] = r[(at + j) / 32];
              if (p.bias) {
                const float b = col + at + j + lane < p.n ? bias_at(p, col + at + j + lane) : 0.0f;
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  v[k] = __float_as_uint(__uint_as_float(v[k]) + __shfl_sync(0xffffffffu, b, k));
              }
              constexpr int kEach = 16 / sizeof(T);
#pragma unroll
              for (int k = 0; k < 32; k += kEach) {
                float f[kEach];
#pragma unroll
                for (int q = 0; q < kEach; ++q) f[q] = __uint_as_float(v[k + q]);
                store_pack(reinterpret_cast<T*>(chunk + lane * 128 + (((j + k) / kEach) ^ (lane & 7)) * 16), f);
              }
            }
            if (p.packs) {
              async_fence();
              __syncwarp();
              if (lane == 0) store_matrix_tile(&out_map, smem_at(chunk), (int)(col + at), (int)row);
            } else {  // rows that begin anywhere: a row of the chunk at a time, a value a lane
              __syncwarp();
              T* to = static_cast<T*>(p.out) + (uint64_t)row * p.n + col + at + lane;
              const int rows = (int)min(p.m - row, 32u), wide = (int)min(p.n - col - at, (uint32_t)kWide) - lane;
              const uintptr_t mine = reinterpret_cast<uintptr_t>(chunk) + lane * sizeof(T);
#pragma unroll 1
              for (int i = 0; i < rows; i += 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k, to += p.n) {
#pragma unroll
                  for (int j = 0; j < kWide; j += 32) {
                    const T v = *reinterpret_cast<const T*>((mine ^ (k * 16) ^ (j * sizeof(T))) + (i + k) * 128);
                    if (i + k < rows && j < wide) to[j] = v;
                  }
                }
              }
            }
          }
        }
      }
    }();
    if (lane == 0) stores_done();
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (*reinterpret_cast<volatile uint32_t*>(&flag)) {
    for (int i = 0; i < 1000; ++i) __nanosleep(10000);
    const float f[4] = {NAN, NAN, NAN, NAN};
    for (uint32_t tile = pair; tile < tiles; tile += pairs) {
      const Place place = place_of(tile, p.row_tiles, p.col_tiles);
      const uint32_t row = place.row * kPairTile + rank * kBlock, col = place.col * kPairTile;
      for (uint32_t i = threadIdx.x; i < kBlock * (kPairTile / 4); i += kPairThreads)
        if (row + i / (kPairTile / 4) < p.m && col + i % (kPairTile / 4) * 4 < p.n)
          emit<T>(p, row + i / (kPairTile / 4), col + i % (kPairTile / 4) * 4, 1, f);
    }
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t*>(p.status) = 1;
      __threadfence_system();
    }
  }
  cluster_meet();  // the other CTA's tensor and shared memory is used until then
  if (warp == 3) tmem_free_pair<512>(tmem);
}

// ---- host -----------------------------------------------------------------------------------------------------------
bool operand_of(Operand* o, const Fp8Matrix& m, bool across, int rows_of_box) {
  const TileEncoder encode = tile_encoder();
  if (!encode) return false;
  const cuuint64_t dims[2] = {m.cols, m.rows}, strides[1] = {m.stride};
  const cuuint32_t box[2] = {kBlock, (cuuint32_t)(across ? kBlock : rows_of_box)}, steps[2] = {1, 1};
  o->scales = m.scales;
  const uint32_t blocks = (uint32_t)fp8_blocks(m.cols);
  o->scale_step = across ? 1 : blocks, o->scale_k_step = across ? blocks : 1;
  o->across = across;
  return encode(&o->map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(m.codes), dims, strides, box, steps,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a product is computed: tiles of so many columns, 0 for those of pairs, and parts of the reduction.  By the time that each
// way takes, in microseconds, as measured over 36 sizes (the way chosen by it took 1 % longer than the best, in the mean): two for
// the launch; a tile's beginning and end, and its blocks of the reduction, where a CTA has an SM to itself or shares it with
// another; for parts of the reduction their way through the cluster.  Some of them (m x n x k, the best way in front):
//   1 x 4096 x 4096     32 columns, 4 parts 7.2, 2 parts 8.0, whole 9.1
//   768 x 768 x 16384   64 columns, 2 parts 19.1, 128 columns, 2 parts 20.3, whole 28.1, pairs 41.8
//   1024 x 1024 x 1024  64 columns 5.8, 128 columns 6.5, 32 columns 6.7, pairs 8.3
//   4096 x 4096 x 4096  pairs 51.6, 256 columns 67.3, 128 columns 69.0, 64 columns 89.4
// Clusters take one round only: a second one starts some ten microseconds late.
struct Way {
  int columns;
  uint32_t parts;
};
Way way_for(const Product& p) {
  constexpr int kColumns[] = {32, 64, 128, 256};
  constexpr float kEnds[] = {2.0f, 2.4f, 3.4f, 5.5f}, kStep[] = {0.17f, 0.175f, 0.185f, 0.28f};        // alone on an SM
  constexpr float kEndsShared[] = {3.4f, 4.2f, 5.7f}, kStepShared[] = {0.215f, 0.265f, 0.43f};         // two on an SM
  constexpr float kRoom[] = {1.0f, 1.0f, 0.89f, 0.81f};  // of the SMs, for clusters of 1, 2, 4, 8: they stay within a part of the chip
  const float sms = (float)sm_count();
  auto rounds = [](uint64_t tiles, float at_once) { return std::ceil((float)tiles / at_once); };
  Way best{32, 1};
  float least = 1e30f;
  auto consider = [&](int columns, uint32_t parts, float time) {
    if (time < least) least = time, best = {columns, parts};
  };
  for (int i = 0; i < 4; ++i) {
    if (i && (uint32_t)kColumns[i] >= 2 * p.n) break;  // half of each tile would be empty
    const uint64_t tiles = (uint64_t)p.row_tiles * ((p.n + kColumns[i] - 1) / kColumns[i]);
    if (i == 3) consider(256, 1, 2.0f + rounds(tiles, sms) * (kEnds[3] + p.steps * kStep[3]));
    else if ((float)tiles <= sms) consider(kColumns[i], 1, 2.0f + kEnds[i] + p.steps * kStep[i]);
    else consider(kColumns[i], 1, 2.0f + rounds(tiles, 2 * sms) * (kEndsShared[i] + p.steps * kStepShared[i]));
    for (int j = 1; i < 3 && j < 4 && (1u << j) <= p.steps; ++j)
      if ((float)(tiles << j) <= sms * kRoom[j])
        consider(kColumns[i], 1u << j, 3.6f + 0.4f * j + kEnds[i] + ((p.steps + (1u << j) - 1) >> j) * kStep[i]);
  }
  if (p.steps && !p.exchanged && sms >= 2.0f) {
    const uint64_t tiles = (uint64_t)((p.m + kPairTile - 1) / kPairTile) * ((p.n + kPairTile - 1) / kPairTile);
    consider(0, 1, 6.0f + rounds(tiles, std::floor(sms / 2)) * (p.steps * 0.3f + (p.packs ? 0.7f : 2.3f)));
  }
  return best;
}

template <int BN, class X = void>
cudaError_t product(Product& p, const Fp8Matrix& r, const Fp8Matrix& c, bool r_across, bool c_across, cudaStream_t stream) {
  using L = Plan<BN>;
  if (p.steps && !operand_of(&p.r, r, r_across, kBlock)) return cudaErrorInvalidValue;
  if (p.steps && !p.x && !operand_of(&p.c, c, c_across, std::min(BN, kBlock))) return cudaErrorInvalidValue;
  p.col_tiles = (p.n + BN - 1) / BN;
  const uint32_t ctas = p.row_tiles * p.col_tiles * p.parts;
  const bool alone = BN > kBlock || p.parts > 1 || ctas <= (uint32_t)sm_count();
  p.stages = L::stages(c_across, alone, p.parts > 1, p.steps / p.parts + 1);
  const size_t shared = L::shared(c_across, p.parts > 1, p.stages);
  // the most of any call, so that calls at the same time need not agree
  if (const cudaError_t e = taken(
          cudaFuncSetAttribute(fp8_product_kernel<BN, X>, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024)))
    return e;
  return pdl_launch_clusters(fp8_product_kernel<BN, X>, ctas, p.parts, kThreads, shared, stream, p);
}

template <class T>
cudaError_t pair_product(Product& p, const Fp8Matrix& r, const Fp8Matrix& c, bool r_across, bool c_across, cudaStream_t stream) {
  if (!operand_of(&p.r, r, r_across, kBlock) || !operand_of(&p.c, c, c_across, kBlock)) return cudaErrorInvalidValue;
  CUtensorMap out{};
  if (p.packs) {
    const cuuint64_t dims[2] = {p.n, p.m}, strides[1] = {(cuuint64_t)p.n * sizeof(T)};
    const cuuint32_t box[2] = {128 / sizeof(T), 32}, steps[2] = {1, 1};
    const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    if (tile_encoder()(&out, type, 2, p.out, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  if (const cudaError_t e =
          taken(cudaFuncSetAttribute(fp8_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairShared)))
    return e;
  p.row_tiles = (p.m + kPairTile - 1) / kPairTile, p.col_tiles = (p.n + kPairTile - 1) / kPairTile;
  const uint32_t pairs = std::min(p.row_tiles * p.col_tiles, std::max((uint32_t)sm_count() / 2, 1u));
  return pdl_launch_clusters(fp8_pair_kernel<T>, 2 * pairs, 2, kPairThreads, kPairShared, stream, p, out);
}

}  // namespace

cudaError_t fp8_quantize_launch(const Fp8Quantize& a, cudaStream_t stream) {
  if (a.cols == 0) return cudaSuccess;
  if (a.rows == 0)
    return a.sums ? taken(cudaMemsetAsync(a.sums, 0, a.cols * (a.sums_type == 0 ? 4 : 2), stream)) : cudaSuccess;
  const uint64_t parts = fp8_blocks(a.rows), grid = parts * fp8_blocks(a.cols);
  cudaError_t e = cudaSuccess;
  void* const sums = parts > 1 ? a.partials : a.sums;
  with_type(a.type, [&](auto v) {
    using T = decltype(v);
    const bool packs = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.stride * sizeof(T) % 16 == 0;
    const auto kernel = a.sums ? fp8_quantize_kernel<T, true> : fp8_quantize_kernel<T, false>;
    e = pdl_launch(kernel, (unsigned)grid, kQuantizeThreads, 0, stream, static_cast<const T*>(a.x), a.rows, a.cols, a.stride,
                   packs, static_cast<uint8_t*>(a.codes), a.code_stride, a.scales, sums, parts > 1 ? 0 : a.sums_type);
  });
  if (e == cudaSuccess && a.sums && parts > 1)
    e = pdl_launch(fp8_sums_kernel, (unsigned)((a.cols + 31) / 32), 256, 0, stream, (const float*)a.partials, parts, a.cols,
                   a.sums, a.sums_type);
  return e;
}

cudaError_t fp8_dequantize_launch(const void* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols,
                                  void* out, int type, cudaStream_t stream) {
  if (rows == 0 || cols == 0) return cudaSuccess;
  cudaError_t e = cudaSuccess;
  with_type(type, [&](auto v) {
    using T = decltype(v);
    const bool packs = cols % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    e = pdl_launch(fp8_dequantize_kernel<T>, (unsigned)(fp8_blocks(rows) * fp8_blocks(cols)), kQuantizeThreads, 0, stream,
                   static_cast<const uint8_t*>(codes), code_stride, scales, rows, cols, packs, static_cast<T*>(out));
  });
  return e;
}

namespace {
// what a product of m x k and k x n needs besides its operands
cudaError_t begin_product(Product* p, uint64_t m, uint64_t n, uint64_t k, const void* bias, int bias_type, void* out, int type) {
  if (const cudaError_t e = bind_context()) return e;
  *p = Product{};
  if (const cudaError_t e = status_word(&p->status)) return e;
  const long long limit = wait_limit();
  p->patience = limit < 0 ? -limit : limit, p->idle = limit < 0;
  p->out = out, p->bias = bias, p->type = type, p->bias_type = bias_type;
  p->steps = (uint32_t)fp8_blocks(k);
  p->exchanged = m <= 64 && n > m;
  p->packs = n * (type == 0 ? 4 : 2) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  p->m = (uint32_t)(p->exchanged ? n : m), p->n = (uint32_t)(p->exchanged ? m : n);
  p->row_tiles = (uint32_t)fp8_blocks(p->m);
  return cudaSuccess;
}
}  // namespace

cudaError_t fp8_matmul_launch(const Fp8Matrix& a, const Fp8Matrix& b, const void* bias, int bias_type, void* out, int type,
                              cudaStream_t stream) {
  const uint64_t m = a.transposed ? a.cols : a.rows, k = a.transposed ? a.rows : a.cols;
  const uint64_t n = b.transposed ? b.rows : b.cols;
  if (m == 0 || n == 0) return cudaSuccess;
  Product p;
  if (const cudaError_t e = begin_product(&p, m, n, k, bias, bias_type, out, type)) return e;
  const Fp8Matrix &r = p.exchanged ? b : a, &c = p.exchanged ? a : b;
  const bool r_across = p.exchanged ? !b.transposed : a.transposed, c_across = p.exchanged ? a.transposed : !b.transposed;
  const Way way = way_for(p);
  p.parts = way.parts;
  switch (way.columns) {
    case 32: return product<32>(p, r, c, r_across, c_across, stream);
    case 64: return product<64>(p, r, c, r_across, c_across, stream);
    case 128: return product<128>(p, r, c, r_across, c_across, stream);
    case 256: return product<256>(p, r, c, r_across, c_across, stream);
  }
  cudaError_t e = cudaErrorInvalidValue;
  with_type(type, [&](auto v) { e = pair_product<decltype(v)>(p, r, c, r_across, c_across, stream); });
  return e;
}

bool fp8_linear_at_once(uint64_t rows, uint64_t cols, uint64_t outs) {
  return rows <= 32 && outs > rows && fp8_blocks(cols) <= kMostHeld;
}

cudaError_t fp8_linear_launch(const Fp8Quantize& x, const Fp8Matrix& weight, const void* bias, int bias_type, void* out,
                              int type, cudaStream_t stream) {
  if (x.rows == 0 || weight.rows == 0) return cudaSuccess;
  if (!fp8_linear_at_once(x.rows, x.cols, weight.rows)) {
    const cudaError_t e = fp8_quantize_launch(x, stream);
    const Fp8Matrix held{x.codes, x.scales, x.rows, x.cols, x.code_stride, false};
    return e != cudaSuccess ? e : fp8_matmul_launch(held, weight, bias, bias_type, out, type, stream);
  }
  Product p;
  if (const cudaError_t e = begin_product(&p, x.rows, weight.rows, x.cols, bias, bias_type, out, type)) return e;
  p.parts = way_for(p).parts;
  p.x = x.x, p.x_stride = x.stride, p.x_cols = (uint32_t)x.cols;
  cudaError_t e = cudaErrorInvalidValue;
  with_type(x.type, [&](auto v) {
    using X = decltype(v);
    p.x_packs = reinterpret_cast<uintptr_t>(x.x) % (4 * sizeof(X)) == 0 && x.stride % 4 == 0;
    e = product<32, X>(p, weight, Fp8Matrix{}, false, false, stream);
  });
  return e;
}

}  // namespace csw
