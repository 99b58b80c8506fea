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

#include "internal.h"
#include "pdl.cuh"
#include "tensor_core.cuh"
#include "values.cuh"
#include "waits.h"

namespace csw {
namespace {

constexpr int kBlock = (int)kFp8Block;

// ---- quantizing -----------------------------------------------------------------------------------------------------
// A CTA a block, its values in registers: 16 threads a row of 8 values each, 16 rows at a time, so that a value is read
// once.  The columns' sums (what a bias's gradient is) leave each block of rows once and are added up in order.
constexpr int kQuantizeThreads = 256;

// the scale of a block whose largest magnitude has these bits, and what its values are multiplied with
__device__ __forceinline__ int exponent_of(uint32_t top) {
  return max((int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);  // 448 is 1.75 2^8
}
__device__ __forceinline__ float power_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <class T, bool SUMS>
__global__ void __launch_bounds__(kQuantizeThreads) fp8_quantize_kernel(const T* __restrict__ x, uint64_t rows, uint64_t cols,
                                                                        uint64_t stride, bool packs, uint8_t* codes,
                                                                        uint64_t code_stride, uint8_t* scales, float* sums) {
  __shared__ uint32_t tops[kQuantizeThreads / 32];
  __shared__ float column[SUMS ? 16 : 1][SUMS ? kBlock : 1];
  pdl_wait(x);
  const uint64_t blocks = (cols + kBlock - 1) / kBlock, bi = blockIdx.x / blocks, bj = blockIdx.x % blocks;
  const int t = threadIdx.x, r0 = t / 16, c = t % 16 * 8;
  const uint64_t col = bj * kBlock + c;
  const int live = (int)min((int64_t)8, max((int64_t)cols - (int64_t)col, (int64_t)0));  // of this thread's columns
  float f[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t row = bi * kBlock + r0 + 16 * i;
    const T* from = x + row * stride + col;
    if (row < rows && live == 8 && packs) {
      constexpr int kEach = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 8; j += kEach) {
        float v[kEach];
        load_pack(from + j, v);
#pragma unroll
        for (int k = 0; k < kEach; ++k) f[i][j + k] = v[k];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = row < rows && j < live ? widen(from[j]) : 0.0f;
    }
  }
  uint32_t top = 0;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = __float_as_uint(f[i][j]) & 0x7fffffffu;
      const bool number = bits < 0x7f800000u;
      odd |= !number;
      top = max(top, number ? bits : 0u);
    }
  top = __reduce_max_sync(0xffffffffu, top);
  if (t % 32 == 0) tops[t / 32] = top;
  if constexpr (SUMS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = f[0][j];
#pragma unroll
      for (int i = 1; i < 8; ++i) s += f[i][j];
      column[r0][c + j] = s;
    }
  }
  odd = __syncthreads_or(odd);
#pragma unroll
  for (int w = 0; w < kQuantizeThreads / 32; ++w) top = max(top, tops[w]);
  const int e = exponent_of(top);
  if (t == 0) scales[blockIdx.x] = (uint8_t)(e + 127);
  if constexpr (SUMS) {
    if (t < kBlock && bj * kBlock + t < cols) {
      float s = column[0][t];
#pragma unroll
      for (int i = 1; i < 16; ++i) s += column[i][t];
      sums[bi * cols + bj * kBlock + t] = s;
    }
  }
  const float factor = power_of(-e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t row = bi * kBlock + r0 + 16 * i;
    uint32_t word[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float2 v = {f[i][j] * factor, f[i][j + 1] * factor};
      if (odd) {  // the conversion would make the largest number of an infinity
        if (isinf(v.x)) v.x = NAN;
        if (isinf(v.y)) v.y = NAN;
      }
      word[j / 4] |= (uint32_t)__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3) << (j % 4 * 8);
    }
    // up to 7 bytes behind the last column belong to the row's stride
    if (row < rows && live > 0) *reinterpret_cast<uint2*>(codes + row * code_stride + col) = make_uint2(word[0], word[1]);
  }
}

// The sums of the blocks of rows, in their order: 8 threads a column, each a part of the blocks.
__global__ void __launch_bounds__(256) fp8_sums_kernel(const float* __restrict__ partials, uint64_t parts, uint64_t cols,
                                                       float* sums) {
  __shared__ float part[8][32];
  pdl_wait(partials);
  const uint64_t col = (uint64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const int p = threadIdx.x / 32;
  float s = 0.0f;
  if (col < cols)
    for (uint64_t i = p; i < parts; i += 8) s += partials[i * cols + col];
  part[p][threadIdx.x % 32] = s;
  __syncthreads();
  if (p || col >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
  sums[col] = s;
}

template <class T>
__global__ void __launch_bounds__(256) fp8_dequantize_kernel(const uint8_t* __restrict__ codes, uint64_t code_stride,
                                                             const uint8_t* __restrict__ scales, uint64_t rows, uint64_t cols,
                                                             uint64_t packs, bool whole, T* out) {
  pdl_wait(codes);
  pdl_behind(scales);
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x, row = i / packs, col = i % packs * 8;
  if (row >= rows) return;
  const uint2 word = *reinterpret_cast<const uint2*>(codes + row * code_stride + col);
  const float scale = power_of((int)scales[row / kBlock * ((cols + kBlock - 1) / kBlock) + col / kBlock] - 127);
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const __half2_raw h =
        __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 4 ? word.x : word.y) >> (j % 4 * 8)), __NV_E4M3);
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[j] = v.x * scale, f[j + 1] = v.y * scale;
  }
  T* to = out + row * cols + col;
  if (whole) {
    constexpr int kEach = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8; j += kEach) {
      float v[kEach];
#pragma unroll
      for (int k = 0; k < kEach; ++k) v[k] = f[j + k];
      store_pack(to + j, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < cols) to[j] = narrow<T>(f[j]);
  }
}

// ---- products -------------------------------------------------------------------------------------------------------
using namespace tc;

constexpr uint32_t kTileBytes = kBlock * kBlock;
constexpr int kThreads = 256;

// Tiles of 128 x BN of the result, 128 of the reduction at a time.  A stage of the ring: the row operand's tile, the column
// operand's, and 512 bytes of scales for each 128 rows or columns.
template <int BN>
struct Plan {
  static constexpr int kPanels = (BN + kBlock - 1) / kBlock;  // tiles of 128 columns
  static constexpr uint32_t kScales = kTileBytes * (1 + kPanels);
  static constexpr uint32_t kStage = kScales + 512 * (1 + kPanels);
  static constexpr int kStages = BN > kBlock ? 4 : 3;
  static constexpr size_t kShared = kStages * kStage + 1024;
  static constexpr int kNeeded = BN + 4 + 4 * kPanels;  // columns of tensor memory: sums, then scales
  static constexpr int kColumns = kNeeded > 256 ? 512 : kNeeded > 128 ? 256 : kNeeded > 64 ? 128 : 64;
  static_assert(BN * 512 <= kStages * kStage, "a tile's sums lie where the stages were");
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
  uint32_t row_tiles, parts;
  // the result: [m][n], or [n][m] where the operands were exchanged; the bias goes by its last axis
  void* out;
  const void* bias;
  int type, bias_type;
  bool exchanged, packs;  // packs: rows of the result begin on 16 bytes
  long long patience;
  bool idle;
  uint32_t* status;
};

__device__ __forceinline__ float bias_at(const Product& p, uint32_t i) {
  return p.bias_type == 0   ? static_cast<const float*>(p.bias)[i]
         : p.bias_type == 1 ? widen(static_cast<const __half*>(p.bias)[i])
                            : widen(static_cast<const __nv_bfloat16*>(p.bias)[i]);
}
// N neighbouring columns of one row, bias added and rounded
template <class T, int N>
__device__ __forceinline__ void emit(const Product& p, uint32_t row, uint32_t col, float (&f)[N]) {
  if (row >= p.m) return;
  T* out = static_cast<T*>(p.out);
  if (p.exchanged) {
    const float b = p.bias ? bias_at(p, row) : 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (col + j < p.n) out[(uint64_t)(col + j) * p.m + row] = narrow<T>(f[j] + b);
    return;
  }
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (col + j < p.n) f[j] += bias_at(p, col + j);
  }
  out += (uint64_t)row * p.n + col;
  constexpr int kEach = 16 / sizeof(T);
  if (N % kEach == 0 && p.packs && col + N <= p.n) {
#pragma unroll
    for (int j = 0; j + kEach <= N; j += kEach) {
      float v[kEach];
#pragma unroll
      for (int k = 0; k < kEach; ++k) v[k] = f[j + k];
      store_pack(out + j, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (col + j < p.n) out[j] = narrow<T>(f[j]);
  }
}
template <int N>
__device__ __forceinline__ void emit_any(const Product& p, uint32_t row, uint32_t col, float (&f)[N]) {
  if (p.type == 0) emit<float>(p, row, col, f);
  else if (p.type == 1) emit<__half>(p, row, col, f);
  else emit<__nv_bfloat16>(p, row, col, f);
}

__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a word of another CTA's shared memory, at the address that it has in this one's
__device__ __forceinline__ float peer_float(uint32_t at, uint32_t rank) {
  float v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
               : "=f"(v)
               : "r"(at), "r"(rank)
               : "memory");
  return v;
}

#define CSW_WAIT_WARP(bar, parity)                                         \
  if (!__all_sync(0xffffffffu, bar_wait(bar, parity, p.patience))) {       \
    *reinterpret_cast<volatile uint32_t*>(&flag) = 1;                      \
    return;                                                                \
  }

// One warp copies tiles, one writes their scales, one issues the products, four take the sums out.  Where there are few
// tiles, a cluster of `parts` CTAs shares one: each takes a part of the reduction, and the parts' sums, in shared memory, are
// added in their order, each CTA a part of the columns.
template <int BN>
__global__ void __launch_bounds__(kThreads) fp8_product_kernel(const __grid_constant__ Product p) {
  using L = Plan<BN>;
  extern __shared__ char shared[];
  __shared__ uint64_t bars[2 * L::kStages + 1];
  __shared__ uint32_t tmem_at, flag;
  char* const ring = shared + (1024 - smem_at(shared) % 1024) % 1024;
  const uint32_t ring_at = smem_at(ring);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t full = smem_at(bars), empty = full + 8 * L::kStages, done = empty + 8 * L::kStages;
  const uint32_t part = blockIdx.x % p.parts, tile = blockIdx.x / p.parts;
  const uint32_t row = tile % p.row_tiles * kBlock, col = tile / p.row_tiles * BN;
  const uint32_t begin = (uint64_t)p.steps * part / p.parts, count = (uint32_t)((uint64_t)p.steps * (part + 1) / p.parts) - begin;
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) bar_init(full + 8 * s, 2), bar_init(empty + 8 * s, 1);
    bar_init(done, 1);
    flag = 0;
    init_visible();
    prefetch_map(&p.r.map);
    prefetch_map(&p.c.map);
  }
  pdl_wait();  // before tensor memory is taken, which a kernel in front may still hold
  if (warp == 3) tmem_alloc<L::kColumns>(smem_at(&tmem_at));
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;
  if (warp == 0) {
    [&] {
      for (uint32_t i = 0; i < count; ++i) {
        const uint32_t s = i % L::kStages, round = i / L::kStages;
        if (round) CSW_WAIT_WARP(empty + 8 * s, (round - 1) & 1);
        if (p.idle) return;
        if (elected()) {
          const uint32_t bar = full + 8 * s, to = ring_at + s * L::kStage;
          const int k = (int)(begin + i) * kBlock;
          bar_expect(bar, kTileBytes + (p.c.across ? L::kPanels * kTileBytes : BN * kBlock));
          copy_bytes_tile(to, &p.r.map, bar, p.r.across ? (int)row : k, p.r.across ? k : (int)row);
#pragma unroll
          for (int j = 0; j < L::kPanels; ++j)
            copy_bytes_tile(to + (1 + j) * kTileBytes, &p.c.map, bar, p.c.across ? (int)col + j * kBlock : k,
                            p.c.across ? k : (int)col + j * kBlock);
        }
        __syncwarp();
      }
    }();
  } else if (warp == 2) {
    [&] {
      uint32_t held[1 + L::kPanels];
      for (uint32_t i = 0; i < count; ++i) {
        if (i % 32 == 0) {  // 32 blocks' scales at a time, one to a lane
          const uint32_t k = begin + i + lane;
          const bool is = i + lane < count;
          held[0] = is ? p.r.scales[(uint64_t)(row / kBlock) * p.r.scale_step + (uint64_t)k * p.r.scale_k_step] : 0;
#pragma unroll
          for (int j = 0; j < L::kPanels; ++j)
            held[1 + j] = is && col + j * kBlock < p.n
                              ? p.c.scales[(uint64_t)(col / kBlock + j) * p.c.scale_step + (uint64_t)k * p.c.scale_k_step]
                              : 0;
        }
        const uint32_t s = i % L::kStages, round = i / L::kStages;
        if (round) CSW_WAIT_WARP(empty + 8 * s, (round - 1) & 1);
        uint4* to = reinterpret_cast<uint4*>(ring + s * L::kStage + L::kScales);
#pragma unroll
        for (int j = 0; j < 1 + L::kPanels; ++j) {
          const uint32_t w = __shfl_sync(0xffffffffu, held[j], i % 32) * 0x01010101u;
          to[32 * j + lane] = make_uint4(w, w, w, w);
        }
        async_fence();
        __syncwarp();
        if (lane == 0) bar_arrive(full + 8 * s);
      }
    }();
  } else if (warp == 1) {
    [&] {
      const uint32_t desc = scaled_desc(BN, p.r.across, p.c.across);
      const uint32_t r_step = p.r.across ? 4096 / 16 : 32 / 16, c_step = p.c.across ? 4096 / 16 : 32 / 16;
      const uint32_t r_scales = tmem + BN, c_scales = r_scales + 4;
      for (uint32_t i = 0; i < count; ++i) {
        const uint32_t s = i % L::kStages, round = i / L::kStages;
        CSW_WAIT_WARP(full + 8 * s, round & 1);
        fence_after();
        const uint32_t at = ring_at + s * L::kStage;
        const uint64_t r = tile_desc(at, kTileBytes), c = tile_desc(at + kTileBytes, kTileBytes);
        const uint64_t scales = scales_desc(at + L::kScales);
        if (elected()) {
#pragma unroll
          for (int j = 0; j < 1 + L::kPanels; ++j) copy_scales(r_scales + 4 * j, scales + j * (512 / 16));
#pragma unroll
          for (int k = 0; k < kBlock / 32; ++k)
            mma_scaled(tmem, r + k * r_step, c + k * c_step, desc, r_scales, c_scales, i || k);
          commit(empty + 8 * s);
          if (i + 1 == count) commit(done);
        }
        __syncwarp();
      }
    }();
  } else if (warp >= 4) {
    [&] {
      if (count) CSW_WAIT_WARP(done, 0);
      fence_after();
      const uint32_t lanes = (uint32_t)(32 * (warp % 4)) << 16, line = 32 * (warp % 4) + lane;
      float* const sums = reinterpret_cast<float*>(ring);
#pragma unroll 1
      for (int j = 0; j < BN; j += 32) {
        uint32_t r[32];
        float f[32];
        if (count) {
          load32(tmem + lanes + j, r);
          wait_loads(r);
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) f[k] = count ? __uint_as_float(r[k]) : 0.0f;
        if (p.parts == 1) {
          emit_any(p, row + line, col + j, f);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) sums[(j + k) * kBlock + line] = f[k];
        }
      }
    }();
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  bool bad = *reinterpret_cast<volatile uint32_t*>(&flag);
  if (bad) {  // copies on their way get time to land
    for (int i = 0; i < 1000; ++i) __nanosleep(10000);
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t*>(p.status) = 1;
      __threadfence_system();
    }
  }
  // Before the other CTAs of a cluster are waited for: one of them may wait for this tensor memory.
  if (warp == 3) tmem_free<L::kColumns>(tmem);
  if (p.parts > 1) {
    cluster_meet();
    for (uint32_t q = 0; q < p.parts; ++q) bad |= __float_as_uint(peer_float(smem_at(&flag), q)) != 0;
    const uint32_t width = BN / p.parts, each = width / 2, line = threadIdx.x % kBlock;
    const uint32_t first = part * width + threadIdx.x / kBlock * each;
    for (uint32_t j = 0; j < each; j += 2) {
      float f[2] = {0.0f, 0.0f};
      for (uint32_t q = 0; q < p.parts; ++q)
#pragma unroll
        for (int k = 0; k < 2; ++k) f[k] += peer_float(ring_at + ((first + j + k) * kBlock + line) * 4, q);
      if (bad) f[0] = f[1] = NAN;
      emit_any(p, row + line, col + first + j, f);
    }
    cluster_meet();  // nobody leaves while its sums are read
  } else if (bad) {
    float f[2] = {NAN, NAN};
    for (uint32_t j = threadIdx.x / kBlock * 2; j < BN; j += 4) emit_any(p, row + threadIdx.x % kBlock, col + j, f);
  }
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

template <int BN>
cudaError_t product(Product& p, const Fp8Matrix& r, const Fp8Matrix& c, bool r_across, bool c_across, cudaStream_t stream) {
  using L = Plan<BN>;
  if (p.steps && (!operand_of(&p.r, r, r_across, kBlock) || !operand_of(&p.c, c, c_across, std::min(BN, kBlock))))
    return cudaErrorInvalidValue;
  if (const cudaError_t e = taken(
          cudaFuncSetAttribute(fp8_product_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kShared)))
    return e;
  const uint64_t tiles = (uint64_t)p.row_tiles * ((p.n + BN - 1) / BN);
  return pdl_launch_clusters(fp8_product_kernel<BN>, (unsigned)(tiles * p.parts), p.parts, kThreads, L::kShared, stream, p);
}

}  // namespace

cudaError_t fp8_quantize_launch(const Fp8Quantize& a, cudaStream_t stream) {
  if (a.cols == 0) return cudaSuccess;
  if (a.rows == 0) return a.sums ? taken(cudaMemsetAsync(a.sums, 0, a.cols * sizeof(float), stream)) : cudaSuccess;
  const uint64_t parts = fp8_blocks(a.rows), grid = parts * fp8_blocks(a.cols);
  cudaError_t e = cudaSuccess;
  float* sums = parts > 1 ? a.partials : a.sums;
  with_type(a.type, [&](auto v) {
    using T = decltype(v);
    const bool packs = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.stride * sizeof(T) % 16 == 0;
    const auto kernel = a.sums ? fp8_quantize_kernel<T, true> : fp8_quantize_kernel<T, false>;
    e = pdl_launch(kernel, (unsigned)grid, kQuantizeThreads, 0, stream, static_cast<const T*>(a.x), a.rows, a.cols, a.stride,
                   packs, static_cast<uint8_t*>(a.codes), a.code_stride, a.scales, sums);
  });
  if (e == cudaSuccess && a.sums && parts > 1)
    e = pdl_launch(fp8_sums_kernel, (unsigned)((a.cols + 31) / 32), 256, 0, stream, (const float*)a.partials, parts, a.cols,
                   a.sums);
  return e;
}

cudaError_t fp8_dequantize_launch(const void* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols,
                                  void* out, int type, cudaStream_t stream) {
  if (rows == 0 || cols == 0) return cudaSuccess;
  cudaError_t e = cudaSuccess;
  with_type(type, [&](auto v) {
    using T = decltype(v);
    const uint64_t packs = (cols + 7) / 8;
    const bool whole = cols * sizeof(T) % 16 == 0 && cols % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    e = pdl_launch(fp8_dequantize_kernel<T>, (unsigned)((rows * packs + 255) / 256), 256, 0, stream,
                   static_cast<const uint8_t*>(codes), code_stride, scales, rows, cols, packs, whole, static_cast<T*>(out));
  });
  return e;
}

cudaError_t fp8_matmul_launch(const Fp8Matrix& a, const Fp8Matrix& b, const void* bias, int bias_type, void* out, int type,
                              cudaStream_t stream) {
  const uint64_t m = a.transposed ? a.cols : a.rows, k = a.transposed ? a.rows : a.cols;
  const uint64_t n = b.transposed ? b.rows : b.cols;
  if (m == 0 || n == 0) return cudaSuccess;
  if (const cudaError_t e = bind_context()) return e;
  Product p{};
  if (const cudaError_t e = status_word(&p.status)) return e;
  const long long limit = wait_limit();
  p.patience = limit < 0 ? -limit : limit, p.idle = limit < 0;
  p.out = out, p.bias = bias, p.type = type, p.bias_type = bias_type;
  p.steps = (uint32_t)fp8_blocks(k);
  p.exchanged = m <= 64 && n > m;
  p.packs = n * (type == 0 ? 4 : 2) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const Fp8Matrix &r = p.exchanged ? b : a, &c = p.exchanged ? a : b;
  const bool r_across = p.exchanged ? !b.transposed : a.transposed, c_across = p.exchanged ? a.transposed : !b.transposed;
  p.m = (uint32_t)(p.exchanged ? n : m), p.n = (uint32_t)(p.exchanged ? m : n);
  p.row_tiles = (uint32_t)fp8_blocks(p.m);
  const int bn = p.n <= 32 ? 32 : p.n <= 64 ? 64 : p.n <= 128 ? 128 : 256;
  const uint64_t tiles = (uint64_t)p.row_tiles * ((p.n + bn - 1) / bn), sms = sm_count();
  p.parts = 1;
  while (p.parts < 8 && p.parts * 2 <= p.steps && tiles * p.parts * 2 <= sms * (bn > kBlock ? 1 : 2)) p.parts *= 2;
  switch (bn) {
    case 32: return product<32>(p, r, c, r_across, c_across, stream);
    case 64: return product<64>(p, r, c, r_across, c_across, stream);
    case 128: return product<128>(p, r, c, r_across, c_across, stream);
    default: return product<256>(p, r, c, r_across, c_across, stream);
  }
}

}  // namespace csw
