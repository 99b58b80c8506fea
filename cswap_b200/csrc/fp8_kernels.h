// Matrices in 8-bit floating point with a scale for each 128 x 128 block, and their products: launchers.  Arguments are
// checked by the callers (ops_abi.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace csw {

constexpr uint64_t kFp8Block = 128;  // rows and columns of a block
inline uint64_t fp8_blocks(uint64_t n) { return n / kFp8Block + (n % kFp8Block != 0); }

struct Fp8Quantize {
  const void* x;
  int type;
  uint64_t rows, cols, stride;  // stride: of a row of x, in values
  void* codes;
  uint64_t code_stride;         // a multiple of 16, cols at least
  uint8_t* scales;              // [blocks of rows][blocks of columns]
  void* sums;                   // may be null
  int sums_type;
  float* partials;              // fp8_blocks(rows) x cols where sums is not null and rows > 128
};
cudaError_t fp8_quantize_launch(const Fp8Quantize& a, cudaStream_t stream);
cudaError_t fp8_dequantize_launch(const void* codes, uint64_t code_stride, const uint8_t* scales, uint64_t rows, uint64_t cols,
                                  void* out, int type, cudaStream_t stream);

// A matrix as it is stored, and whether the product takes it transposed
struct Fp8Matrix {
  const void* codes;
  const uint8_t* scales;
  uint64_t rows, cols, stride;
  bool transposed;
};
// out[m][n] = a b + bias[n]; a is m x k and b k x n as the product takes them
cudaError_t fp8_matmul_launch(const Fp8Matrix& a, const Fp8Matrix& b, const void* bias, int bias_type, void* out, int type,
                              cudaStream_t stream);

// Whether x weight^T is one launch, which quantizes x itself: x.codes and x.scales are then not used.
bool fp8_linear_at_once(uint64_t rows, uint64_t cols, uint64_t outs);
// out = x weight^T + bias; weight is taken transposed
cudaError_t fp8_linear_launch(const Fp8Quantize& x, const Fp8Matrix& weight, const void* bias, int bias_type, void* out,
                              int type, cudaStream_t stream);

}  // namespace csw
