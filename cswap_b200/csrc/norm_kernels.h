// Layer norm, forward and backward: launchers.  Arguments are checked by the callers (ops_abi.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace csw {

struct NormForward {
  const void *x, *residual, *weight, *bias;  // residual, weight and bias may be null
  void *y, *sum;                             // sum: x + residual in the values' type, where residual is given
  float *mean, *rstd;
  int type, param_type;
  uint64_t rows, cols;
  float eps;
};
struct NormBackward {
  const void *dy, *x;
  const float *mean, *rstd;
  const void* weight;  // may be null
  void *dx, *dweight, *dbias;  // dweight and dbias may be null
  float* workspace;            // norm_backward_partials(rows, cols) x 2 x cols
  int type, param_type;
  uint64_t rows, cols;
};

cudaError_t norm_forward_launch(const NormForward& a, cudaStream_t stream);
// rows of partial sums that a backward pass leaves behind for its second launch
uint64_t norm_backward_partials(uint64_t rows, uint64_t cols);
cudaError_t norm_backward_launch(const NormBackward& a, cudaStream_t stream);

}  // namespace csw
