// The optimizer's step over many tensors, the norm of their gradients, and its 8-bit state: launchers.  Arguments are checked
// by the callers (ops_abi.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/cswap_b200.h"

namespace csw {

cudaError_t adamw_launch(const csw_adamw_tensor* tensors, size_t count, const csw_adamw_options& o, cudaStream_t stream);
// pack: averages in 32 bits to the 8-bit state, else the other way round
cudaError_t adamw8_convert_launch(const csw_adamw_tensor* tensors, size_t count, bool pack, cudaStream_t stream);
// doubles of workspace that the norm of these tensors needs on the CURRENT device
uint64_t gradient_norm_partials(const csw_adamw_tensor* tensors, size_t count);
cudaError_t gradient_norm_launch(const csw_adamw_tensor* tensors, size_t count, float* norm, double* partials,
                                 cudaStream_t stream);

}  // namespace csw
