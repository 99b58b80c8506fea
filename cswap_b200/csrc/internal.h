// Declarations shared between the translation units of the library.
#pragma once
#include <cuda_runtime.h>

#include "../../include/cswap_b200.h"

namespace csw {

// records the runtime error for csw_last_cuda_error() and returns CSW_ERR_CUDA
csw_status cuda_fail(cudaError_t e);

// the status word of the CURRENT device (created on first use; it is zero unless a
// kernel gave up on a bounded wait)
csw_status device_state(int** d_status);

// SMs of the CURRENT device: 148, or what a partition of it has.  Touches no memory of the
// device and synchronises nothing.
int sm_count();

// Reads (and clears) the status word of the kernels that wait on their own copies, of the CURRENT device, without waiting for
// them; set by the translation unit that has them, null in a program linked without it.
extern cudaError_t (*take_kernel_status)(int* value);

}  // namespace csw
