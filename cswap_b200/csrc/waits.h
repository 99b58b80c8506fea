// What the kernels that wait on their own copies and products share on the host: the word that tells of a wait that ran
// out, the limit of the waits, and the descriptions of tensors for tile copies.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace csw {

// The CURRENT device's word of host memory, which kernels set where a wait ran out and the host reads without waiting for
// anything.
cudaError_t status_word(uint32_t** word);
// Whether a kernel on the CURRENT device has given up on a wait since this was last asked; waits for nothing.
cudaError_t take_status(int* gave_up);
// Clocks that a wait may last, of calls from now on; negative: as csw_attention_wait_limit says.
long long wait_limit();
void set_wait_limit(long long clocks);

// The driver's function that describes a tensor for tile copies; null where there is none.
using TileEncoder = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
TileEncoder tile_encoder();
// Describing a tensor for tile copies is a call of the driver, which needs the device's context on this thread; a
// thread that has made no call of the runtime yet (autograd's, say) has none.
cudaError_t bind_context();

}  // namespace csw
