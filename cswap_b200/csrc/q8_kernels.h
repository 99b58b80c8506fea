// 8-bit checkpoints and GELU on them: launchers.  Arguments are checked by the callers (ops_abi.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace csw {

constexpr uint64_t kQ8Group = 128;  // values that share a scale
// bytes of the codes of n values, and with them the offset of the scales
inline uint64_t q8_scales_at(uint64_t n) { return (n + 15) / 16 * 16; }
inline uint64_t q8_groups(uint64_t n) { return n / kQ8Group + (n % kQ8Group != 0); }

cudaError_t q8_compress_launch(const void* x, int type, uint64_t n, void* packed, cudaStream_t stream);
cudaError_t q8_decompress_launch(const void* packed, uint64_t n, void* out, int type, cudaStream_t stream);
cudaError_t gelu_forward_launch(const void* x, int type, uint64_t n, void* y, void* packed, cudaStream_t stream);
cudaError_t gelu_backward_launch(const void* dy, int type, const void* packed, uint64_t n, void* dx, void* again,
                                 cudaStream_t stream);

}  // namespace csw
