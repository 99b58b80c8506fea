// Attention, forward and backward: launchers.  Arguments are checked by the callers (ops_abi.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/cswap_b200.h"

namespace csw {

cudaError_t attention_forward_launch(const csw_attention_shape& s, const csw_attention_operand& q,
                                     const csw_attention_operand& k, const csw_attention_operand& v,
                                     const csw_attention_operand& o, float* lse, cudaStream_t stream);
struct AttentionBackward {
  csw_attention_operand q, k, v, o, dout, dq, dk, dv;
  const float* lse;
  float* workspace;  // attention_workspace_values(s)
};
// float32 values that a backward pass needs on the CURRENT device
uint64_t attention_workspace_values(const csw_attention_shape& s);
cudaError_t attention_backward_launch(const csw_attention_shape& s, const AttentionBackward& a, cudaStream_t stream);

}  // namespace csw
