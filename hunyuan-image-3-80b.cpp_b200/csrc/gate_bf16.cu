// gate_bf16.cu — the routing kernels for BF16 logits.
#include "gate.cuh"

namespace hymoe {
template cudaError_t launch_gate<__nv_bfloat16>(const hymoe_mat&, uint32_t, const GateArgs&, cudaStream_t);
template cudaError_t launch_gate_grad<__nv_bfloat16>(const hymoe_mat&, const hymoe_mat&, uint32_t, const GateGradArgs&, cudaStream_t);
}  // namespace hymoe
