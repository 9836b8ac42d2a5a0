// gate_f16.cu — the routing kernels for F16 logits.
#include "gate.cuh"

namespace hymoe {
template cudaError_t launch_gate<__half>(const hymoe_mat&, uint32_t, const GateArgs&, cudaStream_t);
template cudaError_t launch_gate_grad<__half>(const hymoe_mat&, const hymoe_mat&, uint32_t, const GateGradArgs&, cudaStream_t);
}  // namespace hymoe
