// gate_f32.cu — the routing kernels for F32 logits.
#include "gate.cuh"

namespace hymoe {
template cudaError_t launch_gate<float>(const hymoe_mat&, uint32_t, const GateArgs&, cudaStream_t);
template cudaError_t launch_gate_grad<float>(const hymoe_mat&, const hymoe_mat&, uint32_t, const GateGradArgs&, cudaStream_t);
}  // namespace hymoe
