// gate_f32.cu — the routing kernels for F32 logits.
#include "gate.cuh"

namespace hymoe {
template cudaError_t launch_gate<float>(const hymoe_mat&, uint32_t, const GateArgs&, cudaStream_t);
template cudaError_t launch_gate_grad<float>(const hymoe_mat&, const hymoe_mat&, uint32_t, const GateGradArgs&, cudaStream_t);

namespace {

// The block's top-K step by a gate: one CTA per dispatch chunk of 16 tokens, a warp per token, and
// the chunk's pairs per slot.  Launched in programmatic chains like the block's other kernels.
template <bool RUN, bool SIG>
__global__ __launch_bounds__(32 * kRouterTok) void route_block_kernel(const float* logits, int T,
                                                                      const __grid_constant__ GateArgs a, int* chunk_counts) {
    __shared__ int cnt[64];
    __shared__ float gbuf[kRouterTok][64];
    griddep_wait();
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x < 64) cnt[threadIdx.x] = 0;
    __syncthreads();
    const int t = blockIdx.x * kRouterTok + warp;
    if (t < T) {
        const float* row = logits + static_cast<size_t>(t) * a.E;
        float bias[2];
        load_bias<2, RUN>(a, bias);
        Vec<float, 2> raw;
        fetch_row<float, 2, RUN>(row, a.E, raw);
        int sel;
        float w;
        if (route_token<float, 2, RUN, SIG, true>(row, raw, a.scores != nullptr ? a.scores + static_cast<size_t>(t) * a.E : nullptr,
                                                  a, bias, gbuf[warp], sel, w))
            put_choice(a, t, sel, w, cnt);
        else
            route_exact<float>(row, t, a, cnt);
    }
    __syncthreads();
    if (threadIdx.x < static_cast<unsigned>(a.E)) chunk_counts[static_cast<size_t>(blockIdx.x) * a.E + threadIdx.x] = cnt[threadIdx.x];
}

}  // namespace

cudaError_t launch_gate_block(const float* logits, int T, int E, int K, const hymoe_gate& gate, const float* bias,
                              float* probs, float* topk_w, int* topk_idx, int* chunk_counts, const int* slot_of,
                              cudaStream_t st, bool pdl) {
    if (T <= 0) return cudaSuccess;
    if (E < 1 || E > 64 || K < 1 || K > E || K > 32) return cudaErrorInvalidValue;
    GateArgs a{bias, E, K, gate.score, static_cast<int>(gate.n_group), static_cast<int>(gate.topk_group),
               gate.group_score, gate.norm_topk_prob != 0, 63u, gate.routed_scaling_factor, topk_idx, topk_w, probs, nullptr,
               slot_of};
    const bool run = E == 64 && (gate.n_group == 0 || 32 % gate.n_group == 0) && row_runs(logits, E, sizeof(float), E) &&
                     (probs == nullptr || row_runs(probs, E, sizeof(float), E));
    const bool sig = gate.score == HYMOE_SCORE_SIGMOID;
    auto kern = run ? (sig ? route_block_kernel<true, true> : route_block_kernel<true, false>)
                    : (sig ? route_block_kernel<false, true> : route_block_kernel<false, false>);
    return launch_kernel(pdl, kern, dim3((T + kRouterTok - 1) / kRouterTok), dim3(32 * kRouterTok), 0, st, logits, T, a,
                         chunk_counts);
}

}  // namespace hymoe
