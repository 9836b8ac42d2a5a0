// gate.cu — hymoe_route and hymoe_route_backward: the checks and launches (kernels in gate.cuh).
#include "gate.cuh"

namespace hymoe {
extern template cudaError_t launch_gate<float>(const hymoe_mat&, uint32_t, const GateArgs&, cudaStream_t);
extern template cudaError_t launch_gate<__half>(const hymoe_mat&, uint32_t, const GateArgs&, cudaStream_t);
extern template cudaError_t launch_gate<__nv_bfloat16>(const hymoe_mat&, uint32_t, const GateArgs&, cudaStream_t);
extern template cudaError_t launch_gate_grad<float>(const hymoe_mat&, const hymoe_mat&, uint32_t, const GateGradArgs&, cudaStream_t);
extern template cudaError_t launch_gate_grad<__half>(const hymoe_mat&, const hymoe_mat&, uint32_t, const GateGradArgs&, cudaStream_t);
extern template cudaError_t launch_gate_grad<__nv_bfloat16>(const hymoe_mat&, const hymoe_mat&, uint32_t, const GateGradArgs&, cudaStream_t);

// Why a gate cannot route E experts, K of them to a token; nullptr where it can.
const char* gate_problem(const hymoe_gate* g, uint32_t E, uint32_t K) {
    if (!g) return "null gate";
    if (E == 0 || E > HYMOE_GATE_MAX_EXPERTS) return "n_experts must be 1..HYMOE_GATE_MAX_EXPERTS (512)";
    if (K == 0 || K > HYMOE_GATE_MAX_TOPK || K > E) return "topk must be 1..HYMOE_GATE_MAX_TOPK (32), at most n_experts";
    if (g->score != HYMOE_SCORE_SOFTMAX && g->score != HYMOE_SCORE_SIGMOID) return "unknown score";
    if (g->group_score != HYMOE_GROUP_MAX && g->group_score != HYMOE_GROUP_TOP2) return "unknown group_score";
    if (g->n_group != 0 && (g->n_group > 32 || E % g->n_group != 0 || g->topk_group == 0 || g->topk_group > g->n_group))
        return "n_group must be 1..32 and divide n_experts, topk_group 1..n_group";
    if (!isfinite(g->routed_scaling_factor)) return "routed_scaling_factor is not finite";
    return nullptr;
}

namespace {

bool any_overlap(const EntrySpan* out, int n_out, const EntrySpan* in, int n_in) {
    for (int i = 0; i < n_out; ++i) {
        for (int j = i + 1; j < n_out; ++j)
            if (entry_overlap(out[i], out[j])) return true;
        for (int j = 0; j < n_in; ++j)
            if (entry_overlap(out[i], in[j])) return true;
    }
    return false;
}

}  // namespace
}  // namespace hymoe

using namespace hymoe;

extern "C" hymoe_status hymoe_route(const hymoe_gate* gate, const hymoe_mat* logits, const float* bias,
                                    uint32_t n_tokens, uint32_t n_experts, uint32_t topk, int32_t* idx,
                                    float* weights, float* scores, int32_t* counts, void* stream) {
    set_thread_error("");
    if (const char* why = gate_problem(gate, n_experts, topk)) return entry_fail(HYMOE_ERR_INVALID_ARG, why);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t T = n_tokens, E = n_experts, K = topk;
    int dev = -1;
    if (T > 0) {
        if (!entry_mat_ok(logits, n_experts) || !idx || !weights)
            return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route: logits must be an F32/F16/BF16 matrix with ld >= "
                                                     "n_experts, idx and weights not null");
        if (!entry_aligned(bias, 4) || !entry_aligned(idx, 4) || !entry_aligned(weights, 4) ||
            !entry_aligned(scores, 4) || !entry_aligned(counts, 4))
            return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route: pointers must be 4-byte aligned");
        const EntrySpan out[4] = {entry_span(idx, T * K * 4), entry_span(weights, T * K * 4),
                                  entry_span(scores, scores ? T * E * 4 : 0), entry_span(counts, counts ? E * 4 : 0)};
        const EntrySpan in[2] = {entry_span(logits, n_tokens, n_experts), entry_span(bias, bias ? E * 4 : 0)};
        if (any_overlap(out, 4, in, 2)) return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route: outputs overlap");
    }
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return entry_fail(HYMOE_ERR_CUDA, "hymoe_route: cudaGetDevice failed");
    }
    if (T > 0 && (!entry_on_device(logits->data, dev) || !entry_on_device(idx, dev) || !entry_on_device(weights, dev) ||
                  (bias && !entry_on_device(bias, dev)) || (scores && !entry_on_device(scores, dev))))
        return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route: every pointer must be memory of the current device");
    if (counts) {
        if (!entry_aligned(counts, 4) || !entry_on_device(counts, dev))
            return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route: every pointer must be memory of the current device");
        // (one CTA writes the counts itself)
        if ((T == 0 || T > kGateWarps) && cudaMemsetAsync(counts, 0, E * 4, st) != cudaSuccess) {
            cudaGetLastError();
            return entry_fail(HYMOE_ERR_CUDA, "hymoe_route: cudaMemsetAsync failed");
        }
    }
    if (T == 0) return HYMOE_OK;
    GateArgs a{bias, static_cast<int>(E), static_cast<int>(K), gate->score, static_cast<int>(gate->n_group),
               static_cast<int>(gate->topk_group), gate->group_score, gate->norm_topk_prob != 0, 0u,
               gate->routed_scaling_factor, idx, weights, scores, counts, nullptr};
    while (a.mask + 1 < n_experts) a.mask = 2 * a.mask + 1;
    const cudaError_t e = logits->type == HYMOE_TYPE_F32   ? launch_gate<float>(*logits, n_tokens, a, st)
                          : logits->type == HYMOE_TYPE_F16 ? launch_gate<__half>(*logits, n_tokens, a, st)
                                                           : launch_gate<__nv_bfloat16>(*logits, n_tokens, a, st);
    if (e != cudaSuccess) return entry_fail(HYMOE_ERR_CUDA, "hymoe_route: kernel launch failed");
    return HYMOE_OK;
}

extern "C" hymoe_status hymoe_route_backward(const hymoe_gate* gate, const hymoe_mat* logits, const int32_t* idx,
                                             const float* d_weights, const float* d_scores, uint32_t n_tokens,
                                             uint32_t n_experts, uint32_t topk, const hymoe_mat* d_logits,
                                             void* stream) {
    set_thread_error("");
    if (const char* why = gate_problem(gate, n_experts, topk)) return entry_fail(HYMOE_ERR_INVALID_ARG, why);
    if (n_tokens == 0) return HYMOE_OK;
    const size_t T = n_tokens, E = n_experts, K = topk;
    if (!entry_mat_ok(logits, n_experts) || !entry_mat_ok(d_logits, n_experts) || logits->type != d_logits->type ||
        !idx || !d_weights)
        return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route_backward: logits and d_logits must be matrices of one "
                                                 "type (F32/F16/BF16) with ld >= n_experts, idx and d_weights not null");
    if (!entry_aligned(idx, 4) || !entry_aligned(d_weights, 4) || !entry_aligned(d_scores, 4))
        return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route_backward: pointers must be 4-byte aligned");
    const EntrySpan out = entry_span(d_logits, n_tokens, n_experts);
    const bool in_place = d_logits->data == logits->data && d_logits->ld == logits->ld;
    if ((!in_place && entry_overlap(out, entry_span(logits, n_tokens, n_experts))) ||
        entry_overlap(out, entry_span(idx, T * K * 4)) || entry_overlap(out, entry_span(d_weights, T * K * 4)) ||
        (d_scores && entry_overlap(out, entry_span(d_scores, T * E * 4))))
        return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_route_backward: d_logits overlaps an input");
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return entry_fail(HYMOE_ERR_CUDA, "hymoe_route_backward: cudaGetDevice failed");
    }
    if (!entry_on_device(logits->data, dev) || !entry_on_device(d_logits->data, dev) || !entry_on_device(idx, dev) ||
        !entry_on_device(d_weights, dev) || (d_scores && !entry_on_device(d_scores, dev)))
        return entry_fail(HYMOE_ERR_INVALID_ARG,
                          "hymoe_route_backward: every pointer must be memory of the current device");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    GateGradArgs a{idx, d_weights, d_scores, static_cast<int>(E), static_cast<int>(K), gate->score,
                   gate->norm_topk_prob != 0, gate->routed_scaling_factor};
    const cudaError_t e =
        logits->type == HYMOE_TYPE_F32   ? launch_gate_grad<float>(*logits, *d_logits, n_tokens, a, st)
        : logits->type == HYMOE_TYPE_F16 ? launch_gate_grad<__half>(*logits, *d_logits, n_tokens, a, st)
                                         : launch_gate_grad<__nv_bfloat16>(*logits, *d_logits, n_tokens, a, st);
    if (e != cudaSuccess) return entry_fail(HYMOE_ERR_CUDA, "hymoe_route_backward: kernel launch failed");
    return HYMOE_OK;
}
