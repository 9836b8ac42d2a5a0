// gate.cu — hymoe_route and hymoe_route_backward: a router's logits to every token's experts
// and weights, and the gradient back to the logits.
//
// One warp per token, the token's experts spread over the lanes (expert e = lane + 32 i in
// register i).  The selection is decided in double precision; the weights of the selected
// experts are formed with their largest score's exponent taken out, so a renormalised row is
// right however small its scores are.
#include <math.h>

#include "common.cuh"
#include "entry.h"
#include "kernels.h"

namespace hymoe {
namespace {

constexpr int kGateWarps = 16;  // tokens per CTA
constexpr unsigned kAll = 0xffffffffu;

template <typename T>
__device__ __forceinline__ float gate_load(const T* p);
template <>
__device__ __forceinline__ float gate_load<float>(const float* p) { return __ldg(p); }
template <>
__device__ __forceinline__ float gate_load<__half>(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float gate_load<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }

template <typename T>
__device__ __forceinline__ T gate_store(float v);
template <>
__device__ __forceinline__ float gate_store<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half gate_store<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 gate_store<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
}

// The logit as the definition takes it: -inf closes the expert, +inf is FLT_MAX.
__device__ __forceinline__ float clean_logit(float z) {
    return z != z ? -INFINITY : fminf(z, 3.402823466e38f);
}

struct GateArgs {
    const float* bias;
    int E, K, score, n_group, topk_group, group_score, norm;
    float scale;
    int* idx;
    float* weights;
    float* scores;
    int* counts;
};

// Best (value, expert) of the warp: the larger value, the lower expert where they tie.
__device__ __forceinline__ void warp_best(double& v, int& e) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const double ov = __shfl_xor_sync(kAll, v, o);
        const int oe = __shfl_xor_sync(kAll, e, o);
        if (ov > v || (ov == v && oe < e)) {
            v = ov;
            e = oe;
        }
    }
}

template <typename T, int EPL>
__global__ __launch_bounds__(32 * kGateWarps) void gate_kernel(const T* __restrict__ logits, size_t ld,
                                                               uint32_t n_tok, GateArgs a) {
    extern __shared__ double cbuf[];  // groups only: [kGateWarps][E]
    __shared__ int cnt[HYMOE_GATE_MAX_EXPERTS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int E = a.E, K = a.K;
    if (a.counts != nullptr) {
        for (int e = threadIdx.x; e < E; e += blockDim.x) cnt[e] = 0;
        __syncthreads();
    }
    for (size_t t = static_cast<size_t>(blockIdx.x) * kGateWarps + warp; t < n_tok;
         t += static_cast<size_t>(gridDim.x) * kGateWarps) {
        float z[EPL];
        double s[EPL], c[EPL];
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = lane + 32 * i;
            z[i] = e < E ? clean_logit(gate_load(logits + t * ld + e)) : -INFINITY;
            m = fmaxf(m, z[i]);
        }
        if (a.score == HYMOE_SCORE_SIGMOID) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] = z[i] == -INFINITY ? 0.0 : 1.0 / (1.0 + exp(-static_cast<double>(z[i])));
        } else {
            m = warp_max(m);
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                s[i] = z[i] == -INFINITY ? 0.0 : exp(static_cast<double>(z[i]) - m);
                sum += s[i];
            }
            sum = warp_sum(sum);
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = lane + 32 * i;
            if (a.scores != nullptr && e < E) a.scores[t * E + e] = static_cast<float>(s[i]);
            double b = 0.0;
            if (a.bias != nullptr && e < E) b = clean_logit(__ldg(a.bias + e));
            c[i] = z[i] == -INFINITY ? -INFINITY : a.bias != nullptr ? s[i] + b : static_cast<double>(z[i]);
        }
        if (a.n_group > 0) {
            // group g = lane: its value from the warp's row of c (or of s: two scores are added)
            const int gs = E / a.n_group;
            double* row = cbuf + static_cast<size_t>(warp) * E;
            const bool two = a.group_score == HYMOE_GROUP_TOP2;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const int e = lane + 32 * i;
                if (e < E) row[e] = two && a.bias == nullptr && z[i] != -INFINITY ? s[i] : c[i];
            }
            __syncwarp();
            double b1 = -INFINITY, b2 = -INFINITY;
            if (lane < a.n_group)
                for (int j = 0; j < gs; ++j) {
                    const double v = row[lane * gs + j];
                    if (v > b1) {
                        b2 = b1;
                        b1 = v;
                    } else if (v > b2) {
                        b2 = v;
                    }
                }
            const double val = two && b2 > -INFINITY ? b1 + b2 : b1;
            bool mine = lane < a.n_group;  // still a candidate
            unsigned kept = 0;
            for (int r = 0; r < a.topk_group; ++r) {
                double v = mine ? val : -INFINITY;
                int g = mine ? lane : 64;
                warp_best(v, g);
                if (v == -INFINITY) break;
                kept |= 1u << g;
                if (g == lane) mine = false;
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const int e = lane + 32 * i;
                if (e < E && !((kept >> (e / gs)) & 1u)) c[i] = -INFINITY;
            }
        }
        int sel = -1;  // lane k: the k-th selection
        float zsel = -INFINITY;
        double ssel = 0.0;
        for (int k = 0; k < K; ++k) {
            double v = -INFINITY;
            int e = 1 << 20;
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (c[i] > v) {
                    v = c[i];
                    e = lane + 32 * i;
                }
            warp_best(v, e);
            if (v == -INFINITY) break;
            float zk = 0.f;
            double sk = 0.0;
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (e == lane + 32 * i) {
                    c[i] = -INFINITY;
                    zk = z[i];
                    sk = s[i];
                }
            zk = __shfl_sync(kAll, zk, e & 31);
            sk = __shfl_sync(kAll, sk, e & 31);
            if (lane == k) {
                sel = e;
                zsel = zk;
                ssel = sk;
            }
        }
        double w = ssel;
        if (a.norm) {
            // s_k / sum s: both over e^M, M the largest selected logit (at most 0 for a sigmoid)
            double mm = warp_max(zsel);
            if (a.score == HYMOE_SCORE_SIGMOID) mm = fmin(mm, 0.0);
            double x = 0.0;
            if (sel >= 0)
                x = a.score == HYMOE_SCORE_SIGMOID
                        ? exp(fmin(static_cast<double>(zsel), 0.0) - mm) / (1.0 + exp(-fabs(static_cast<double>(zsel))))
                        : exp(static_cast<double>(zsel) - mm);
            const double tot = warp_sum(x);
            w = tot > 0.0 ? x / tot : 0.0;
        }
        if (lane < K) {
            a.idx[t * K + lane] = sel;
            a.weights[t * K + lane] = static_cast<float>(w * a.scale);
            if (a.counts != nullptr && sel >= 0) atomicAdd(&cnt[sel], 1);
        }
    }
    if (a.counts != nullptr) {
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += blockDim.x)
            if (cnt[e]) atomicAdd(a.counts + e, cnt[e]);  // whole numbers: any order gives the same
    }
}

struct GateGradArgs {
    const int* idx;
    const float* dw;
    const float* ds;
    int E, K, score, norm;
    float scale;
};

// dz = (ds/dz)^T (dL/ds), with dL/ds the score gradient plus, at the selected experts,
//   norm: scale (dw_k - sum_j dw_j n_j) n_k / s_k (n = the renormalised weights), else scale dw_k.
// The factor n_k / s_k is never formed: it meets s_k (1 - s_k) or s_k in the product.
template <typename T, int EPL>
__global__ __launch_bounds__(32 * kGateWarps) void gate_grad_kernel(const T* logits, size_t ld, T* d_logits,
                                                                    size_t ldd, uint32_t n_tok, GateGradArgs a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int E = a.E, K = a.K;
    const size_t t = static_cast<size_t>(blockIdx.x) * kGateWarps + warp;
    if (t >= n_tok) return;
    float z[EPL];
    double s[EPL], gw[EPL], gs[EPL];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = lane + 32 * i;
        z[i] = e < E ? clean_logit(gate_load(logits + t * ld + e)) : -INFINITY;
        m = fmaxf(m, z[i]);
        gw[i] = 0.0;
        gs[i] = a.ds != nullptr && e < E && z[i] != -INFINITY ? a.ds[t * E + e] : 0.0;
    }
    if (a.score == HYMOE_SCORE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) s[i] = z[i] == -INFINITY ? 0.0 : 1.0 / (1.0 + exp(-static_cast<double>(z[i])));
    } else {
        m = warp_max(m);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            s[i] = z[i] == -INFINITY ? 0.0 : exp(static_cast<double>(z[i]) - m);
            sum += s[i];
        }
        sum = warp_sum(sum);
#pragma unroll
        for (int i = 0; i < EPL; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
    }
    // lane k: selection k, its logit and score
    int sel = lane < K ? a.idx[t * K + lane] : -1;
    double dw = sel >= 0 && sel < E ? static_cast<double>(a.dw[t * K + lane]) * a.scale : 0.0;
    if (sel < 0 || sel >= E) sel = -1;
    float zsel = -INFINITY;
    double ssel = 0.0;
    for (int k = 0; k < K; ++k) {
        const int e = __shfl_sync(kAll, sel, k);
        if (e < 0) continue;
        float zk = 0.f;
        double sk = 0.0;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (i == (e >> 5)) {
                zk = z[i];
                sk = s[i];
            }
        zk = __shfl_sync(kAll, zk, e & 31);
        sk = __shfl_sync(kAll, sk, e & 31);
        if (lane == k) {
            zsel = zk;
            ssel = sk;
        }
    }
    if (zsel == -INFINITY) {
        sel = -1;
        dw = 0.0;
    }
    // lane k's term: dL/ds_k * s_k
    double term = dw * ssel;
    if (a.norm) {
        double mm = warp_max(zsel);
        if (a.score == HYMOE_SCORE_SIGMOID) mm = fmin(mm, 0.0);
        double x = 0.0;
        if (sel >= 0)
            x = a.score == HYMOE_SCORE_SIGMOID
                    ? exp(fmin(static_cast<double>(zsel), 0.0) - mm) / (1.0 + exp(-fabs(static_cast<double>(zsel))))
                    : exp(static_cast<double>(zsel) - mm);
        const double tot = warp_sum(x);
        const double n = tot > 0.0 ? x / tot : 0.0;
        term = n * (dw - warp_sum(dw * n));
    }
    for (int k = 0; k < K; ++k) {
        const int e = __shfl_sync(kAll, sel, k);
        const double v = __shfl_sync(kAll, term, k);
        if (e < 0) continue;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (e == lane + 32 * i) gw[i] += v;
    }
    double dot = 0.0;  // softmax: sum_e (dL/ds_e) s_e
    if (a.score == HYMOE_SCORE_SOFTMAX) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) dot += gw[i] + gs[i] * s[i];
        dot = warp_sum(dot);
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = lane + 32 * i;
        if (e >= E) continue;
        double d = gw[i] + gs[i] * s[i];
        if (a.score == HYMOE_SCORE_SIGMOID)
            d *= 1.0 / (1.0 + exp(static_cast<double>(z[i])));  // 1 - s without the cancellation
        else
            d -= s[i] * dot;
        d_logits[t * ldd + e] = gate_store<T>(z[i] == -INFINITY ? 0.f : static_cast<float>(d));
    }
}

template <typename T>
cudaError_t launch_gate_t(const hymoe_mat& x, uint32_t n_tok, const GateArgs& a, cudaStream_t st) {
    const size_t chunks = (static_cast<size_t>(n_tok) + kGateWarps - 1) / kGateWarps;
    const int grid = static_cast<int>(chunks < 148 * 8 ? chunks : 148 * 8);
    const size_t smem = a.n_group > 0 ? sizeof(double) * kGateWarps * a.E : 0;
    const T* p = static_cast<const T*>(x.data);
    const size_t ld = static_cast<size_t>(x.ld);
    auto go = [&](auto kern) {
        if (smem > 40 * 1024) {  // with the static counters beyond the default 48 KB
            const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (e != cudaSuccess) return e;
        }
        kern<<<grid, 32 * kGateWarps, smem, st>>>(p, ld, n_tok, a);
        return cudaGetLastError();
    };
    if (a.E <= 32) return go(gate_kernel<T, 1>);
    if (a.E <= 64) return go(gate_kernel<T, 2>);
    if (a.E <= 128) return go(gate_kernel<T, 4>);
    if (a.E <= 256) return go(gate_kernel<T, 8>);
    return go(gate_kernel<T, 16>);
}

template <typename T>
cudaError_t launch_gate_grad_t(const hymoe_mat& x, const hymoe_mat& d, uint32_t n_tok, const GateGradArgs& a,
                               cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>((static_cast<size_t>(n_tok) + kGateWarps - 1) / kGateWarps);
    auto go = [&](auto kern) {
        kern<<<grid, 32 * kGateWarps, 0, st>>>(static_cast<const T*>(x.data), static_cast<size_t>(x.ld),
                                               static_cast<T*>(d.data), static_cast<size_t>(d.ld), n_tok, a);
        return cudaGetLastError();
    };
    if (a.E <= 32) return go(gate_grad_kernel<T, 1>);
    if (a.E <= 64) return go(gate_grad_kernel<T, 2>);
    if (a.E <= 128) return go(gate_grad_kernel<T, 4>);
    if (a.E <= 256) return go(gate_grad_kernel<T, 8>);
    return go(gate_grad_kernel<T, 16>);
}

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
        if (cudaMemsetAsync(counts, 0, E * 4, st) != cudaSuccess) {
            cudaGetLastError();
            return entry_fail(HYMOE_ERR_CUDA, "hymoe_route: cudaMemsetAsync failed");
        }
    }
    if (T == 0) return HYMOE_OK;
    GateArgs a{bias, static_cast<int>(E), static_cast<int>(K), gate->score, static_cast<int>(gate->n_group),
               static_cast<int>(gate->topk_group), gate->group_score, gate->norm_topk_prob != 0,
               gate->routed_scaling_factor, idx, weights, scores, counts};
    const cudaError_t e = logits->type == HYMOE_TYPE_F32   ? launch_gate_t<float>(*logits, n_tokens, a, st)
                          : logits->type == HYMOE_TYPE_F16 ? launch_gate_t<__half>(*logits, n_tokens, a, st)
                                                           : launch_gate_t<__nv_bfloat16>(*logits, n_tokens, a, st);
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
        logits->type == HYMOE_TYPE_F32   ? launch_gate_grad_t<float>(*logits, *d_logits, n_tokens, a, st)
        : logits->type == HYMOE_TYPE_F16 ? launch_gate_grad_t<__half>(*logits, *d_logits, n_tokens, a, st)
                                         : launch_gate_grad_t<__nv_bfloat16>(*logits, *d_logits, n_tokens, a, st);
    if (e != cudaSuccess) return entry_fail(HYMOE_ERR_CUDA, "hymoe_route_backward: kernel launch failed");
    return HYMOE_OK;
}
