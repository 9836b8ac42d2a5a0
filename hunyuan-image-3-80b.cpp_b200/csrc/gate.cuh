// gate.cuh — the routing kernels (gate_f32.cu, gate_f16.cu and gate_bf16.cu compile them for their
// type of logits; gate.cu has the entry points).
//
// One warp per token, the token's experts in registers: EPL consecutive ones per lane where the
// experts are 32 EPL and the rows are aligned (whole vectors are loaded, the lower of two equal
// experts is in the lower lane, and a group of experts is a run of lanes), else expert lane + 32 i.
//
// Selection.  Without a bias the order is that of the logits; with one, and for the sum of a group's
// two best, it is that of s + b in double precision.  Every expert's value becomes a key: its bits
// mapped to a whole number of the same order, the lowest bits replaced by E - 1 - expert.  The lanes
// sort their keys once; a round of the selection is one warp-wide maximum of the lanes' first keys,
// which names the expert by itself, and a shift in the lane that held it.
//
// What the replaced bits and fp32 hide is then checked.  16-bit logits lose nothing.  The selected
// experts' values are formed again in fp32 and neighbours compared: with the documented errors of the
// fp32 functions (ex2.approx 2^-22 relative and half a step of its argument, times s (1 - s),
// rcp.approx 1 ulp; expf 1 ulp and the roundings of a softmax's sum) a value is off by less than 2^-21
// (sigmoid) or 2^-20 (softmax) plus 2^-23 of itself, so values further apart than twice that are in
// the exact order, and two experts of the same logit and bias tie in any precision; the best one left
// out is compared too, and the next one as the most that its key can stand for.
//
// Weights come from the selected logits with the largest one's exponent taken out, so a
// renormalised row is right however small its scores are.
//
// A token whose choices cannot be proven has its K + 1 best ordered in double precision (settle);
// only where that does not prove them either, or which groups are kept is in doubt, all its experts
// are (route_exact).
//
// Bound by instructions, and by latency in short calls: 128 experts and 6 choices with a bias,
// bf16, take 3.0 us for 256 tokens (a warp each), 27.6 us for 131072 (a thread each, some 39 instructions
// an expert: issue slots 55% busy; 60.6 by warps, some 400 warp instructions a token, while its logits
// are 256 bytes); 256 experts in 8 groups 12 us for 8323 tokens (26 before the candidates were settled by themselves: one token selected again in
// full took longer than all the others).
#pragma once

#include <math.h>

#include "common.cuh"
#include "entry.h"
#include "kernels.h"

namespace hymoe {

struct GateArgs {
    const float* bias;
    int E, K, score, n_group, topk_group, group_score, norm;
    unsigned mask;  // the key bits that hold the expert: 2^b - 1 >= E - 1
    float scale;
    int* idx;
    float* weights;
    float* scores;
    int* counts;
    const int* slot_of;  // in the block: expert -> placement slot, what idx and the counts then hold
};
struct GateGradArgs {
    const int* idx;
    const float* dw;
    const float* ds;
    int E, K, score, norm;
    float scale;
};


template <typename T>
cudaError_t launch_gate(const hymoe_mat& x, uint32_t n_tok, const GateArgs& a, cudaStream_t st);
template <typename T>
cudaError_t launch_gate_grad(const hymoe_mat& x, const hymoe_mat& d, uint32_t n_tok, const GateGradArgs& a, cudaStream_t st);

constexpr int kGateWarps = 8;  // tokens per CTA
constexpr unsigned kAll = 0xffffffffu;
constexpr float kBig = 3.402823466e38f;

__device__ __forceinline__ float gate_value(float v) { return v; }
__device__ __forceinline__ float gate_value(__half v) { return __half2float(v); }
__device__ __forceinline__ float gate_value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void gate_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void gate_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void gate_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// N consecutive values, 16 bytes at a time (the address is aligned to min(16, N values)).
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec {
    T v[N];
};

// The logit (or bias) as the definition takes it: NaN is -inf (closed), +inf is FLT_MAX.
__device__ __forceinline__ float clean_logit(float z) { return fminf(fmaxf(z, -INFINITY), kBig); }

__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}

template <int EPL, bool RUN>
__device__ __forceinline__ int expert_at(int lane, int i) {
    return RUN ? lane * EPL + i : lane + 32 * i;
}

// A token's logits as they are in memory, and cleaned.
template <typename T, int EPL, bool RUN>
__device__ __forceinline__ void fetch_row(const T* row, int E, Vec<T, EPL>& v) {
    const int lane = threadIdx.x & 31;
    if constexpr (RUN) {
        v = *reinterpret_cast<const Vec<T, EPL>*>(row + lane * EPL);
    } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (lane + 32 * i < E) v.v[i] = row[lane + 32 * i];
            else gate_store(&v.v[i], -INFINITY);
    }
}
template <typename T, int EPL>
__device__ __forceinline__ void clean_row(const Vec<T, EPL>& v, float (&z)[EPL]) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) z[i] = clean_logit(gate_value(v.v[i]));
}

template <typename T, int EPL, bool RUN>
__device__ __forceinline__ void store_row(T* row, int E, const float (&v)[EPL]) {
    const int lane = threadIdx.x & 31;
    if constexpr (RUN) {
        Vec<T, EPL> o;
#pragma unroll
        for (int i = 0; i < EPL; ++i) gate_store(&o.v[i], v[i]);
        *reinterpret_cast<Vec<T, EPL>*>(row + lane * EPL) = o;
    } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (lane + 32 * i < E) gate_store(row + lane + 32 * i, v[i]);
    }
}

// Best (value, index) of the warp: the larger value, the lower index where they tie.
__device__ __forceinline__ void warp_best(double& v, int& e) {
#pragma unroll 1
    for (int o = 16; o; o >>= 1) {
        const double ov = __shfl_xor_sync(kAll, v, o);
        const int oe = __shfl_xor_sync(kAll, e, o);
        if (ov > v || (ov == v && oe < e)) {
            v = ov;
            e = oe;
        }
    }
}

// 2^x and 1 / x in one instruction each (PTX bounds: 2^-22 and 1 ulp, relative).
__device__ __forceinline__ float quick_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float quick_rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float quick_sigmoid(float z) { return quick_rcp(1.f + quick_exp2(z * -1.44269504f)); }

// Bits of a float as a whole number of the same order, and back.
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned u = __float_as_uint(v);
    return u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// A closed expert's key is 0, or that of -inf: under this one and so under every open expert's.
constexpr unsigned kOpenKey = 0x00800000u;  // order_key(-FLT_MAX)

// Descending, by Batcher's odd-even merge sort: every index is known at compile time.
template <int A, int B, int N>
__device__ __forceinline__ void order_pair(unsigned (&k)[N]) {
    const unsigned hi = max(k[A], k[B]), lo = min(k[A], k[B]);
    k[A] = hi;
    k[B] = lo;
}
template <int I, int END, int STEP, int N>
__device__ __forceinline__ void order_pairs(unsigned (&k)[N]) {
    if constexpr (I + STEP < END) {
        order_pair<I, I + STEP>(k);
        order_pairs<I + 2 * STEP, END, STEP>(k);
    }
}
template <int LO, int CNT, int STEP, int N>
__device__ __forceinline__ void merge_keys(unsigned (&k)[N]) {
    if constexpr (2 * STEP < CNT) {
        merge_keys<LO, CNT, 2 * STEP>(k);
        merge_keys<LO + STEP, CNT, 2 * STEP>(k);
        order_pairs<LO + STEP, LO + CNT, STEP>(k);
    } else {
        order_pair<LO, LO + STEP>(k);
    }
}
template <int LO, int CNT, int N>
__device__ __forceinline__ void sort_run(unsigned (&k)[N]) {
    if constexpr (CNT > 1) {
        sort_run<LO, CNT / 2>(k);
        sort_run<LO + CNT / 2, CNT / 2>(k);
        merge_keys<LO, CNT, 1>(k);
    }
}
template <int N>
__device__ __forceinline__ void sort_keys(unsigned (&k)[N]) {
    sort_run<0, N>(k);
}

// Two largest values of a run of values and of another one's.
__device__ __forceinline__ void two_best(float& b1, float& b2, float o1, float o2) {
    b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
    b1 = fmaxf(b1, o1);
}

// A group's value from its two best: half of their sum (which itself can lie beyond fp32, as with
// experts that a bias of the lowest value masks: still open), its only one by half as well, or its
// best; -inf: closed.  And a bound on its error.  An expert's value is off by less than delta plus
// 2^-23 of itself (above), so half a sum by delta + 2^-23 of half the magnitudes, and its own rounding
// and that of value -+ error by 2^-24 of the same each.  A magnitude belongs to its group alone: one
// masked group does not make the others doubtful.
__device__ __forceinline__ float group_value(bool two, float b1, float b2) {
    return !two ? b1 : b2 > -INFINITY ? 0.5f * b1 + 0.5f * b2 : 0.5f * b1;
}
template <bool SIG>
__device__ __forceinline__ float group_error(bool two, float b1, float b2) {
    constexpr float delta = SIG ? 0x1p-21f : 0x1p-20f;
    const float mag = !two ? fabsf(b1) : b2 > -INFINITY ? 0.5f * fabsf(b1) + 0.5f * fabsf(b2) : 0.5f * fabsf(b1);
    return 1.25f * delta + 0x1p-22f * mag;
}

// Weight of a selected logit z (-inf: none selected in this lane): all lanes of the warp.  m, sum: a
// plain softmax's largest logit and sum.
template <bool SIG>
__device__ __forceinline__ float gate_weight(float z, bool norm, float m, float sum, float scale) {
    const bool any = z > -INFINITY;
    float w = 0.f;
    if (norm) {
        // s_k / sum s, both over e^M: M the largest selected logit (at most 0 for a sigmoid)
        float mm = warp_max(z);
        if (SIG) mm = fminf(mm, 0.f);
        if (any) w = SIG ? expf(fminf(z, 0.f) - mm) * quick_rcp(1.f + expf(-fabsf(z))) : expf(z - mm);
        const float tot = warp_sum(w);
        if (any) w *= quick_rcp(tot);
    } else if (any) {
        w = SIG ? __fdiv_rn(1.f, 1.f + expf(-z)) : expf(z - m) * quick_rcp(sum);
    }
    return w * scale;
}

// Selection of one token in double precision by a warp: lane k returns the k-th expert, or -1.  Rare
// and cold: the loops stay loops, as fetching long straight code took longer than running it (15 us
// against 6 for 256 experts in 8 groups).
template <typename T>
__device__ int select_exact(const T* __restrict__ row, const GateArgs& a) {
    constexpr int kMost = HYMOE_GATE_MAX_EXPERTS / 32;
    const int lane = threadIdx.x & 31, E = a.E, n = (E + 31) / 32;
    const bool sig = a.score == HYMOE_SCORE_SIGMOID, two = a.group_score == HYMOE_GROUP_TOP2;
    double c[kMost], gv[kMost];  // what orders expert lane + 32 i, and what its group counts
    float m = -INFINITY;
#pragma unroll 1
    for (int i = 0; i < n; ++i)
        if (lane + 32 * i < E) m = fmaxf(m, clean_logit(gate_value(row[lane + 32 * i])));
    m = warp_max(m);
    double sum = 0.0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const float z = lane + 32 * i < E ? clean_logit(gate_value(row[lane + 32 * i])) : -INFINITY;
        double s = 0.0;
        if (z > -INFINITY && (a.bias != nullptr || two)) {
            s = exp(sig ? -static_cast<double>(z) : static_cast<double>(z) - m);
            if (sig) s = 1.0 / (1.0 + s);
        }
        sum += s;
        c[i] = z;
        gv[i] = s;
    }
    sum = warp_sum(sum);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int e = lane + 32 * i;
        if (c[i] == -INFINITY) {
            gv[i] = -INFINITY;
            continue;
        }
        const double s = sig ? gv[i] : sum > 0.0 ? gv[i] / sum : 0.0;
        if (a.bias != nullptr) c[i] = s + static_cast<double>(clean_logit(__ldg(a.bias + e)));
        gv[i] = two && a.bias == nullptr ? s : c[i];
    }
    if (a.n_group > 0) {
        const int gs = E / a.n_group;
        double val = -INFINITY;  // lane g: group g's value
#pragma unroll 1
        for (int g = 0; g < a.n_group; ++g) {
            double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll 1
            for (int i = g * gs / 32; i < n && 32 * i < (g + 1) * gs; ++i) {
                const int e = lane + 32 * i;
                if (e < g * gs || e >= (g + 1) * gs) continue;
                b2 = fmax(b2, fmin(b1, gv[i]));
                b1 = fmax(b1, gv[i]);
            }
#pragma unroll 1
            for (int o = 16; o; o >>= 1) {
                const double o1 = __shfl_xor_sync(kAll, b1, o), o2 = __shfl_xor_sync(kAll, b2, o);
                b2 = fmax(fmin(b1, o1), fmax(b2, o2));
                b1 = fmax(b1, o1);
            }
            if (lane == g) val = two && b2 > -INFINITY ? b1 + b2 : b1;
        }
        int better = 0;
#pragma unroll 1
        for (int g = 0; g < a.n_group; ++g) {
            const double v = __shfl_sync(kAll, val, g);
            better += v > val || (v == val && g < lane);
        }
        const unsigned kept = __ballot_sync(kAll, lane < a.n_group && val > -INFINITY && better < a.topk_group);
#pragma unroll 1
        for (int i = 0; i < n; ++i)
            if (lane + 32 * i < E && !(kept >> ((lane + 32 * i) / gs) & 1u)) c[i] = -INFINITY;
    }
    int sel = -1;
#pragma unroll 1
    for (int k = 0; k < a.K; ++k) {
        double v = -INFINITY;
        int e = 1 << 20;
#pragma unroll 1
        for (int i = 0; i < n; ++i)
            if (c[i] > v) {
                v = c[i];
                e = lane + 32 * i;
            }
        warp_best(v, e);
        if (v == -INFINITY) break;
        if ((e & 31) == lane) c[e >> 5] = -INFINITY;
        if (lane == k) sel = e;
    }
    return sel;
}

// Lane k's selection of token t to memory; cnt: the CTA's counters, or nullptr.
__device__ __forceinline__ void put_choice(const GateArgs& a, size_t t, int sel, float w, int* cnt) {
    const int lane = threadIdx.x & 31;
    if (lane >= a.K) return;
    if (a.slot_of != nullptr && sel >= 0) sel = __ldg(a.slot_of + sel);
    a.idx[t * a.K + lane] = sel;
    a.weights[t * a.K + lane] = w;
    if (cnt != nullptr && sel >= 0) atomicAdd(cnt + sel, 1);
}

// Lane k's weight for its selection and both to memory.
template <typename T>
__device__ void finish_choice(const T* __restrict__ row, size_t t, const GateArgs& a, int sel, int* cnt) {
    const int lane = threadIdx.x & 31;
    const float z = sel >= 0 ? clean_logit(gate_value(row[sel])) : -INFINITY;
    if (a.score == HYMOE_SCORE_SIGMOID) {
        put_choice(a, t, sel, gate_weight<true>(z, a.norm, 0.f, 0.f, a.scale), cnt);
        return;
    }
    float m = -INFINITY, sum = 0.f;
    if (!a.norm) {
#pragma unroll 1
        for (int e = lane; e < a.E; e += 32) m = fmaxf(m, clean_logit(gate_value(row[e])));
        m = warp_max(m);
        m = m == -INFINITY ? 0.f : m;
#pragma unroll 1
        for (int e = lane; e < a.E; e += 32) sum += expf(clean_logit(gate_value(row[e])) - m);
        sum = warp_sum(sum);
    }
    put_choice(a, t, sel, gate_weight<false>(z, a.norm, m, sum, a.scale), cnt);
}

// A token in double precision where its order could not be proven in fp32: outputs and counts.
template <typename T>
__device__ __noinline__ void route_exact(const T* __restrict__ row, size_t t, const GateArgs& a, int* cnt) {
    finish_choice(row, t, a, select_exact(row, a), cnt);
}

// The order of a few candidates in double precision, by a warp: lane j < K + 1 brings candidate j's
// key (0: none); second: the largest key among the experts that are no candidates.  Sigmoid scores
// with a bias, or logits.  Lane k returns the k-th expert, or -1; -2 in every lane where an expert
// that is no candidate may come in.
template <typename T>
__device__ __forceinline__ int settle(const T* __restrict__ row, const GateArgs& a, unsigned cand, unsigned second) {
    const int lane = threadIdx.x & 31;
    const bool have = cand >= kOpenKey;
    int e = have ? static_cast<int>(a.mask - (cand & a.mask)) : (1 << 20) + lane;
    double d = -INFINITY;
    if (have) {
        d = clean_logit(gate_value(row[e]));
        if (a.bias != nullptr) d = 1.0 / (1.0 + exp(-d)) + static_cast<double>(clean_logit(__ldg(a.bias + e)));
    }
    int rank = 0, from = 0;
#pragma unroll 1
    for (int j = 0; j <= a.K; ++j) {
        const double dj = __shfl_sync(kAll, d, j);
        const int ej = __shfl_sync(kAll, e, j);
        rank += dj > d || (dj == d && ej < e);
    }
#pragma unroll 1
    for (int j = 0; j <= a.K; ++j)
        if (__shfl_sync(kAll, rank, j) == lane) from = j;
    e = __shfl_sync(kAll, e, from);
    d = __shfl_sync(kAll, d, from);
    const double last = __shfl_sync(kAll, d, a.K - 1), most = key_value(second | a.mask);
    const double slack = a.bias != nullptr ? 0x1p-20 + 0x1p-22 * fabs(last) : 0.0;
    if (second >= kOpenKey && !(last - most > slack)) return -2;
    return lane < a.K && e < (1 << 20) ? e : -1;
}

// One token: lane k gets its k-th expert (-1: none left) and weight; false where the selection has
// to be made again in double precision (then nothing but the scores is valid).  VALUED: the scores
// are needed (a bias, scores wanted, or groups by two values); else the logits order the experts.
// bias: this lane's cleaned biases (0 without).  grow: this warp's E floats of shared memory (groups
// with spread experts only).
template <typename T, int EPL, bool RUN, bool SIG, bool VALUED>
__device__ __forceinline__ bool route_token(const T* row, const Vec<T, EPL>& raw, float* scores, const GateArgs& a,
                                            const float (&bias)[EPL], float* grow, int& sel_out, float& w_out) {
    const int lane = threadIdx.x & 31, E = a.E, K = a.K;
    const bool biased = VALUED && a.bias != nullptr;
    float c[EPL];  // the value that orders the experts; -inf: closed
    clean_row(raw, c);
    float m = 0.f, sum = 0.f;  // softmax: the largest open logit and the sum over it
    if (!SIG && (VALUED || !a.norm)) {
        m = c[0];
#pragma unroll
        for (int i = 1; i < EPL; ++i) m = fmaxf(m, c[i]);
        m = warp_max(m);
        m = m == -INFINITY ? 0.f : m;
    }
    constexpr float delta = SIG ? 0x1p-21f : 0x1p-20f;  // error of a score
    bool unsure = false;                                // the same in every lane
    float b1 = -INFINITY, b2 = -INFINITY;               // this lane's two best
    const bool two = VALUED && a.group_score == HYMOE_GROUP_TOP2;
    if constexpr (VALUED) {
        float s[EPL];
        if (SIG) {
            if (scores != nullptr) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) s[i] = __fdiv_rn(1.f, 1.f + expf(-c[i]));
            } else {
#pragma unroll
                for (int i = 0; i < EPL; ++i) s[i] = quick_sigmoid(c[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                s[i] = expf(c[i] - m);
                sum += s[i];
            }
            sum = warp_sum(sum);
            const float inv = sum > 0.f ? __frcp_rn(sum) : 0.f;
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] *= inv;
        }
        if (scores != nullptr) store_row<float, EPL, RUN>(scores, E, s);
        if (biased) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) c[i] = c[i] == -INFINITY ? -INFINITY : s[i] + bias[i];
        } else if (two) {  // the groups are valued by scores, the experts ordered by logits
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const float v = c[i] == -INFINITY ? -INFINITY : s[i];
                if (RUN) {
                    b2 = fmaxf(b2, fminf(b1, v));
                    b1 = fmaxf(b1, v);
                } else if (a.n_group > 0 && lane + 32 * i < E) {
                    grow[lane + 32 * i] = v;
                }
            }
        }
    } else if (!SIG && !a.norm) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) sum += expf(c[i] - m);
        sum = warp_sum(sum);
    }
    if (a.n_group > 0) {
        float val;  // RUN: the value of this lane's group; else lane g holds group g's
        const int gs = E / a.n_group, lanes = RUN ? 32 / a.n_group : 1, mine = lane / lanes;
        if constexpr (RUN) {
            if (biased || !two) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) {
                    b2 = fmaxf(b2, fminf(b1, c[i]));
                    b1 = fmaxf(b1, c[i]);
                }
            }
            for (int o = 1; o < lanes; o <<= 1)
                two_best(b1, b2, __shfl_xor_sync(kAll, b1, o), __shfl_xor_sync(kAll, b2, o));
        } else {
            if (biased || !two) {
#pragma unroll
                for (int i = 0; i < EPL; ++i)
                    if (lane + 32 * i < E) grow[lane + 32 * i] = c[i];
            }
            __syncwarp();
            if (lane < a.n_group)
                for (int j = 0; j < gs; ++j) {
                    const float v = grow[lane * gs + j];
                    b2 = fmaxf(b2, fminf(b1, v));
                    b1 = fmaxf(b1, v);
                }
            __syncwarp();
        }
        val = group_value(two, b1, b2);
        const bool is_group = RUN || lane < a.n_group;
        int better = 0;
        for (int g = 0; g < a.n_group; ++g) {
            const float v = __shfl_sync(kAll, val, g * lanes);
            better += v > val || (v == val && g < mine);
        }
        const bool open = is_group && val > -INFINITY, keep = open && better < a.topk_group;
        if (biased || two) {
            const float err = group_error<SIG>(two, b1, b2);
            const float lowest = -warp_max(keep ? err - val : -INFINITY);
            const float first_out = warp_max(open && !keep ? val + err : -INFINITY);
            unsure = first_out > -INFINITY && !(lowest > first_out);
        }
        if constexpr (RUN) {
            if (!keep) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) c[i] = -INFINITY;
            }
        } else {
            const unsigned kept = __ballot_sync(kAll, keep);
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (lane + 32 * i < E && !(kept >> ((lane + 32 * i) / gs) & 1u)) c[i] = -INFINITY;
        }
    }
    unsigned key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const unsigned k = order_key(VALUED && biased ? c[i] : c[i] + 0.f);  // -0 is 0
        key[i] = c[i] == -INFINITY ? 0u : (k & ~a.mask) | (a.mask - expert_at<EPL, RUN>(lane, i));
    }
    sort_keys(key);
    unsigned chosen = 0;  // lane k: the k-th key
    for (int k = 0; k < K; ++k) {
        const unsigned v = __reduce_max_sync(kAll, key[0]);
        if (lane == k) chosen = v;
        const bool pop = key[0] == v;  // (a lane without experts shifts zeros)
#pragma unroll
        for (int i = 0; i + 1 < EPL; ++i) key[i] = pop ? key[i + 1] : key[i];
        key[EPL - 1] = pop ? 0u : key[EPL - 1];
    }
    int sel = chosen != 0 ? static_cast<int>(a.mask - (chosen & a.mask)) : -1;
    float z = -INFINITY;
    if (biased || sizeof(T) == 4) {
        if (sel >= 0) z = clean_logit(gate_value(row[sel]));
        // every selected key against the one after it (the last against the best one left), first as
        // the least and the largest value they can stand for: nearly every token ends there
        const int last = __popc(__ballot_sync(kAll, sel >= 0)) - 1;
        const unsigned best_left = __reduce_max_sync(kAll, key[0]);
        unsigned after = __shfl_down_sync(kAll, chosen, 1);
        if (lane == last) after = best_left;
        const float lo = key_value(chosen & ~a.mask), hi = key_value(after | a.mask);
        const float slack = biased ? 2.f * delta + 0x1p-22f * fabsf(lo) : 0.f;
        if (__any_sync(kAll, lane <= last && after != 0 && !(lo - hi > slack))) {
            // the best one left by its own value, the next by the most that its key can stand for
            unsigned second = 0;
            float zl = -INFINITY, bl = 0.f;
            if (best_left != 0) {
                second = __reduce_max_sync(kAll, key[0] == best_left ? key[1] : key[0]);
                const int el = static_cast<int>(a.mask - (best_left & a.mask));
                zl = clean_logit(gate_value(row[el]));
                if (biased) bl = clean_logit(__ldg(a.bias + el));
            }
            const float pz = __shfl_up_sync(kAll, z, 1);
            bool bad = false;
            if (biased) {
                const auto value = [&](float zz) { return SIG ? quick_sigmoid(zz) : sum > 0.f ? expf(zz - m) * quick_rcp(sum) : 0.f; };
                const float b = sel >= 0 ? clean_logit(__ldg(a.bias + sel)) : 0.f, v = value(z) + b;
                const float pv = __shfl_up_sync(kAll, v, 1), pb = __shfl_up_sync(kAll, b, 1);
                if (lane > 0 && lane <= last)
                    bad = !(pv - v > 2.f * delta + 0x1p-22f * fabsf(pv)) && !(pz == z && pb == b);
                if (lane == last && best_left != 0) {
                    const float least = 2.f * delta + 0x1p-22f * fabsf(v);
                    bad = bad || (!(v - (value(zl) + bl) > least) && !(z == zl && b == bl));
                    bad = bad || (second != 0 && !(v - key_value(second | a.mask) > least));
                }
            } else {
                bad = (lane > 0 && lane <= last && pz < z) ||
                      (lane == last && best_left != 0 && (z < zl || ((chosen ^ second) & ~a.mask) == 0));
            }
            if (__any_sync(kAll, bad)) {
                int e = -2;
                if ((SIG || !biased) && K < 32)
                    e = settle(row, a, lane < K ? chosen : lane == K ? best_left : 0u, second);
                unsure = unsure || __any_sync(kAll, e == -2);
                sel = e;
                z = sel >= 0 ? clean_logit(gate_value(row[sel])) : -INFINITY;
            }
        }
    } else if (sel >= 0) {  // the key is the logit: its replaced bits were those of a 16-bit value
        z = fminf(key_value(chosen & 0x80000000u ? chosen & ~a.mask : chosen | a.mask), kBig);
        if (z >= 3.38953138e38f) z = clean_logit(gate_value(row[sel]));  // +inf became FLT_MAX
    }
    sel_out = sel;
    w_out = gate_weight<SIG>(z, a.norm, m, sum, a.scale);
    return !unsure;
}

template <int EPL, bool RUN>
__device__ __forceinline__ void load_bias(const GateArgs& a, float (&bias)[EPL]) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = expert_at<EPL, RUN>(threadIdx.x & 31, i);
        bias[i] = a.bias != nullptr && e < a.E ? clean_logit(__ldg(a.bias + e)) : 0.f;
    }
}

template <typename T, int EPL, bool RUN, bool SIG, bool VALUED>
__global__ __launch_bounds__(32 * kGateWarps, EPL <= 2 ? 6 : EPL == 4 ? 5 : EPL == 8 ? 4 : 2) void gate_kernel(
    const T* __restrict__ logits, size_t ld, uint32_t n_tok, const __grid_constant__ GateArgs a) {
    extern __shared__ float gbuf[];  // groups with spread experts only: [kGateWarps][E]
    __shared__ int cnt[HYMOE_GATE_MAX_EXPERTS];
    const int warp = threadIdx.x >> 5;
    if (a.counts != nullptr) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) cnt[e] = 0;
        __syncthreads();
    }
    float bias[EPL];
    if (VALUED) load_bias<EPL, RUN>(a, bias);
    const size_t step = static_cast<size_t>(gridDim.x) * kGateWarps;
    size_t t = static_cast<size_t>(blockIdx.x) * kGateWarps + warp;
    while (t < n_tok) {
        const size_t first = t;
        unsigned again = 0;  // tokens of these 32 that need double precision
        for (int i = 0; i < 32 && t < n_tok; ++i, t += step) {
            Vec<T, EPL> raw;
            fetch_row<T, EPL, RUN>(logits + t * ld, a.E, raw);
            int sel;
            float w;
            if (!route_token<T, EPL, RUN, SIG, VALUED>(logits + t * ld, raw, VALUED && a.scores != nullptr ? a.scores + t * a.E : nullptr,
                                                       a, bias, gbuf + static_cast<size_t>(warp) * a.E, sel, w)) {
                again |= 1u << i;
            } else {
                put_choice(a, t, sel, w, a.counts != nullptr ? cnt : nullptr);
            }
        }
        for (; again != 0; again &= again - 1) {
            const size_t u = first + static_cast<size_t>(__ffs(again) - 1) * step;
            route_exact<T>(logits + u * ld, u, a, a.counts != nullptr ? cnt : nullptr);
        }
    }
    if (a.counts != nullptr) {
        __syncthreads();
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
            if (gridDim.x == 1) a.counts[e] = cnt[e];
            else if (cnt[e]) atomicAdd(a.counts + e, cnt[e]);  // whole numbers: any order gives the same
        }
    }
}

// ---- a token per thread
//
// For many tokens, without scores to write: a thread takes its token's experts eight at a time, sorts
// their keys and merges them into the eight best so far (two sorting networks: some 11 operations per
// expert, where a warp per token pays a reduction and a shift per choice for one token alone).  Keys,
// certificates and weights are those of route_token; a thread's sums are its own.  A token that
// cannot be proven is left to its warp at the end.
constexpr int kRowsTopk = 8;

// The eight best of l (descending) and of eight keys (descending); rest: the largest key left out.
__device__ __forceinline__ void merge_best(unsigned (&l)[8], const unsigned (&k)[8], unsigned& rest) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rest = max(rest, min(l[i], k[7 - i]));
        l[i] = max(l[i], k[7 - i]);
    }
#pragma unroll
    for (int d = 4; d; d >>= 1)  // what is left rises and falls: halves compared, quarters, pairs
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((i & d) == 0) {
                const unsigned hi = max(l[i], l[i + d]), lo = min(l[i], l[i + d]);
                l[i] = hi;
                l[i + d] = lo;
            }
}

// Eight values that order the experts (or their groups): s + b, scores or logits; -inf: closed.
template <typename T, bool BIASED>
__device__ __forceinline__ void eight_values(const Vec<T, 8>& raw, const float* bias, bool scored, float (&v)[8]) {
    Vec<float, 8> b;
    if (BIASED) b = *reinterpret_cast<const Vec<float, 8>*>(bias);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float z = BIASED ? fmaxf(gate_value(raw.v[i]), -INFINITY) : clean_logit(gate_value(raw.v[i]));
        v[i] = z;
        if (BIASED) v[i] = z == -INFINITY ? z : quick_sigmoid(z) + b.v[i];
        else if (scored) v[i] = z == -INFINITY ? z : quick_sigmoid(z);
    }
}

template <typename T, bool BIASED, bool GROUPS>
__global__ __launch_bounds__(128, 8) void gate_rows_kernel(const T* __restrict__ logits, size_t ld, uint32_t n_tok,
                                                        const __grid_constant__ GateArgs a) {
    extern __shared__ __align__(16) float rbuf[];  // [E] biases, [n_group][threads] values and, with biases, errors
    __shared__ int cnt[HYMOE_GATE_MAX_EXPERTS];
    const int tid = threadIdx.x, E = a.E, K = a.K;
    for (int e = tid; e < E; e += blockDim.x) {
        cnt[e] = 0;
        if (BIASED) rbuf[e] = clean_logit(__ldg(a.bias + e));
    }
    __syncthreads();
    const size_t t = static_cast<size_t>(blockIdx.x) * blockDim.x + tid;
    const bool live = t < n_tok, sig = a.score == HYMOE_SCORE_SIGMOID;
    const T* row = logits + (live ? t : n_tok - 1) * ld;
    const auto eight = [&](int e) { return *reinterpret_cast<const Vec<T, 8>*>(row + e); };
    constexpr float delta = 0x1p-21f;
    bool unsure_groups = false;

    unsigned kept = kAll;
    if constexpr (GROUPS) {
        const bool two = a.group_score == HYMOE_GROUP_TOP2;
        const int gs = E / a.n_group;
        // with a bias a group's error too, by its magnitude; scores alone are at most 1
        float* gv = rbuf + (BIASED ? E : 0) + tid;
        // (rounded up to 16 bits: floats kept blocks off an SM at 32 groups, 156 us instead of 151)
        __nv_bfloat16* ge = reinterpret_cast<__nv_bfloat16*>(rbuf + (BIASED ? E : 0) + a.n_group * blockDim.x) + tid;
        for (int g = 0; g < a.n_group; ++g) {
            float b1 = -INFINITY, b2 = -INFINITY;
            for (int e = g * gs; e < (g + 1) * gs; e += 8) {
                float v[8];
                eight_values<T, BIASED>(eight(e), rbuf + e, two, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    b2 = fmaxf(b2, fminf(b1, v[i]));
                    b1 = fmaxf(b1, v[i]);
                }
            }
            gv[g * blockDim.x] = group_value(two, b1, b2);
            if (BIASED) ge[g * blockDim.x] = __float2bfloat16_ru(group_error<true>(two, b1, b2));
        }
        kept = 0;
        float lowest = INFINITY, first_out = -INFINITY;
        for (int g = 0; g < a.n_group; ++g) {
            const float v = gv[g * blockDim.x], err = BIASED ? __bfloat162float(ge[g * blockDim.x]) : group_error<true>(two, 1.f, 1.f);
            int better = 0;
            for (int h = 0; h < a.n_group; ++h) {
                const float o = gv[h * blockDim.x];
                better += o > v || (o == v && h < g);
            }
            if (v > -INFINITY && better < a.topk_group) {
                kept |= 1u << g;
                lowest = fminf(lowest, v - err);
            } else if (v > -INFINITY) {
                first_out = fmaxf(first_out, v + err);
            }
        }
        if (BIASED || two) unsure_groups = first_out > -INFINITY && !(lowest > first_out);
    }

    unsigned l[8], rest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) l[i] = 0;
    {
        const int gs = GROUPS ? E / a.n_group : E;
        Vec<T, 8> next = eight(0);
        for (int e0 = 0, g = 0; e0 < E; e0 += gs, ++g) {
            const bool keep = !GROUPS || (kept >> g & 1u);
            for (int e = e0; e < e0 + gs; e += 8) {
                const Vec<T, 8> raw = next;
                if (e + 8 < E) next = eight(e + 8);
                float v[8];
                eight_values<T, BIASED>(raw, rbuf + e, false, v);
                unsigned key[8];
                const unsigned id = a.mask - e;  // its lowest three bits are set
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    key[i] = (order_key(BIASED ? v[i] : v[i] + 0.f) & ~a.mask) | (id ^ i);  // -0 is 0
                    if (GROUPS && !keep) key[i] = 0;
                }
                sort_keys(key);
                merge_best(l, key, rest);
            }
        }
    }

    float m = 0.f, sum = 0.f;
    if (!BIASED && !sig && !a.norm) {  // a plain softmax: its sum, in trees of 8 and runs of 8 trees
        m = -INFINITY;
        for (int e = 0; e < E; e += 8) {
            float v[8];
            eight_values<T, false>(eight(e), nullptr, false, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, v[i]);
        }
        m = m == -INFINITY ? 0.f : m;
        float part = 0.f;
        for (int e = 0; e < E; e += 8) {
            float v[8];
            eight_values<T, false>(eight(e), nullptr, false, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = expf(v[i] - m);
            part += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            if ((e & 56) == 56 || e + 8 == E) {
                sum += part;
                part = 0.f;
            }
        }
    }

    // the choices' logits, and whether their order is certain
    bool unsure = unsure_groups;
    int sel[8];
    float z[8], w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const bool have = k < K && l[k] >= kOpenKey;
        sel[k] = have ? static_cast<int>(a.mask - (l[k] & a.mask)) : -1;
        z[k] = -INFINITY;
        if (!have) continue;
        if (BIASED || sizeof(T) == 4) {
            z[k] = clean_logit(gate_value(row[sel[k]]));
        } else {  // the key is the logit: its replaced bits were those of a 16-bit value
            z[k] = fminf(key_value(l[k] & 0x80000000u ? l[k] & ~a.mask : l[k] | a.mask), kBig);
            if (z[k] >= 3.38953138e38f) z[k] = clean_logit(gate_value(row[sel[k]]));  // +inf became FLT_MAX
        }
    }
    if (BIASED || sizeof(T) == 4) {
        bool close = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const unsigned after = k < 7 ? l[k < 7 ? k + 1 : 7] : rest;
            const float lo = key_value(l[k] & ~a.mask), hi = key_value(after | a.mask);
            const float slack = BIASED ? 2.f * delta + 0x1p-22f * fabsf(lo) : 0.f;
            close = close || (k < K && after >= kOpenKey && !(lo - hi > slack));
        }
        if (close) {
            float pv = 0.f, pb = 0.f, pz = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (sel[k] < 0) continue;
                const unsigned after = k < 7 ? l[k < 7 ? k + 1 : 7] : rest;
                const bool last = k + 1 == K && after >= kOpenKey;  // the best one left is next
                if (BIASED) {
                    const float b = rbuf[sel[k]], v = quick_sigmoid(z[k]) + b;
                    if (k > 0) unsure = unsure || (!(pv - v > 2.f * delta + 0x1p-22f * fabsf(pv)) && !(pz == z[k] && pb == b));
                    if (last) unsure = unsure || !(v - key_value(after | a.mask) > 2.f * delta + 0x1p-22f * fabsf(v));
                    pv = v;
                    pb = b;
                } else {
                    unsure = unsure || (k > 0 && pz < z[k]) || (last && ((l[k] ^ after) & ~a.mask) == 0);
                }
                pz = z[k];
            }
        }
    }

    if (a.norm) {
        float mm = z[0], tot = 0.f;
#pragma unroll
        for (int k = 1; k < 8; ++k) mm = fmaxf(mm, z[k]);
        if (sig) mm = fminf(mm, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            w[k] = 0.f;
            if (sel[k] >= 0) w[k] = sig ? expf(fminf(z[k], 0.f) - mm) * quick_rcp(1.f + expf(-fabsf(z[k]))) : expf(z[k] - mm);
            tot += w[k];
        }
        const float inv = tot > 0.f ? quick_rcp(tot) * a.scale : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] *= inv;
    } else {
        const float inv = sum > 0.f ? quick_rcp(sum) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            w[k] = 0.f;
            if (sel[k] >= 0) w[k] = (sig ? __fdiv_rn(1.f, 1.f + expf(-z[k])) : expf(z[k] - m) * inv) * a.scale;
        }
    }
    if (live && !unsure) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (k >= K) break;
            a.idx[t * K + k] = sel[k];
            a.weights[t * K + k] = w[k];
            if (a.counts != nullptr && sel[k] >= 0) atomicAdd(cnt + sel[k], 1);
        }
    }
    // tokens in doubt, one after another by the whole warp: whichever groups are kept, the candidates'
    // order is settled among themselves
    int* c = a.counts != nullptr ? cnt : nullptr;
    for (unsigned again = __ballot_sync(kAll, live && unsure); again != 0; again &= again - 1) {
        const int who = __ffs(again) - 1, lane = tid & 31;
        const size_t u = t - lane + who;
        const T* row_u = logits + u * ld;
        unsigned cand = 0, second = __shfl_sync(kAll, rest, who);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned v = __shfl_sync(kAll, l[i], who);
            if (i <= K && lane == i) cand = v;
            if (i == K + 1) second = v;
        }
        if (K == 8) {  // the ninth is the last candidate: look for the tenth
            const unsigned keep = __shfl_sync(kAll, kept, who);
            if (lane == 8) cand = second;
            unsigned most = 0;
#pragma unroll 1
            for (int e = lane; e < E; e += 32) {
                if (GROUPS && !(keep >> (e / (E / a.n_group)) & 1u)) continue;
                const float zz = clean_logit(gate_value(row_u[e]));
                const float v = !BIASED ? zz + 0.f : zz == -INFINITY ? zz : quick_sigmoid(zz) + rbuf[e];
                const unsigned k = (order_key(v) & ~a.mask) | (a.mask - e);
                if (k < second) most = max(most, k);
            }
            second = __reduce_max_sync(kAll, most);
        }
        int e = -2;
        if (!__shfl_sync(kAll, unsure_groups, who)) e = settle(row_u, a, cand, second);
        if (__any_sync(kAll, e == -2)) route_exact<T>(row_u, u, a, c);
        else finish_choice(row_u, u, a, e, c);
    }
    if (a.counts != nullptr) {
        __syncthreads();
        for (int e = tid; e < E; e += blockDim.x)
            if (cnt[e]) atomicAdd(a.counts + e, cnt[e]);  // whole numbers: any order gives the same
    }
}

// dz = (ds/dz)^T (dL/ds), with dL/ds the score gradient plus, at the selected experts,
//   norm: scale (dw_k - sum_j dw_j n_j) n_k / s_k (n = the renormalised weights), else scale dw_k.
// The factor n_k / s_k is never formed: it meets s_k (1 - s_k) or s_k in the product.  SPARSE (no
// score gradient, and not a softmax's plain scores): only the selected logits are read, every other
// gradient is 0; renormalised softmax weights do not depend on the other logits at all.
template <typename T, int EPL, bool RUN, bool SPARSE>
__global__ __launch_bounds__(32 * kGateWarps) void gate_grad_kernel(const T* logits, size_t ld, T* d_logits,
                                                                    size_t ldd, uint32_t n_tok, GateGradArgs a) {
    extern __shared__ float gbuf[];  // [kGateWarps][32 * EPL]: the selected experts' terms
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int E = a.E, K = a.K;
    const bool sig = a.score == HYMOE_SCORE_SIGMOID;
    float* row = gbuf + warp * (32 * EPL);
    const size_t step = static_cast<size_t>(gridDim.x) * kGateWarps;
    size_t t = static_cast<size_t>(blockIdx.x) * kGateWarps + warp;
    // the selections are fetched two tokens ahead, their logits one token ahead
    int sel_next = lane < K && t < n_tok ? a.idx[t * K + lane] : -1;
    int sel_2nd = lane < K && t + step < n_tok ? a.idx[(t + step) * K + lane] : -1;
    float dw_next = sel_next >= 0 && sel_next < E ? a.dw[t * K + lane] : 0.f;
    float z_next = sel_next >= 0 && sel_next < E ? clean_logit(gate_value(logits[t * ld + sel_next])) : -INFINITY;
    for (; t < n_tok; t += step) {
        int sel = sel_next;
        const float z = z_next;
        if (z == -INFINITY) sel = -1;
        const float dw = sel >= 0 ? dw_next * a.scale : 0.f;
        sel_next = sel_2nd;
        sel_2nd = lane < K && t + 2 * step < n_tok ? a.idx[(t + 2 * step) * K + lane] : -1;
        const bool ok = sel_next >= 0 && sel_next < E;
        dw_next = ok ? a.dw[(t + step) * K + lane] : 0.f;
        z_next = ok ? clean_logit(gate_value(logits[(t + step) * ld + sel_next])) : -INFINITY;
        float v[EPL], s[EPL], m = 0.f, sum = 0.f;
        if constexpr (!SPARSE) {
            Vec<T, EPL> raw;
            fetch_row<T, EPL, RUN>(logits + t * ld, E, raw);
            clean_row(raw, v);
            if (sig) {
#pragma unroll
                for (int i = 0; i < EPL; ++i) s[i] = __fdiv_rn(1.f, 1.f + expf(-v[i]));
            } else {
                m = v[0];
#pragma unroll
                for (int i = 1; i < EPL; ++i) m = fmaxf(m, v[i]);
                m = warp_max(m);
                m = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int i = 0; i < EPL; ++i) {
                    s[i] = expf(v[i] - m);
                    sum += s[i];
                }
                sum = warp_sum(sum);
#pragma unroll
                for (int i = 0; i < EPL; ++i) s[i] = sum > 0.f ? __fdiv_rn(s[i], sum) : 0.f;
            }
        }
        float term;  // lane k: (dL/ds_k) s_k
        if (a.norm) {
            float mm = warp_max(z), n = 0.f;
            if (sig) mm = fminf(mm, 0.f);
            if (sel >= 0) n = sig ? __fdividef(expf(fminf(z, 0.f) - mm), 1.f + expf(-fabsf(z))) : expf(z - mm);
            const float tot = warp_sum(n);
            n = sel >= 0 ? __fdividef(n, tot) : 0.f;
            term = n * (dw - warp_sum(dw * n));
        } else {
            term = sel < 0 ? 0.f : dw * (sig ? __fdividef(1.f, 1.f + expf(-z)) : __fdividef(expf(z - m), sum));
        }
        if (SPARSE && sig && sel >= 0) term *= __fdividef(1.f, 1.f + expf(z));  // 1 - s without the cancellation
        // the terms to their experts' places; an expert named more than once gets their sum in order
        __syncwarp();
#pragma unroll
        for (int i = 0; i < EPL; ++i) row[lane + 32 * i] = 0.f;
        __syncwarp();
        const unsigned same = __match_any_sync(kAll, sel);
        if (!__any_sync(kAll, sel >= 0 && (same & (same - 1)))) {
            if (sel >= 0) row[sel] = term;
        } else {
            for (int k = 0; k < K; ++k) {
                if (lane == k && sel >= 0) row[sel] += term;
                __syncwarp();
            }
        }
        __syncwarp();
        float d[EPL];
        if constexpr (SPARSE) {
#pragma unroll
            for (int i = 0; i < EPL; ++i) d[i] = row[expert_at<EPL, RUN>(lane, i)];
        } else {
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                const int e = expert_at<EPL, RUN>(lane, i);
                d[i] = row[e];
                if (a.ds != nullptr && e < E && v[i] != -INFINITY) d[i] += a.ds[t * E + e] * s[i];
                dot += d[i];
            }
            if (!sig) dot = warp_sum(dot);
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                if (sig) d[i] *= __fdiv_rn(1.f, 1.f + expf(v[i]));
                else d[i] -= s[i] * dot;
                if (v[i] == -INFINITY) d[i] = 0.f;
            }
        }
        store_row<T, EPL, RUN>(d_logits + t * ldd, E, d);
    }
}

// Whether rows of E values of `es` bytes, `ld` apart, can be read as a run of vectors per lane.
inline bool row_runs(const void* p, size_t ld, size_t es, int E) {
    if (E < 64 || E > 512 || (E & (E - 1))) return false;
    const size_t lane_bytes = E / 32 * es, unit = lane_bytes < 16 ? lane_bytes : 16;
    return entry_aligned(p, unit) && ld * es % unit == 0;
}

inline int gate_grid(size_t n_tok) {  // (one wave of what fits was 4 to 15% slower)
    const size_t chunks = (n_tok + kGateWarps - 1) / kGateWarps;
    return static_cast<int>(chunks < 148 * 8 ? chunks : 148 * 8);
}

template <typename T, int EPL, bool RUN>
cudaError_t launch_gate_epl(const T* x, size_t ld, uint32_t n_tok, const GateArgs& a, cudaStream_t st) {
    const size_t smem = a.n_group > 0 && !RUN ? sizeof(float) * kGateWarps * a.E : 0;
    const int grid = gate_grid(n_tok), block = 32 * kGateWarps;
    const bool valued = a.bias || a.scores || (a.n_group > 0 && a.group_score == HYMOE_GROUP_TOP2);
    if (a.score == HYMOE_SCORE_SIGMOID) {
        if (valued) gate_kernel<T, EPL, RUN, true, true><<<grid, block, smem, st>>>(x, ld, n_tok, a);
        else gate_kernel<T, EPL, RUN, true, false><<<grid, block, smem, st>>>(x, ld, n_tok, a);
    } else {
        if (valued) gate_kernel<T, EPL, RUN, false, true><<<grid, block, smem, st>>>(x, ld, n_tok, a);
        else gate_kernel<T, EPL, RUN, false, false><<<grid, block, smem, st>>>(x, ld, n_tok, a);
    }
    return cudaGetLastError();
}
template <typename T, int EPL, bool RUN>
cudaError_t launch_grad_epl(const T* x, size_t ld, T* d, size_t ldd, uint32_t n_tok, const GateGradArgs& a, cudaStream_t st) {
    const int grid = gate_grid(n_tok), block = 32 * kGateWarps;
    const size_t smem = sizeof(float) * kGateWarps * 32 * EPL;
    if (a.ds == nullptr && (a.norm || a.score == HYMOE_SCORE_SIGMOID))
        gate_grad_kernel<T, EPL, RUN, true><<<grid, block, smem, st>>>(x, ld, d, ldd, n_tok, a);
    else
        gate_grad_kernel<T, EPL, RUN, false><<<grid, block, smem, st>>>(x, ld, d, ldd, n_tok, a);
    return cudaGetLastError();
}

// Whether a thread per token takes the call: pieces of eight experts on 16-byte boundaries, at most
// eight choices, nothing to sum over the experts for their order, and tokens enough to fill the GPU
// with threads.  By warps against by threads, us, bf16: 128 experts, 6 choices, bias: 6.8 / 10.9 at
// 8192 tokens, 10.8 / 9.6 at 16384, 60.6 / 27.7 at 131072; 64 experts, 8 choices: 4.2 / 4.9, 6.5 / 5.5,
// 37.8 / 16.6; 512 experts, 8 choices: 9.0 / 16.2, 15.8 / 17.0, 114 / 81.  Groups cost a second pass
// (256 experts, 8 groups): 44.9 / 46.4 at 32768, 136 / 88 at 131072.
constexpr uint32_t kGateRowsMin = 16384, kGateRowsMinGroups = 65536;
inline bool gate_by_rows(const hymoe_mat& x, size_t es, uint32_t n_tok, const GateArgs& a) {
    const bool sig = a.score == HYMOE_SCORE_SIGMOID, two = a.n_group > 0 && a.group_score == HYMOE_GROUP_TOP2;
    return n_tok >= (a.n_group > 0 ? kGateRowsMinGroups : kGateRowsMin) && a.K <= kRowsTopk && a.E % 8 == 0 && entry_aligned(x.data, 16) &&
           static_cast<size_t>(x.ld) * es % 16 == 0 && a.scores == nullptr && (sig || (a.bias == nullptr && !two)) &&
           (a.n_group == 0 || a.E / a.n_group % 8 == 0);
}
template <typename T>
cudaError_t launch_gate_rows(const T* x, size_t ld, uint32_t n_tok, const GateArgs& a, cudaStream_t st) {
    const int block = n_tok < 148u * 512u ? 32 : 128;
    const size_t smem = sizeof(float) * (a.bias ? a.E : 0) + static_cast<size_t>(a.n_group) * block * (sizeof(float) + (a.bias ? sizeof(__nv_bfloat16) : 0));
    const unsigned grid = static_cast<unsigned>((static_cast<size_t>(n_tok) + block - 1) / block);
    if (a.bias && a.n_group) gate_rows_kernel<T, true, true><<<grid, block, smem, st>>>(x, ld, n_tok, a);
    else if (a.bias) gate_rows_kernel<T, true, false><<<grid, block, smem, st>>>(x, ld, n_tok, a);
    else if (a.n_group) gate_rows_kernel<T, false, true><<<grid, block, smem, st>>>(x, ld, n_tok, a);
    else gate_rows_kernel<T, false, false><<<grid, block, smem, st>>>(x, ld, n_tok, a);
    return cudaGetLastError();
}

// EPL: the smallest of 2, 4, 8, 16 that holds the experts; runs where the rows allow it.
template <typename T>
cudaError_t launch_gate(const hymoe_mat& x, uint32_t n_tok, const GateArgs& a, cudaStream_t st) {
    const bool run = row_runs(x.data, static_cast<size_t>(x.ld), sizeof(T), a.E) &&
                     (a.scores == nullptr || row_runs(a.scores, a.E, sizeof(float), a.E)) &&
                     (a.n_group == 0 || 32 % a.n_group == 0);
    const T* p = static_cast<const T*>(x.data);
    const size_t ld = static_cast<size_t>(x.ld);
    if (gate_by_rows(x, sizeof(T), n_tok, a)) return launch_gate_rows<T>(p, ld, n_tok, a, st);
    auto go = [&](auto kern_run, auto kern_spread) { return run ? kern_run(p, ld, n_tok, a, st) : kern_spread(p, ld, n_tok, a, st); };
    if (a.E <= 64) return go(launch_gate_epl<T, 2, true>, launch_gate_epl<T, 2, false>);
    if (a.E <= 128) return go(launch_gate_epl<T, 4, true>, launch_gate_epl<T, 4, false>);
    if (a.E <= 256) return go(launch_gate_epl<T, 8, true>, launch_gate_epl<T, 8, false>);
    return go(launch_gate_epl<T, 16, true>, launch_gate_epl<T, 16, false>);
}
template <typename T>
cudaError_t launch_gate_grad(const hymoe_mat& x, const hymoe_mat& d, uint32_t n_tok, const GateGradArgs& a, cudaStream_t st) {
    const bool run = row_runs(x.data, static_cast<size_t>(x.ld), sizeof(T), a.E) &&
                     row_runs(d.data, static_cast<size_t>(d.ld), sizeof(T), a.E);
    const T* p = static_cast<const T*>(x.data);
    T* q = static_cast<T*>(d.data);
    const size_t ld = static_cast<size_t>(x.ld), ldd = static_cast<size_t>(d.ld);
    auto go = [&](auto kern_run, auto kern_spread) {
        return run ? kern_run(p, ld, q, ldd, n_tok, a, st) : kern_spread(p, ld, q, ldd, n_tok, a, st);
    };
    if (a.E <= 64) return go(launch_grad_epl<T, 2, true>, launch_grad_epl<T, 2, false>);
    if (a.E <= 128) return go(launch_grad_epl<T, 4, true>, launch_grad_epl<T, 4, false>);
    if (a.E <= 256) return go(launch_grad_epl<T, 8, true>, launch_grad_epl<T, 8, false>);
    return go(launch_grad_epl<T, 16, true>, launch_grad_epl<T, 16, false>);
}

}  // namespace hymoe
