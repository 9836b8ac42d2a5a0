// adapt_grad_tc.cu — the adapters' gradients on the 5th-generation tensor cores, for long rows of the
// weights' 16-bit type on 16-byte boundaries: for every adapter, the sum over its tokens of the outer
// products of a long row (x or dy) and its narrow counterpart (low).
//
// A CTA takes 256 columns of the long rows and one item of the plan, 64 tokens a stage; both
// gradients' CTAs are one grid.  The tensor core sums over the tokens: D[128 columns, RP] +=
// X^T low, twice.
//   A  the rows as they lie in memory, [64 tokens][64 columns] panels: an MN-major operand; by TMA
//      where a stage's tokens are consecutive, else copied
//   B  low, split into three 16-bit parts and turned to [RP][64 tokens] on the way: K-major
// bf16 parts hold fp32 whole; fp16 ones hold 33 bits below the adapter's largest value, by a power of
// two that the narrow product left behind.  The sums go to several accumulators in turn (the pipe
// truncates what it adds: with four, an eighth of the error of one), which are added at the end.
// A stage that is not whole is copied with its last row repeated, so that nothing of other rows
// meets low's zeros.  Bound by reading the long rows.
#include "adapt_tc.cuh"

namespace hymoe {
namespace {

constexpr int kGtcTok = 64;
constexpr int kGtcCols = 256;                     // columns per CTA: two products of 128
constexpr int kGtcConv = 2;                       // groups of four converting warps, in turn
constexpr int kGtcThreads = 64 + (kGtcConv + 1) * 128;  // TMA, MMA, converting and copying warps
constexpr int kGtcPanel = kGtcTok * 128;          // 64 columns of the stage's rows
constexpr int kGtcX = kGtcCols / 64 * kGtcPanel;
constexpr int kGtcParts = 3;

template <int RP>
struct GtcTile {
    static constexpr int kPart = RP * 128;
    static constexpr int kStage = kGtcX + kGtcParts * kPart;
    static constexpr int kStages = 224 * 1024 / kStage < 4 ? 224 * 1024 / kStage : 4;
    static_assert(kStages % kGtcConv == 0, "a group of converting warps always meets the same stages");
    static constexpr int kSmem = 1024 + kStages * kStage;
    static constexpr int kSet = kGtcCols / 128 * RP;           // accumulator columns of a set
    static constexpr int kSets = 512 / kSet < 4 ? 512 / kSet : 4;
    static constexpr int kTmem = kSet * kSets;
};

template <typename W, int RP>
__global__ __launch_bounds__(kGtcThreads, 1) void grad_tc_kernel(const __grid_constant__ AdaptGradPair pair) {
    using L = GtcTile<RP>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[L::kStages], empty[L::kStages], done;
    __shared__ uint32_t tmem_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool second = static_cast<int>(blockIdx.y) >= pair.groups0;
    const AdaptGrad& a = second ? pair.g[1] : pair.g[0];
    const CUtensorMap* map = second ? &pair.rows[1] : &pair.rows[0];
    const int m0 = (static_cast<int>(blockIdx.y) - (second ? pair.groups0 : 0)) * kGtcCols;
    griddep_wait();
    griddep_launch_dependents();
    if (static_cast<int>(blockIdx.x) >= a.plan.n_lists[2]) return;
    const int4 item = a.plan.items[blockIdx.x];
    const int n_st = (item.z + kGtcTok - 1) / kGtcTok;
    const int* perm = a.plan.perm + item.y;
    // Of stages it .. it + 31, one per lane: the first token, and those that TMA takes (whole, of
    // consecutive tokens); the others are copied.
    const auto look = [&](int it, int* first) {
        const int t = (it + lane) * kGtcTok;
        const bool whole = t + kGtcTok <= item.z;
        *first = whole ? __ldg(perm + t) : 0;
        return __ballot_sync(0xffffffffu, whole && __ldg(perm + min(t, item.z - kGtcTok) + kGtcTok - 1) - *first == kGtcTok - 1);
    };
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full[s], 9);  // TMA's thread, a group of converting warps, four copying warps
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_s, L::kTmem);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    int* err = a.plan.n_lists;
    // fp16 parts: low times 2^shift, its largest value (over the adapter) in [2^14, 2^15)
    float scale = 1.f, unscale = 1.f;
    if (AdType<W>::kScaled) {
        const int e = max(16, min(239, static_cast<int>(a.plan.amax[(second ? a.n : 0) + item.x] >> 23)));
        scale = __uint_as_float(static_cast<uint32_t>(254 + 14 - e) << 23);
        unscale = __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
    }

    if (warp == 0) {
        int it = 0, firsts = 0;
        uint32_t tma = 0;
        for (; it < n_st; ++it) {
            const int s = it % L::kStages;
            if (it % 32 == 0) tma = look(it, &firsts);
            const int first = __shfl_sync(0xffffffffu, firsts, it % 32);
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ((it / L::kStages) & 1) ^ 1, err, DEVERR_TIMEOUT_PRODUCER))) break;
            if (lane == 0) {
                uint8_t* sx = smem + s * L::kStage;
                if (tma >> (it % 32) & 1) {
                    mbar_arrive_expect_tx(&full[s], kGtcX);
#pragma unroll
                    for (int p = 0; p < kGtcCols / 64; ++p) tma_load_2d(sx + p * kGtcPanel, map, &full[s], m0 + p * 64, first);
                } else {
                    mbar_arrive(&full[s]);
                }
            }
        }
        if (lane == 0) {
            for (int j = it > L::kStages ? it - L::kStages : 0; j < it; ++j) mbar_drain(&full[j % L::kStages], (j / L::kStages) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = ad_idesc<W>(RP, true, false);
            for (int it = 0; it < n_st; ++it) {
                const int s = it % L::kStages, set = it % L::kSets;
                if (!mbar_wait(&full[s], (it / L::kStages) & 1, err, DEVERR_TIMEOUT_MMA)) break;
                tc_fence_after();
                const uint32_t sx = smem_u32(smem + s * L::kStage), sl = sx + kGtcX;
#pragma unroll
                for (int h = 0; h < kGtcCols / 128; ++h) {
                    uint32_t more = it >= L::kSets ? 1u : 0u;
#pragma unroll
                    for (int p = kGtcParts - 1; p >= 0; --p)
#pragma unroll
                        for (int kk = 0; kk < kGtcTok / 16; ++kk) {
                            mma_f16_ss(tmem + set * L::kSet + h * RP,
                                       sw128_mnmajor_desc(sx + 2 * h * kGtcPanel + kk * 2048, kGtcPanel),
                                       sw128_kmajor_desc(sl + p * L::kPart + kk * 32), idesc, more);
                            more = 1u;
                        }
                }
                mma_commit(&empty[s]);
            }
            mma_commit(&done);
            mbar_drain(&done, 0);
        }
        __syncwarp();
    } else if (warp < 2 + kGtcConv * 4) {
        // ------------------------------------------------------------ low's parts, then the results
        const int ct = (tid - 64) & 127, group = (tid - 64) >> 7;
        constexpr int kJ = RP < 128 ? RP : 128;             // rank columns side by side over the threads
        constexpr int kOct = kGtcTok / 8;                   // groups of eight tokens
        constexpr int kPer = RP * kOct / 128;               // (column, octet) pairs of a thread
        for (int it = group; it < n_st; it += kGtcConv) {
            const int s = it % L::kStages;
            bool ok = true;
#pragma unroll
            for (int i0 = 0; i0 < kPer; i0 += 4) {
                constexpr int kNow = kPer < 4 ? kPer : 4;
                float v[kNow][8];
#pragma unroll
                for (int i = 0; i < kNow; ++i) {
                    const int idx = ct + (i0 + i) * 128, j = idx % kJ, t0 = it * kGtcTok + idx / kJ * 8;
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        v[i][t] = t0 + t < item.z ? a.low[static_cast<size_t>(item.y + t0 + t) * RP + j] : 0.f;
                }
                if (i0 == 0) ok = mbar_wait(&empty[s], ((it / L::kStages) & 1) ^ 1, err, DEVERR_TIMEOUT_DEQUANT);
                uint8_t* sl = smem + s * L::kStage + kGtcX;
#pragma unroll
                for (int i = 0; i < kNow; ++i) {
                    const int idx = ct + (i0 + i) * 128, j = idx % kJ, oct = idx / kJ;
                    if (AdType<W>::kScaled) {
#pragma unroll
                        for (int t = 0; t < 8; ++t) v[i][t] *= scale;
                    }
#pragma unroll
                    for (int p = 0; p < kGtcParts; ++p) {
                        uint32_t w[4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            w[t] = AdType<W>::pack(v[i][2 * t], v[i][2 * t + 1]);
                            const float2 b = AdType<W>::unpack(w[t]);
                            v[i][2 * t] -= b.x;
                            v[i][2 * t + 1] -= b.y;
                        }
                        *reinterpret_cast<uint4*>(sl + p * L::kPart + sw128_offset(j, oct)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (!__all_sync(0xffffffffu, ok)) break;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[s]);
        }
        if (n_st > 0) mbar_wait(&done, 0, err, DEVERR_TIMEOUT_EPILOGUE);
        tc_fence_after();
        const int q = warp & 3;
        float* out = item.w >= 0 ? a.part + static_cast<size_t>(item.w) * a.M * a.R : a.g + static_cast<size_t>(item.x) * a.M * a.R;
        const int sets = n_st < L::kSets ? n_st : L::kSets;
#pragma unroll 1
        for (int h = group; h < kGtcCols / 128; h += kGtcConv) {
            const int m = m0 + h * 128 + q * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < RP; c += 16) {
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = 0.f;
                for (int set = 0; set < sets; ++set) {
                    uint32_t u[16];
                    tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(q * 32) << 16) + set * L::kSet + h * RP + c, u);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] += __uint_as_float(u[j]);
                }
                if (m < a.M) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (AdType<W>::kScaled) v[j] *= unscale;
                        if (a.gm == 1 && c + j < a.R) out[static_cast<size_t>(c + j) * a.gj + m] = v[j];
                    }
                    if (a.gm != 1) {  // [M][R], R a multiple of 8
                        float4* o = reinterpret_cast<float4*>(out + static_cast<size_t>(m) * a.gm + c);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c + 4 * j < a.R) o[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                }
            }
        }
        tc_fence_before();
    } else {
        // ------------------------------------------------------------ rows in any order, and short stages
        const int ct = tid - 64 - kGtcConv * 128, piece = ct & 31, row0 = ct >> 5;  // pieces of 16 bytes of rows row0 + 4 i
        const bool in = m0 + piece * 8 < a.M;                       // M is a multiple of 8
        int it = 0, firsts;
        uint32_t tma = 0;
        for (; it < n_st; ++it) {
            const int s = it % L::kStages;
            if (it % 32 == 0) tma = look(it, &firsts);
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ((it / L::kStages) & 1) ^ 1, err, DEVERR_TIMEOUT_PRODUCER))) break;
            if (!(tma >> (it % 32) & 1)) {
                uint8_t* dst = smem + s * L::kStage + piece / 8 * kGtcPanel;
#pragma unroll
                for (int i = 0; i < kGtcTok / 4; ++i) {
                    const int r = row0 + 4 * i, at = min(it * kGtcTok + r, item.z - 1);
                    const char* src = static_cast<const char*>(a.x);
                    if (in) src += (static_cast<size_t>(__ldg(perm + at)) * a.ldx + m0 + piece * 8) * 2;
                    cp_async16_part(dst + sw128_offset(r, piece % 8), src, in ? 16 : 0);
                }
            }
            cp_async_commit();
            if (it > 0) {
                cp_async_wait<1>();
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[(it - 1) % L::kStages]);
            }
        }
        cp_async_wait<0>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && it > 0) mbar_arrive(&full[(it - 1) % L::kStages]);
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, L::kTmem);
    }
}

template <typename W, int RP>
cudaError_t launch_t(const AdaptGradPair& p, cudaStream_t st) {
    using L = GtcTile<RP>;
    auto kern = grad_tc_kernel<W, RP>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    const int groups1 = p.g[1].g ? (p.g[1].M + kGtcCols - 1) / kGtcCols : 0;
    return launch_kernel(true, kern, dim3(p.g[0].plan.max_items, p.groups0 + groups1), dim3(kGtcThreads), L::kSmem, st, p);
}

template <typename W>
cudaError_t launch_w(const AdaptGradPair& p, cudaStream_t st) {
    switch (adapt_rp(p.g[0].R)) {
        case 16: return launch_t<W, 16>(p, st);
        case 32: return launch_t<W, 32>(p, st);
        case 64: return launch_t<W, 64>(p, st);
        default: return launch_t<W, 128>(p, st);
    }
}

}  // namespace

cudaError_t launch_adapt_grad_tc(AdaptGradPair p, int type_w, cudaStream_t st) {
    p.groups0 = p.g[0].g ? (p.g[0].M + kGtcCols - 1) / kGtcCols : 0;
    return type_w == HYMOE_TYPE_F16 ? launch_w<__half>(p, st) : launch_w<__nv_bfloat16>(p, st);
}

}  // namespace hymoe
