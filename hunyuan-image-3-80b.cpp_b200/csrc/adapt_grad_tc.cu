// adapt_grad_tc.cu — the adapters' gradients on the 5th-generation tensor cores, for long rows of the
// weights' 16-bit type on 16-byte boundaries: for every adapter, the sum over its tokens of the outer
// products of a long row (x or dy) and its narrow counterpart (low).
//
// split_kernel writes every row of low as three 16-bit parts side by side: bf16 parts hold fp32 whole;
// fp16 ones hold 33 bits below the adapter's largest value, by a power of two that the narrow product
// left behind.  (Splitting within the product, once per column group, held it to a third of what
// memory gives: the converting warps' instructions.)
//
// grad_tc_kernel: a CTA takes 256 columns of the long rows (128 at rank 128) and one item of the plan,
// 64 tokens a stage; both gradients' CTAs are one grid, the longest items first (a long one that
// starts last kept a quarter of the GPU waiting).  The tensor core sums over the tokens: D[128
// columns, parts] += X^T low.
//   A  the rows as they lie in memory, [64 tokens][64 columns] panels: an MN-major operand; by TMA
//      where a stage's tokens are consecutive, else copied
//   B  low's parts, [64 tokens][64 values] panels, MN-major as well; by TMA, a short stage's copied
//      with zeros behind the item's last token
// The pipe truncates what it adds, some 4e-8 of the running sum each time: over 1600 tokens that made
// 2e-6 of a gradient.  So the first part's sums go to two accumulators in turn, 256 tokens each, which
// are added in registers; the other two parts' sums, 2^-8 of them, have one accumulator.  Bound by
// reading the long rows: 8192 tokens of 4096 and 6144 columns, rank 64, 8 adapters take 60 us (2.8
// TB/s; 54 with one accumulator and four times the error), split_kernel 3.
#include "adapt_tc.cuh"

namespace hymoe {
namespace {

constexpr int kGtcTok = 64;
constexpr int kGtcThreads = 448;                  // TMA, MMA, eight warps for the results and four that copy
constexpr int kGtcPanel = kGtcTok * 128;          // 64 values of the stage's rows
constexpr int kGtcParts = 3;
constexpr int kGtcFlush = 4;                      // stages that an accumulator takes

constexpr int gtc_cols(int rp) { return rp < 128 ? 256 : 128; }  // columns per CTA: products of 128

template <int RP>
struct GtcTile {
    static constexpr int kCols = gtc_cols(RP), kHalves = kCols / 128;
    static constexpr int kX = kCols / 64 * kGtcPanel;
    static constexpr int kRest = adapt_rest(RP), kWide = adapt_parts(RP);
    static constexpr int kB = kWide / 64 * kGtcPanel;
    static constexpr int kStage = kX + kB;
    static constexpr int kStages = 224 * 1024 / kStage < 4 ? 224 * 1024 / kStage : 4;
    static constexpr int kSmem = 1024 + kStages * kStage;
    // tensor memory: two sets of the first part's sums, then the others'
    static constexpr int kSet = kHalves * RP, kRestAt = 2 * kSet;
    static_assert(kStages >= 2 && kRestAt + kHalves * 2 * RP <= 512, "a ring, and room for the sums");
};

// fp16 parts: low times 2^shift puts the adapter's largest value in [2^14, 2^15).
__device__ __forceinline__ int gtc_exponent(unsigned amax) { return max(16, min(239, static_cast<int>(amax >> 23))); }

template <typename W, int RP>
__global__ __launch_bounds__(256) void split_kernel(const __grid_constant__ AdaptGradPair pair) {
    using L = GtcTile<RP>;
    const AdaptGrad& a = blockIdx.y == 0 ? pair.g[0] : pair.g[1];
    griddep_wait();
    griddep_launch_dependents();
    if (a.g == nullptr || static_cast<int>(blockIdx.x) >= a.plan.n_lists[3]) return;
    const int4 tile = a.plan.tiles[blockIdx.x];
    float scale = 1.f;
    if (AdType<W>::kScaled) {
        const int e = gtc_exponent(a.plan.amax[blockIdx.y * a.n + tile.x]);
        scale = __uint_as_float(static_cast<uint32_t>(254 + 14 - e) << 23);
    }
    const float4* src = reinterpret_cast<const float4*>(a.low + static_cast<size_t>(tile.y) * RP);
    uint16_t* dst = static_cast<uint16_t*>(pair.parts[blockIdx.y]) + static_cast<size_t>(tile.y) * L::kWide;
    for (int i = threadIdx.x; i < tile.z * (RP / 4); i += 256) {
        const float4 f = src[i];
        float v[4] = {f.x * scale, f.y * scale, f.z * scale, f.w * scale};
        uint16_t* to = dst + static_cast<size_t>(i / (RP / 4)) * L::kWide + i % (RP / 4) * 4;
#pragma unroll
        for (int p = 0; p < kGtcParts; ++p) {
            const uint2 w = make_uint2(AdType<W>::pack(v[0], v[1]), AdType<W>::pack(v[2], v[3]));
            *reinterpret_cast<uint2*>(to + (p == 0 ? 0 : L::kRest + (p - 1) * RP)) = w;
            const float2 lo = AdType<W>::unpack(w.x), hi = AdType<W>::unpack(w.y);
            v[0] -= lo.x;
            v[1] -= lo.y;
            v[2] -= hi.x;
            v[3] -= hi.y;
        }
    }
}

template <typename W, int RP>
__global__ __launch_bounds__(kGtcThreads, 1) void grad_tc_kernel(const __grid_constant__ AdaptGradPair pair) {
    using L = GtcTile<RP>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[L::kStages], empty[L::kStages], acc_full[2], acc_empty[2], done;
    __shared__ uint32_t tmem_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool second = static_cast<int>(blockIdx.x) >= pair.groups0;
    const AdaptGrad& a = second ? pair.g[1] : pair.g[0];
    const CUtensorMap *map_x = second ? &pair.rows[1] : &pair.rows[0], *map_low = second ? &pair.lows[1] : &pair.lows[0];
    const int m0 = (static_cast<int>(blockIdx.x) - (second ? pair.groups0 : 0)) * L::kCols;
    griddep_wait();
    griddep_launch_dependents();
    const int n_items = a.plan.n_lists[2];
    if (static_cast<int>(blockIdx.y) >= n_items) return;
    // a few items: the longest first (ties in their order)
    int which = blockIdx.y;
    if (n_items <= 32) {
        const int len = lane < n_items ? a.plan.items[lane].z : -1;
        int rank = 0;
        for (int j = 0; j < n_items; ++j) {
            const int other = __shfl_sync(0xffffffffu, len, j);
            rank += other > len || (other == len && j < lane) ? 1 : 0;
        }
        which = __ffs(__ballot_sync(0xffffffffu, lane < n_items && rank == which)) - 1;
    }
    const int4 item = a.plan.items[which];
    const int n_st = (item.z + kGtcTok - 1) / kGtcTok;
    const int* perm = a.plan.perm + item.y;
    // Of stages it .. it + 31, one per lane: the first token, and those that TMA takes (whole, of
    // consecutive tokens); the others' rows are copied.
    const auto look = [&](int it, int* first) {
        const int t = (it + lane) * kGtcTok;
        const bool whole = t + kGtcTok <= item.z;
        *first = whole ? __ldg(perm + t) : 0;
        const int last = whole ? __ldg(perm + t + kGtcTok - 1) : 0;
        return __ballot_sync(0xffffffffu, whole && last - *first == kGtcTok - 1);
    };
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full[s], 5);  // TMA's thread and four copying warps
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 8);
        }
        mbar_init(&done, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_s, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    int* err = a.plan.err;

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
                const bool rows = tma >> (it % 32) & 1, low = (it + 1) * kGtcTok <= item.z;
                mbar_arrive_expect_tx(&full[s], (rows ? L::kX : 0) + (low ? L::kB : 0));
                if (rows) {
#pragma unroll
                    for (int p = 0; p < L::kCols / 64; ++p) tma_load_2d(sx + p * kGtcPanel, map_x, &full[s], m0 + p * 64, first);
                }
                if (low) {
#pragma unroll
                    for (int p = 0; p < L::kWide / 64; ++p)
                        tma_load_2d(sx + L::kX + p * kGtcPanel, map_low, &full[s], p * 64, item.y + it * kGtcTok);
                }
            }
        }
        if (lane == 0) {
            for (int j = it > L::kStages ? it - L::kStages : 0; j < it; ++j) mbar_drain(&full[j % L::kStages], (j / L::kStages) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t first_part = ad_idesc<W>(RP, true, true), other_parts = ad_idesc<W>(2 * RP, true, true);
            for (int it = 0; it < n_st; ++it) {
                const int s = it % L::kStages, run = it / kGtcFlush, b = run & 1;
                if (it % kGtcFlush == 0 && run >= 2 && !mbar_wait(&acc_empty[b], ((run >> 1) & 1) ^ 1, err, DEVERR_TIMEOUT_MMA)) break;
                if (!mbar_wait(&full[s], (it / L::kStages) & 1, err, DEVERR_TIMEOUT_MMA)) break;
                tc_fence_after();
                const uint32_t sx = smem_u32(smem + s * L::kStage), sl = sx + L::kX, sr = sl + L::kRest / 64 * kGtcPanel;
#pragma unroll
                for (int h = 0; h < L::kHalves; ++h) {
#pragma unroll
                    for (int kk = 0; kk < kGtcTok / 16; ++kk) {
                        const uint64_t da = sw128_mnmajor_desc(sx + 2 * h * kGtcPanel + kk * 2048, kGtcPanel);
                        mma_f16_ss(tmem + b * L::kSet + h * RP, da, sw128_mnmajor_desc(sl + kk * 2048, kGtcPanel), first_part,
                                   it % kGtcFlush != 0 || kk > 0 ? 1u : 0u);
                        mma_f16_ss(tmem + L::kRestAt + h * 2 * RP, da, sw128_mnmajor_desc(sr + kk * 2048, kGtcPanel), other_parts,
                                   it > 0 || kk > 0 ? 1u : 0u);
                    }
                }
                mma_commit(&empty[s]);
                if (it % kGtcFlush == kGtcFlush - 1 || it == n_st - 1) mma_commit(&acc_full[b]);
            }
            mma_commit(&done);
            mbar_drain(&done, 0);  // every product has ended before tensor memory is freed
        }
        __syncwarp();
    } else if (warp < 10) {
        // ------------------------------------------------------------ the results
        // a warp has 32 columns of the rows (a quarter of the accumulators' lanes) and half of the sums:
        // ranks j0 .. j0 + kOwn of half h
        constexpr int kOwn = L::kHalves * RP / 2;
        const int q = warp & 3, group = (warp - 2) >> 2;
        const int h = L::kHalves == 2 ? group : 0, j0 = L::kHalves == 2 ? 0 : group * kOwn;
        const uint32_t mine = tmem + (static_cast<uint32_t>(q * 32) << 16);
        float v[kOwn];
#pragma unroll
        for (int j = 0; j < kOwn; ++j) v[j] = 0.f;
        const int runs = (n_st + kGtcFlush - 1) / kGtcFlush;
        for (int run = 0; run < runs; ++run) {
            const int b = run & 1;
            // on an expired wait the status word says that the results are not valid
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (run >> 1) & 1, err, DEVERR_TIMEOUT_EPILOGUE))) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < kOwn; c += 16) {
                uint32_t u[16];
                tmem_ld_32x32b_x16(mine + b * L::kSet + h * RP + j0 + c, u);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[c + j] += __uint_as_float(u[j]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
        }
        if (n_st > 0) {
#pragma unroll
            for (int c = 0; c < 2 * kOwn; c += 16) {
                uint32_t u[16];
                tmem_ld_32x32b_x16(mine + L::kRestAt + h * 2 * RP + c / kOwn * RP + j0 + c % kOwn, u);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[c % kOwn + j] += __uint_as_float(u[j]);
            }
        }
        float unscale = 1.f;
        if (AdType<W>::kScaled)
            unscale = __uint_as_float(static_cast<uint32_t>(gtc_exponent(a.plan.amax[(second ? a.n : 0) + item.x]) - 14) << 23);
        float* out = item.w >= 0 ? a.part + static_cast<size_t>(item.w) * a.M * a.R : a.g + static_cast<size_t>(item.x) * a.M * a.R;
        const int m = m0 + h * 128 + q * 32 + lane;
        if (m < a.M) {
            if (AdType<W>::kScaled) {
#pragma unroll
                for (int j = 0; j < kOwn; ++j) v[j] *= unscale;
            }
            if (a.gm == 1) {
#pragma unroll
                for (int j = 0; j < kOwn; ++j)
                    if (j0 + j < a.R) out[static_cast<size_t>(j0 + j) * a.gj + m] = v[j];
            } else {  // [M][R], R a multiple of 8
                float4* o = reinterpret_cast<float4*>(out + static_cast<size_t>(m) * a.gm + j0);
#pragma unroll
                for (int j = 0; j < kOwn / 4; ++j)
                    if (j0 + 4 * j < a.R) o[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            }
        }
        tc_fence_before();
    } else {
        // ------------------------------------------------------------ rows in any order, and short stages
        constexpr int kPieces = L::kCols / 8, kStep = 128 / kPieces;  // pieces of 16 bytes of rows row0 + kStep i
        const int ct = tid - 320, piece = ct % kPieces, row0 = ct / kPieces;
        const bool in = m0 + piece * 8 < a.M;                       // M is a multiple of 8
        int it = 0, firsts;
        uint32_t tma = 0;
        for (; it < n_st; ++it) {
            const int s = it % L::kStages, left = item.z - it * kGtcTok;
            if (it % 32 == 0) tma = look(it, &firsts);
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ((it / L::kStages) & 1) ^ 1, err, DEVERR_TIMEOUT_PRODUCER))) break;
            uint8_t* sx = smem + s * L::kStage;
            if (!(tma >> (it % 32) & 1)) {
                uint8_t* dst = sx + piece / 8 * kGtcPanel;
#pragma unroll
                for (int i = 0; i < kGtcTok / kStep; ++i) {
                    const int r = row0 + kStep * i;
                    const bool have = in && r < left;
                    const char* src = static_cast<const char*>(a.x);
                    if (have) src += (static_cast<size_t>(__ldg(perm + it * kGtcTok + r)) * a.ldx + m0 + piece * 8) * 2;
                    cp_async16_part(dst + sw128_offset(r, piece % 8), src, have ? 16 : 0);
                }
            }
            if (left < kGtcTok) {
                const char* low = static_cast<const char*>(second ? pair.parts[1] : pair.parts[0]);
                for (int i = ct; i < kGtcTok * (L::kWide / 8); i += 128) {
                    const int r = i / (L::kWide / 8), c = i % (L::kWide / 8);
                    const bool have = r < left;
                    const char* src = have ? low + (static_cast<size_t>(item.y + it * kGtcTok + r) * L::kWide + c * 8) * 2 : low;
                    cp_async16_part(sx + L::kX + c / 8 * kGtcPanel + sw128_offset(r, c % 8), src, have ? 16 : 0);
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
        tmem_dealloc(tmem, 512);
    }
}

template <typename W, int RP>
cudaError_t launch_t(const AdaptGradPair& p, cudaStream_t st) {
    using L = GtcTile<RP>;
    auto kern = grad_tc_kernel<W, RP>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e == cudaSuccess) e = launch_kernel(true, split_kernel<W, RP>, dim3(p.g[0].plan.max_tiles, 2), dim3(256), 0, st, p);
    if (e != cudaSuccess) return e;
    const int groups1 = p.g[1].g ? (p.g[1].M + L::kCols - 1) / L::kCols : 0;
    return launch_kernel(true, kern, dim3(p.groups0 + groups1, p.g[0].plan.max_items), dim3(kGtcThreads), L::kSmem, st, p);
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
    const int cols = gtc_cols(adapt_rp(p.g[0].R));
    p.groups0 = p.g[0].g ? (p.g[0].M + cols - 1) / cols : 0;
    return type_w == HYMOE_TYPE_F16 ? launch_w<__half>(p, st) : launch_w<__nv_bfloat16>(p, st);
}

}  // namespace hymoe
