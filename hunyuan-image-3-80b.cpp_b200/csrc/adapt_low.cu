// adapt_low.cu — the adapters' narrow product: low[row] = scale[a] * W_a x[token of row].
//
// A tile of 64 sorted rows of one adapter is shared by S CTAs, each over a part of the long
// dimension.  Every CTA leaves its partial sums [64, RP] in the workspace; the last one of a tile to
// arrive adds them in the order of the parts.  The matrix pipe truncates what it adds, so a stage's
// products (16 additions for F32 rows, 4 for others) start from zero and join fp32 sums outside it: left
// in its accumulators, 4096 columns of a CTA cost 2e-5 of low, and more the longer the rows.  Bound by reading x (the weights, RP / 64 of its
// bytes per tile, come from L2): four stages of 64 columns are in flight per CTA, and S is chosen
// so that the CTAs fill the GPU once.  77 tokens of 4096 columns, rank 16, both narrow products of a
// backward pass: 8.8 us.  Long batches of F32 rows are bound by the tf32 pipe (two products for x's
// two parts): 8192 tokens of 4096 columns, rank 64, 78 us; bf16 rows off 16-byte boundaries by their
// copies of 2 bytes: 85 us (125 with the weights off them too).
#include "adapt.cuh"
#include "kernels.h"

namespace hymoe {
namespace {

constexpr int kLowK = 64;      // columns per stage
constexpr int kLowStages = 4;

template <typename X, typename W, int RP, bool TRANS>
struct LowTile {
    static constexpr bool kF32 = sizeof(X) == 4;
    // Groups of four warps that share the rank: the sums and a stage's accumulators of all 128 columns
    // beside two tf32 parts do not fit one warp's registers (and one warp a scheduler, as large stages
    // leave, waited for its own products).
    static constexpr int kGroups = kF32 && RP == 128 ? 2 : 1;
    static constexpr int kThreads = kGroups * kAdThreads, kOwn = RP / kGroups;  // columns of a warp
    static constexpr int kXRow = kF32 ? kLowK * 4 + 32 : kLowK * 2 + 16;
    static constexpr int kWRow = TRANS ? ad_pad16(RP * 2) : kLowK * 2 + 16;
    static constexpr int kXBytes = kAdRows * kXRow;
    static constexpr int kWBytes = (TRANS ? kLowK : RP) * kWRow;
    static constexpr int kStage = kXBytes + kWBytes;
    static constexpr int kSmem = kStage * kLowStages;
    static constexpr int kPerSm = 226 * 1024 / (kSmem + 1024) < 4 ? 226 * 1024 / (kSmem + 1024) : 4;  // CTAs on an SM
};

template <typename X, typename W, int RP, bool TRANS>
__device__ __forceinline__ void low_tile(const AdaptLow& a, int S, char* smem) {
    using L = LowTile<X, W, RP, TRANS>;
    const int tile_id = blockIdx.x / S, rank = blockIdx.x % S;
    const int4 tile = ad_part_tile(a.plan, tile_id);
    if (tile.x < 0) return;  // none, or rows without an adapter
    const int tid = threadIdx.x, warp = tid >> 5 & 3, lane = tid & 31;
    const int c0 = L::kGroups == 1 ? 0 : (tid >> 7) * L::kOwn;  // this warp's columns of the rank
    const int nk = (a.K + kLowK - 1) / kLowK;
    const int k_lo = static_cast<int>(static_cast<int64_t>(nk) * rank / S);
    const int k_hi = static_cast<int>(static_cast<int64_t>(nk) * (rank + 1) / S);

    // this thread's pieces of every stage: piece xc of rows xr0 + i * (128 / pieces) of x, and piece
    // p % kWPieces of row p / kWPieces of the weights, p = tid + i * 128
    constexpr int P = 16 / static_cast<int>(sizeof(X));
    constexpr int kXPieces = kLowK / P, kXIter = kAdRows * kXPieces / L::kThreads;
    constexpr int kWPieces = TRANS ? RP / 8 : kLowK / 8, kWAll = (TRANS ? kLowK : RP) * kWPieces;
    constexpr int kWIter = kWAll / L::kThreads;
    static_assert(kWAll % L::kThreads == 0, "whole rounds of pieces");
    const int xc = tid % kXPieces, xr0 = tid / kXPieces;
    const char* xp[kXIter];  // the piece in column 0; rows that do not exist have no bytes
    int xn[kXIter];
#pragma unroll
    for (int i = 0; i < kXIter; ++i) {
        const int r = xr0 + i * (L::kThreads / kXPieces);
        const bool ok = r < tile.z;
        const int tok = ok ? __ldg(a.plan.perm + tile.y + r) : 0;
        xp[i] = static_cast<const char*>(a.x) + (static_cast<size_t>(tok) * a.ldx + (ok ? xc * P : 0)) * sizeof(X);
        xn[i] = ok ? 16 : 0;
    }
    const char* wbase = static_cast<const char*>(a.w) + static_cast<size_t>(tile.x) * a.R * a.K * 2;
    const char* wp[kWIter];
    int wn[kWIter];
#pragma unroll
    for (int i = 0; i < kWIter; ++i) {
        const int p = tid + i * L::kThreads, r = p / kWPieces, c = p % kWPieces * 8;
        const bool ok = TRANS ? c < a.R : r < a.R;  // trans: row = k, columns = rank; else row = rank, columns = k
        wp[i] = ok ? wbase + (static_cast<size_t>(r) * (TRANS ? a.R : a.K) + c) * 2 : wbase;
        wn[i] = !ok ? 0 : TRANS ? min(16, (a.R - c) * 2) : 16;
    }
    const bool vec = a.vec_x && a.vec_w;
    auto load = [&](int stage, int kb) {
        char* xs = smem + stage * L::kStage;
        char* ws = xs + L::kXBytes;
        const int k0 = kb * kLowK;
        if (vec && k0 + kLowK <= a.K) {  // a whole block of aligned rows
#pragma unroll
            for (int i = 0; i < kXIter; ++i)
                cp_async16_part(xs + (xr0 + i * (L::kThreads / kXPieces)) * L::kXRow + xc * 16,
                                xp[i] + static_cast<size_t>(k0) * sizeof(X), xn[i]);
            const size_t adv = static_cast<size_t>(k0) * (TRANS ? a.R : 1) * 2;
#pragma unroll
            for (int i = 0; i < kWIter; ++i) {
                const int p = tid + i * L::kThreads;
                cp_async16_part(ws + p / kWPieces * L::kWRow + p % kWPieces * 16, wn[i] ? wp[i] + adv : wbase, wn[i]);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kXIter; ++i) {
            const int r = xr0 + i * (L::kThreads / kXPieces), n = xn[i] ? a.K - (k0 + xc * P) : 0;
            ad_copy_piece<sizeof(X)>(xs + r * L::kXRow + xc * 16,
                                     n > 0 ? xp[i] + static_cast<size_t>(k0) * sizeof(X) : static_cast<const char*>(a.x), n, a.vec_x);
        }
#pragma unroll
        for (int i = 0; i < kWIter; ++i) {
            const int p = tid + i * L::kThreads, r = p / kWPieces, c = p % kWPieces;
            const int n = wn[i] == 0 ? 0 : TRANS ? (k0 + r < a.K ? a.R - c * 8 : 0) : a.K - (k0 + c * 8);
            ad_copy_piece<2>(ws + r * L::kWRow + c * 16,
                             n > 0 ? wp[i] + static_cast<size_t>(k0) * (TRANS ? a.R : 1) * 2 : wbase, n, a.vec_w);
        }
    };

    float sum[L::kOwn / 8][4];
#pragma unroll
    for (int i = 0; i < L::kOwn / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = 0.f;

#pragma unroll
    for (int s = 0; s < kLowStages - 1; ++s) {
        if (k_lo + s < k_hi) load(s, k_lo + s);
        cp_async_commit();
    }
    for (int kb = k_lo; kb < k_hi; ++kb) {
        const int stage = (kb - k_lo) % kLowStages;
        cp_async_wait<kLowStages - 2>();
        __syncthreads();
        const int nxt = kb + kLowStages - 1;
        if (nxt < k_hi) load((nxt - k_lo) % kLowStages, nxt);
        cp_async_commit();
        const char* xs = smem + stage * L::kStage;
        const uint32_t xa = smem_u32(xs), wa = xa + L::kXBytes;
        float acc[L::kOwn / 8][4];  // this stage's products
#pragma unroll
        for (int i = 0; i < L::kOwn / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll
        for (int kk = 0; kk < kLowK / 16; ++kk) {
            uint32_t bf[L::kOwn / 16][4];
#pragma unroll
            for (int j = 0; j < L::kOwn / 16; ++j) {
                if (TRANS)  // blocks (k 0-7, n 0-7), (k 8-15, n 0-7), (k 0-7, n 8-15), (k 8-15, n 8-15)
                    ldsm4_t(bf[j], wa + (kk * 16 + (lane & 15)) * L::kWRow + (c0 + j * 16 + (lane >> 4) * 8) * 2);
                else
                    ldsm4(bf[j], wa + (c0 + j * 16 + (lane >> 4) * 8 + (lane & 7)) * L::kWRow + (kk * 16 + (lane >> 3 & 1) * 8) * 2);
            }
            if constexpr (!L::kF32) {
                uint32_t af[4];
                ldsm4(af, xa + (warp * 16 + (lane & 15)) * L::kXRow + (kk * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
                for (int j = 0; j < L::kOwn / 16; ++j) {
                    AdType<W>::mma(acc[2 * j], af, bf[j][0], bf[j][1]);
                    AdType<W>::mma(acc[2 * j + 1], af, bf[j][2], bf[j][3]);
                }
            } else {
                // fp32 rows as two tf32 parts; the weights are exact in tf32
                const int g = lane >> 2, t = lane & 3;
                float2 v[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        v[h][q] = *reinterpret_cast<const float2*>(xs + (warp * 16 + g + 8 * q) * L::kXRow + (kk * 16 + h * 8 + 2 * t) * 4);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t hi[4], lo[4];
                    const float part[4] = {v[h][0].x, v[h][1].x, v[h][0].y, v[h][1].y};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        split_tf32(part[i], hi[i], lo[i]);
                        lo[i] = __float_as_uint(part_rest(part[i], __uint_as_float(hi[i])));
                    }
#pragma unroll
                    for (int j = 0; j < L::kOwn / 16; ++j)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float2 b = AdType<W>::unpack(bf[j][2 * q + h]);
                            mma_tf32(acc[2 * j + q], lo, __float_as_uint(b.x), __float_as_uint(b.y));
                            mma_tf32(acc[2 * j + q], hi, __float_as_uint(b.x), __float_as_uint(b.y));
                        }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < L::kOwn / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[i][j] += acc[i][j];
    }
    cp_async_wait<0>();
    const float f = a.scale != nullptr ? __ldg(a.scale + tile.x) : 1.f;
    const int g = lane >> 2, t = lane & 3;
    float* dst = S == 1 ? a.low + static_cast<size_t>(tile.y) * RP
                        : a.part + (static_cast<size_t>(tile_id) * S + rank) * (kAdRows * RP);
    const float f1 = S == 1 ? f : 1.f;
    float top = 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = warp * 16 + g + 8 * q;
        if (r >= tile.z) continue;
#pragma unroll
        for (int j = 0; j < L::kOwn / 8; ++j) {
            const int c = c0 + j * 8 + 2 * t;  // (columns behind the rank: 0 times an infinity is none of the result's)
            const float2 v = make_float2(c < a.R ? sum[j][2 * q] * f1 : 0.f, c + 1 < a.R ? sum[j][2 * q + 1] * f1 : 0.f);
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
            *reinterpret_cast<float2*>(dst + static_cast<size_t>(r) * RP + c) = v;
        }
    }
    __syncwarp();
    if (S == 1) {
        if (a.amax != nullptr) ad_amax(a.amax + tile.x, top);
        return;
    }
    // The tile's last CTA adds the parts.  Its counter wraps back to 0 for the next call.
    __shared__ int last;
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicInc(a.plan.counters + tile_id, S - 1) == static_cast<unsigned>(S - 1);
    __syncthreads();
    if (!last) return;
    __threadfence();
    const float* part = a.part + static_cast<size_t>(tile_id) * S * (kAdRows * RP);
    top = 0.f;
    for (int p = tid; p < tile.z * (RP / 4); p += L::kThreads) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int q = 0; q < S; ++q) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part + static_cast<size_t>(q) * (kAdRows * RP)) + p);
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
        s = make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
        top = fmaxf(top, fmaxf(fmaxf(fabsf(s.x), fabsf(s.y)), fmaxf(fabsf(s.z), fabsf(s.w))));
        reinterpret_cast<float4*>(a.low + static_cast<size_t>(tile.y) * RP)[p] = s;
    }
    __syncwarp();
    if (a.amax != nullptr) ad_amax(a.amax + tile.x, top);
}

template <typename X, typename W, int RP, bool TRANS>
__global__ __launch_bounds__(LowTile<X, W, RP, TRANS>::kThreads, LowTile<X, W, RP, TRANS>::kPerSm) void low_kernel(
    const __grid_constant__ AdaptLow a, int S) {
    extern __shared__ __align__(128) char smem[];
    griddep_wait();
    griddep_launch_dependents();
    low_tile<X, W, RP, TRANS>(a, S, smem);
}

// Grid (tiles x the larger S, 2).
template <typename X, typename W, int RP>
__global__ __launch_bounds__(LowTile<X, W, RP, true>::kThreads) void low_pair_kernel(const __grid_constant__ AdaptLow a, int Sa,
                                                              const __grid_constant__ AdaptLow b, int Sb, int tiles) {
    extern __shared__ __align__(128) char smem[];
    griddep_wait();
    griddep_launch_dependents();
    if (static_cast<int>(blockIdx.x) >= tiles * (blockIdx.y == 0 ? Sa : Sb)) return;
    if (blockIdx.y == 0) low_tile<X, W, RP, true>(a, Sa, smem);
    else low_tile<X, W, RP, false>(b, Sb, smem);
}

template <typename X, typename W, int RP>
cudaError_t launch_pair(const AdaptLow& a, const AdaptLow& b, int n_sms, cudaStream_t st) {
    using La = LowTile<X, W, RP, true>;
    using Lb = LowTile<X, W, RP, false>;
    constexpr int smem = La::kSmem > Lb::kSmem ? La::kSmem : Lb::kSmem;
    constexpr int per_sm = La::kPerSm < Lb::kPerSm ? La::kPerSm : Lb::kPerSm;
    auto kern = low_pair_kernel<X, W, RP>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int tiles = a.plan.max_tiles * (a.plan.tile_rows / kAdRows);
    const int Sa = adapt_splits(tiles, a.K, per_sm * n_sms / 2), Sb = adapt_splits(tiles, b.K, per_sm * n_sms / 2);
    return launch_kernel(true, kern, dim3(static_cast<unsigned>(tiles) * (Sa > Sb ? Sa : Sb), 2), dim3(La::kThreads), smem, st, a, Sa,
                         b, Sb, tiles);
}

template <typename X, typename W>
cudaError_t launch_pair_x(const AdaptLow& a, const AdaptLow& b, int n_sms, cudaStream_t st) {
    switch (adapt_rp(a.R)) {
        case 16: return launch_pair<X, W, 16>(a, b, n_sms, st);
        case 32: return launch_pair<X, W, 32>(a, b, n_sms, st);
        case 64: return launch_pair<X, W, 64>(a, b, n_sms, st);
        default: return launch_pair<X, W, 128>(a, b, n_sms, st);
    }
}

template <typename X, typename W, int RP, bool TRANS>
cudaError_t launch_t(const AdaptLow& a, int n_sms, cudaStream_t st) {
    using L = LowTile<X, W, RP, TRANS>;
    auto kern = low_kernel<X, W, RP, TRANS>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    const int tiles = a.plan.max_tiles * (a.plan.tile_rows / kAdRows);
    const int S = adapt_splits(tiles, a.K, L::kPerSm * n_sms);
    return launch_kernel(true, kern, dim3(static_cast<unsigned>(tiles) * S), dim3(L::kThreads), L::kSmem, st, a, S);
}

template <typename X, typename W>
cudaError_t launch_x(const AdaptLow& a, bool trans, int n_sms, cudaStream_t st) {
    switch (adapt_rp(a.R)) {
        case 16: return trans ? launch_t<X, W, 16, true>(a, n_sms, st) : launch_t<X, W, 16, false>(a, n_sms, st);
        case 32: return trans ? launch_t<X, W, 32, true>(a, n_sms, st) : launch_t<X, W, 32, false>(a, n_sms, st);
        case 64: return trans ? launch_t<X, W, 64, true>(a, n_sms, st) : launch_t<X, W, 64, false>(a, n_sms, st);
        default: return trans ? launch_t<X, W, 128, true>(a, n_sms, st) : launch_t<X, W, 128, false>(a, n_sms, st);
    }
}

}  // namespace

cudaError_t launch_adapt_lows(const AdaptLow& a, const AdaptLow& b, int type_x, int type_w, int n_sms, cudaStream_t st) {
    if (type_w == HYMOE_TYPE_F16)
        return type_x == HYMOE_TYPE_F32 ? launch_pair_x<float, __half>(a, b, n_sms, st)
                                        : launch_pair_x<__half, __half>(a, b, n_sms, st);
    return type_x == HYMOE_TYPE_F32 ? launch_pair_x<float, __nv_bfloat16>(a, b, n_sms, st)
                                    : launch_pair_x<__nv_bfloat16, __nv_bfloat16>(a, b, n_sms, st);
}

cudaError_t launch_adapt_low(const AdaptLow& a, int type_x, int type_w, bool trans, int n_sms, cudaStream_t st) {
    if (type_w == HYMOE_TYPE_F16)
        return type_x == HYMOE_TYPE_F32 ? launch_x<float, __half>(a, trans, n_sms, st)
                                        : launch_x<__half, __half>(a, trans, n_sms, st);
    return type_x == HYMOE_TYPE_F32 ? launch_x<float, __nv_bfloat16>(a, trans, n_sms, st)
                                    : launch_x<__nv_bfloat16, __nv_bfloat16>(a, trans, n_sms, st);
}

}  // namespace hymoe
