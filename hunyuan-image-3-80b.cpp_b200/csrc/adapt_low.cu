// adapt_low.cu — the adapters' narrow product: low[row] = scale[a] * W_a x[token of row].
//
// A tile of 64 sorted rows of one adapter is one cluster of S CTAs (S = 1, 2, 4, 8), each over a
// part of the long dimension; the S partial sums [64, RP] meet in distributed shared memory, where
// every CTA adds its share of the rows in the order of the ranks.  Bound by reading x (the weights,
// RP / 64 of its bytes per tile, come from L2): four stages of 64 columns are in flight per CTA.
#include "adapt.cuh"
#include "kernels.h"

namespace hymoe {
namespace {

constexpr int kLowK = 64;      // columns per stage
constexpr int kLowStages = 4;

template <typename X, typename W, int RP, bool TRANS>
struct LowTile {
    static constexpr bool kF32 = sizeof(X) == 4;
    static constexpr int kXRow = kF32 ? kLowK * 4 + 32 : kLowK * 2 + 16;
    static constexpr int kWRow = TRANS ? ad_pad16(RP * 2) : kLowK * 2 + 16;
    static constexpr int kXBytes = kAdRows * kXRow;
    static constexpr int kWBytes = (TRANS ? kLowK : RP) * kWRow;
    static constexpr int kStage = kXBytes + kWBytes;
    static constexpr int kRed = kAdRows * (RP + 4) * 4;  // partial sums
    static constexpr int kSmem = kStage * kLowStages > kRed ? kStage * kLowStages : kRed;
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

template <typename X, typename W, int RP, bool TRANS>
__global__ __launch_bounds__(kAdThreads) void low_kernel(const __grid_constant__ AdaptLow a, int S) {
    using L = LowTile<X, W, RP, TRANS>;
    extern __shared__ __align__(128) char smem[];
    griddep_wait();
    griddep_launch_dependents();
    const int tile_id = blockIdx.x / S, rank = blockIdx.x % S;
    if (tile_id >= a.plan.n_lists[0]) return;  // the whole cluster
    const int4 tile = a.plan.tiles[tile_id];
    if (tile.x < 0) return;  // rows without an adapter
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nk = (a.K + kLowK - 1) / kLowK;
    const int k_lo = static_cast<int>(static_cast<int64_t>(nk) * rank / S);
    const int k_hi = static_cast<int>(static_cast<int64_t>(nk) * (rank + 1) / S);

    // this thread's pieces of every stage's x tile: piece xc of rows xr0 + i * (128 / pieces)
    constexpr int kXPieces = kLowK * static_cast<int>(sizeof(X)) / 16, kXIter = kAdRows * kXPieces / kAdThreads;
    const int xc = tid % kXPieces, xr0 = tid / kXPieces;
    const char* xp[kXIter];
    unsigned xok = 0;
#pragma unroll
    for (int i = 0; i < kXIter; ++i) {
        const int r = xr0 + i * (kAdThreads / kXPieces);
        const bool ok = r < tile.z;
        const int tok = ok ? __ldg(a.plan.perm + tile.y + r) : 0;
        xp[i] = static_cast<const char*>(a.x) + static_cast<size_t>(tok) * a.ldx * sizeof(X);
        if (ok) xok |= 1u << i;
    }
    const char* wbase = static_cast<const char*>(a.w) + static_cast<size_t>(tile.x) * a.R * a.K * 2;
    auto load = [&](int stage, int kb) {
        char* xs = smem + stage * L::kStage;
        char* ws = xs + L::kXBytes;
        const int k0 = kb * kLowK;
        constexpr int P = 16 / static_cast<int>(sizeof(X));
#pragma unroll
        for (int i = 0; i < kXIter; ++i) {
            const int r = xr0 + i * (kAdThreads / kXPieces), k = k0 + xc * P;
            const int n = (xok >> i & 1) ? a.K - k : 0;
            ad_copy_piece<sizeof(X)>(xs + r * L::kXRow + xc * 16,
                                     n > 0 ? xp[i] + static_cast<size_t>(k) * sizeof(X) : static_cast<const char*>(a.x), n, a.vec_x);
        }
        constexpr int kWPieces = TRANS ? RP / 8 : kLowK / 8, kWAll = (TRANS ? kLowK : RP) * kWPieces;
#pragma unroll
        for (int i = 0; i < (kWAll + kAdThreads - 1) / kAdThreads; ++i) {
            const int p = tid + i * kAdThreads;
            if (kWAll % kAdThreads != 0 && p >= kWAll) break;
            const int r = p / kWPieces, c = p % kWPieces;
            int n;
            size_t off;
            if (TRANS) {  // row = k, columns = rank
                n = k0 + r < a.K ? a.R - c * 8 : 0;
                off = static_cast<size_t>(k0 + r) * a.R + c * 8;
            } else {      // row = rank, columns = k
                n = r < a.R ? a.K - (k0 + c * 8) : 0;
                off = static_cast<size_t>(r) * a.K + k0 + c * 8;
            }
            ad_copy_piece<2>(ws + r * L::kWRow + c * 16, n > 0 ? wbase + off * 2 : wbase, n, a.vec_w);
        }
    };

    float acc[RP / 8][4];
#pragma unroll
    for (int i = 0; i < RP / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

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
#pragma unroll
        for (int kk = 0; kk < kLowK / 16; ++kk) {
            uint32_t bf[RP / 16][4];
#pragma unroll
            for (int j = 0; j < RP / 16; ++j) {
                if (TRANS)  // blocks (k 0-7, n 0-7), (k 8-15, n 0-7), (k 0-7, n 8-15), (k 8-15, n 8-15)
                    ldsm4_t(bf[j], wa + (kk * 16 + (lane & 15)) * L::kWRow + (j * 16 + (lane >> 4) * 8) * 2);
                else
                    ldsm4(bf[j], wa + (j * 16 + (lane >> 4) * 8 + (lane & 7)) * L::kWRow + (kk * 16 + (lane >> 3 & 1) * 8) * 2);
            }
            if constexpr (!L::kF32) {
                uint32_t af[4];
                ldsm4(af, xa + (warp * 16 + (lane & 15)) * L::kXRow + (kk * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
                for (int j = 0; j < RP / 16; ++j) {
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
                    split_tf32(v[h][0].x, hi[0], lo[0]);
                    split_tf32(v[h][1].x, hi[1], lo[1]);
                    split_tf32(v[h][0].y, hi[2], lo[2]);
                    split_tf32(v[h][1].y, hi[3], lo[3]);
#pragma unroll
                    for (int j = 0; j < RP / 16; ++j)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float2 b = AdType<W>::unpack(bf[j][2 * q + h]);
                            mma_tf32(acc[2 * j + q], lo, __float_as_uint(b.x), __float_as_uint(b.y));
                            mma_tf32(acc[2 * j + q], hi, __float_as_uint(b.x), __float_as_uint(b.y));
                        }
                }
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();  // the stages become the partial sums
    {
        float* red = reinterpret_cast<float*>(smem);
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < RP / 8; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q)
                *reinterpret_cast<float2*>(red + (warp * 16 + g + 8 * q) * (RP + 4) + j * 8 + 2 * t) =
                    make_float2(acc[j][2 * q], acc[j][2 * q + 1]);
    }
    cluster_sync();
    const float f = a.scale != nullptr ? __ldg(a.scale + tile.x) : 1.f;
    const int rows = kAdRows / S;
    for (int p = tid; p < rows * (RP / 4); p += kAdThreads) {
        const int r = rank * rows + p / (RP / 4), c = p % (RP / 4) * 4;
        if (r >= tile.z) continue;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int q = 0; q < S; ++q) {
            const float4 v = ld_cluster4(mapa_shared(smem + (r * (RP + 4) + c) * 4, q));
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
        *reinterpret_cast<float4*>(a.low + static_cast<size_t>(tile.y + r) * RP + c) =
            make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
    }
    cluster_sync();  // no CTA leaves while another reads its sums
}

template <typename X, typename W, int RP, bool TRANS>
cudaError_t launch_t(const AdaptLow& a, int T, int n_sms, cudaStream_t st) {
    using L = LowTile<X, W, RP, TRANS>;
    auto kern = low_kernel<X, W, RP, TRANS>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    // enough CTAs for two on every SM, each with at least four stages of columns
    const int tiles = (T + kAdRows - 1) / kAdRows, nk = (a.K + kLowK - 1) / kLowK;
    int S = 1;
    while (S < 8 && tiles * S < 2 * n_sms && nk / (2 * S) >= kLowStages) S *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.plan.max_tiles) * S);
    cfg.blockDim = dim3(kAdThreads);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a, S);
}

template <typename X, typename W>
cudaError_t launch_x(const AdaptLow& a, bool trans, int T, int n_sms, cudaStream_t st) {
    switch (adapt_rp(a.R)) {
        case 16: return trans ? launch_t<X, W, 16, true>(a, T, n_sms, st) : launch_t<X, W, 16, false>(a, T, n_sms, st);
        case 32: return trans ? launch_t<X, W, 32, true>(a, T, n_sms, st) : launch_t<X, W, 32, false>(a, T, n_sms, st);
        case 64: return trans ? launch_t<X, W, 64, true>(a, T, n_sms, st) : launch_t<X, W, 64, false>(a, T, n_sms, st);
        default: return trans ? launch_t<X, W, 128, true>(a, T, n_sms, st) : launch_t<X, W, 128, false>(a, T, n_sms, st);
    }
}

}  // namespace

cudaError_t launch_adapt_low(const AdaptLow& a, int type_x, int type_w, bool trans, int T, int n_sms, cudaStream_t st) {
    if (type_w == HYMOE_TYPE_F16)
        return type_x == HYMOE_TYPE_F32 ? launch_x<float, __half>(a, trans, T, n_sms, st)
                                        : launch_x<__half, __half>(a, trans, T, n_sms, st);
    return type_x == HYMOE_TYPE_F32 ? launch_x<float, __nv_bfloat16>(a, trans, T, n_sms, st)
                                    : launch_x<__nv_bfloat16, __nv_bfloat16>(a, trans, T, n_sms, st);
}

}  // namespace hymoe
