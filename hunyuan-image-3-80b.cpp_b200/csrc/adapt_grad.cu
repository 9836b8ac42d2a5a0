// adapt_grad.cu — the adapters' gradients: for every adapter, the sum over its tokens of the outer
// products of a long row (x or dy) and its narrow counterpart (low).
//
// A CTA takes 128 columns of the long rows and one item of the plan (an adapter's tokens, or a
// piece of a long adapter's), 32 tokens at a time; the matrix pipe sums over the 32 tokens, and
// the sums of the blocks are added in fp32 outside it: the pipe truncates what it adds, which over
// a thousand tokens cost 5e-6 of the result instead of 1e-6.  low is held in three bf16 parts beside
// bf16 rows (all its bits; two left 2.4e-6 of a gradient), in two tf32 parts beside others.  Both
// gradients are one launch (a launch after the other took 10 us more for 77 tokens).  Items that are
// pieces of one adapter write partial sums, which a second kernel adds in order.  77 tokens, 4096 and
// 4096 columns, rank 16: 9.8 us, latency; 4096 tokens of F32 rows of 4 adapters: 76 us, bound by the
// matrix pipe and by splitting the rows into tf32 parts.
#include <type_traits>

#include "adapt.cuh"
#include "kernels.h"

namespace hymoe {
namespace {

constexpr int kGradTok = 32;
constexpr int kGradStages = 3;

template <typename X, int RP>
struct GradTile {
    static constexpr bool kF32 = sizeof(X) == 4;
    static constexpr int kXRow = kF32 ? kAdGradCols * 4 + 16 : kAdGradCols * 2 + 16;
    static constexpr int kLRow = (RP + 4) * 4;
    static constexpr int kXBytes = kGradTok * kXRow;
    static constexpr int kLBytes = kGradTok * kLRow;
    static constexpr int kStage = kXBytes + kLBytes;
    static constexpr bool kParts = std::is_same<X, __nv_bfloat16>::value;  // 16-bit parts of low
    static constexpr int kPRow = ad_pad16(RP * 2);
    static constexpr int kPBytes = kGradTok * kPRow;  // one part of a block
    static constexpr int kSmem = kStage * kGradStages + (kParts ? 3 * kPBytes : 0);
};

template <typename X, int RP>
__global__ __launch_bounds__(kAdThreads) void grad_kernel(const __grid_constant__ AdaptGrad a0,
                                                           const __grid_constant__ AdaptGrad a1) {
    using L = GradTile<X, RP>;
    extern __shared__ __align__(128) char smem[];
    griddep_wait();
    griddep_launch_dependents();
    const AdaptGrad& a = blockIdx.z == 0 ? a0 : a1;
    if (a.g == nullptr || static_cast<int>(blockIdx.y) * kAdGradCols >= a.M || static_cast<int>(blockIdx.x) >= a.plan.n_lists[2]) return;
    const int4 item = a.plan.items[blockIdx.x];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int m0 = blockIdx.y * kAdGradCols;
    const int n_blk = (item.z + kGradTok - 1) / kGradTok;

    constexpr int P = 16 / static_cast<int>(sizeof(X));
    constexpr int kXPieces = kAdGradCols / P, kXIter = kGradTok * kXPieces / kAdThreads;
    const int xc = tid % kXPieces, xr0 = tid / kXPieces;
    auto load = [&](int stage, int blk) {
        char* xs = smem + stage * L::kStage;
        char* ls = xs + L::kXBytes;
        const int r0 = blk * kGradTok;
#pragma unroll
        for (int i = 0; i < kXIter; ++i) {
            const int r = xr0 + i * (kAdThreads / kXPieces), m = m0 + xc * P;
            const int n = r0 + r < item.z ? a.M - m : 0;
            const char* src = static_cast<const char*>(a.x);
            if (n > 0) src += (static_cast<size_t>(__ldg(a.plan.perm + item.y + r0 + r)) * a.ldx + m) * sizeof(X);
            ad_copy_piece<sizeof(X)>(xs + r * L::kXRow + xc * 16, src, n, a.vec_x);
        }
        constexpr int kLPieces = RP / 4;
#pragma unroll
        for (int i = 0; i < kGradTok * kLPieces / kAdThreads; ++i) {
            const int p = tid + i * kAdThreads, r = p / kLPieces, c = p % kLPieces;
            const bool ok = r0 + r < item.z;
            cp_async16_part(ls + r * L::kLRow + c * 16,
                            a.low + static_cast<size_t>(ok ? item.y + r0 + r : 0) * RP + c * 4, ok ? 16 : 0);
        }
    };

    float sum[2][RP / 8][4];  // this warp's 32 columns m x RP
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < RP / 8; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[i][j][q] = 0.f;

#pragma unroll
    for (int s = 0; s < kGradStages - 1; ++s) {
        if (s < n_blk) load(s, s);
        cp_async_commit();
    }
    for (int blk = 0; blk < n_blk; ++blk) {
        const int stage = blk % kGradStages;
        cp_async_wait<kGradStages - 2>();
        __syncthreads();
        const int nxt = blk + kGradStages - 1;
        if (nxt < n_blk) load(nxt % kGradStages, nxt);
        cp_async_commit();
        const char* xs = smem + stage * L::kStage;
        const float* ls = reinterpret_cast<const float*>(xs + L::kXBytes);
        float acc[2][RP / 8][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < RP / 8; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][j][q] = 0.f;
        if constexpr (L::kParts) {
            char* ps = smem + kGradStages * L::kStage;
#pragma unroll
            for (int i = 0; i < kGradTok * RP / 4 / kAdThreads; ++i) {
                const int p = tid + i * kAdThreads, r = p / (RP / 4), c = p % (RP / 4) * 4;
                float4 v = *reinterpret_cast<const float4*>(ls + r * (RP + 4) + c);
#pragma unroll
                for (int part = 0; part < 3; ++part) {
                    const uint32_t h0 = AdType<X>::pack(v.x, v.y), h1 = AdType<X>::pack(v.z, v.w);
                    const float2 b0 = AdType<X>::unpack(h0), b1 = AdType<X>::unpack(h1);
                    *reinterpret_cast<uint2*>(ps + part * L::kPBytes + r * L::kPRow + c * 2) = make_uint2(h0, h1);
                    v = make_float4(v.x - b0.x, v.y - b0.y, v.z - b1.x, v.w - b1.y);
                }
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < kGradTok / 16; ++kk) {
                uint32_t af[2][4];  // X^T: rows m, k = tokens
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    ldsm4_t(af[i], smem_u32(xs) + (kk * 16 + (lane >> 4) * 8 + (lane & 7)) * L::kXRow +
                                       (warp * 32 + i * 16 + (lane >> 3 & 1) * 8) * 2);
#pragma unroll
                for (int j = 0; j < RP / 16; ++j)
#pragma unroll
                    for (int part = 2; part >= 0; --part) {
                        uint32_t bf[4];
                        ldsm4_t(bf, smem_u32(ps) + part * L::kPBytes + (kk * 16 + (lane & 15)) * L::kPRow + (j * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            AdType<X>::mma(acc[i][2 * j], af[i], bf[0], bf[1]);
                            AdType<X>::mma(acc[i][2 * j + 1], af[i], bf[2], bf[3]);
                        }
                    }
            }
        } else {
#pragma unroll
        for (int kk = 0; kk < kGradTok / 16; ++kk) {
            // A: X^T, rows m, k = tokens; v[i][h][q]: tokens 8h + 2t, 2t + 1 of column m = 16 i + g + 8 q
            float2 v[2][2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (!L::kF32) {
                    uint32_t r[4];
                    // blocks (k 0-7, m 0-7), (k 0-7, m 8-15), (k 8-15, m 0-7), (k 8-15, m 8-15)
                    ldsm4_t(r, smem_u32(xs) + (kk * 16 + (lane >> 4) * 8 + (lane & 7)) * L::kXRow +
                                   (warp * 32 + i * 16 + (lane >> 3 & 1) * 8) * 2);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int q = 0; q < 2; ++q) v[i][h][q] = AdType<X>::unpack(r[2 * h + q]);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const char* at = xs + (kk * 16 + h * 8 + 2 * t) * L::kXRow + (warp * 32 + i * 16 + g + 8 * q) * 4;
                            v[i][h][q] = make_float2(*reinterpret_cast<const float*>(at),
                                                     *reinterpret_cast<const float*>(at + L::kXRow));
                        }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t ah[2][4], al[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        split_tf32(v[i][h][q].x, ah[i][q], al[i][q]);
                        split_tf32(v[i][h][q].y, ah[i][2 + q], al[i][2 + q]);
                    }
#pragma unroll
                for (int j = 0; j < RP / 8; ++j) {
                    const float* lp = ls + (kk * 16 + h * 8 + 2 * t) * (RP + 4) + j * 8 + g;
                    uint32_t bh[2], bl[2];
                    split_tf32(lp[0], bh[0], bl[0]);
                    split_tf32(lp[RP + 4], bh[1], bl[1]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (L::kF32) mma_tf32(acc[i][j], al[i], bh[0], bh[1]);
                        mma_tf32(acc[i][j], ah[i], bl[0], bl[1]);
                        mma_tf32(acc[i][j], ah[i], bh[0], bh[1]);
                    }
                }
            }
        }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < RP / 8; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[i][j][q] += acc[i][j][q];
    }
    cp_async_wait<0>();
    float* out = item.w >= 0 ? a.part + static_cast<size_t>(item.w) * a.M * a.R : a.g + static_cast<size_t>(item.x) * a.M * a.R;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < RP / 8; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int m = m0 + warp * 32 + i * 16 + g + 8 * (q >> 1), c = j * 8 + 2 * t + (q & 1);
                if (m < a.M && c < a.R) out[static_cast<size_t>(m) * a.gm + static_cast<size_t>(c) * a.gj] = sum[i][j][q];
            }
}

// The pieces of adapters that have several, added in order.  Grid (elements, adapters, gradients).
__global__ __launch_bounds__(256) void grad_join_kernel(const __grid_constant__ AdaptGrad a0, const __grid_constant__ AdaptGrad a1) {
    griddep_wait();
    griddep_launch_dependents();
    const AdaptGrad& a = blockIdx.z == 0 ? a0 : a1;
    if (a.g == nullptr) return;
    const int ad = blockIdx.y, lo = a.plan.pieces[ad], hi = a.plan.pieces[ad + 1];
    if (hi - lo < 2) return;
    const size_t size = static_cast<size_t>(a.M) * a.R, at = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    const size_t step = static_cast<size_t>(gridDim.x) * 256;
    if (size % 4 == 0 && (reinterpret_cast<uintptr_t>(a.g) & 15) == 0) {
        for (size_t i = at; i < size / 4; i += step) {
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int p = lo; p < hi; ++p) {
                const float4 v = reinterpret_cast<const float4*>(a.part + static_cast<size_t>(a.plan.items[p].w) * size)[i];
                s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
            }
            reinterpret_cast<float4*>(a.g + ad * size)[i] = s;
        }
        return;
    }
    for (size_t i = at; i < size; i += step) {
        float s = 0.f;
        for (int p = lo; p < hi; ++p) s += a.part[static_cast<size_t>(a.plan.items[p].w) * size + i];
        a.g[ad * size + i] = s;
    }
}

template <typename X, int RP>
cudaError_t launch_t(const AdaptGrad& a, const AdaptGrad& b, cudaStream_t st) {
    using L = GradTile<X, RP>;
    auto kern = grad_kernel<X, RP>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    const int ma = a.g ? a.M : 0, mb = b.g ? b.M : 0;
    return launch_kernel(true, kern, dim3(a.plan.max_items, ((ma > mb ? ma : mb) + kAdGradCols - 1) / kAdGradCols, b.g ? 2 : 1),
                         dim3(kAdThreads), L::kSmem, st, a, b);
}

template <typename X>
cudaError_t launch_x(const AdaptGrad& a, const AdaptGrad& b, cudaStream_t st) {
    switch (adapt_rp(a.R)) {
        case 16: return launch_t<X, 16>(a, b, st);
        case 32: return launch_t<X, 32>(a, b, st);
        case 64: return launch_t<X, 64>(a, b, st);
        default: return launch_t<X, 128>(a, b, st);
    }
}

}  // namespace

cudaError_t launch_adapt_join(const AdaptGrad& a, const AdaptGrad& b, cudaStream_t st) {
    const size_t ma = a.g ? static_cast<size_t>(a.M) * a.R : 0, mb = b.g ? static_cast<size_t>(b.M) * b.R : 0;
    const size_t blk = ((ma > mb ? ma : mb) + 1023) / 1024;
    return launch_kernel(true, grad_join_kernel, dim3(static_cast<unsigned>(blk < 512 ? blk : 512), a.n, 2), dim3(256), 0, st, a, b);
}

cudaError_t launch_adapt_grad(const AdaptGrad& a, const AdaptGrad& b, int type_x, cudaStream_t st) {
    if (type_x == HYMOE_TYPE_F32) return launch_x<float>(a, b, st);
    if (type_x == HYMOE_TYPE_F16) return launch_x<__half>(a, b, st);
    return launch_x<__nv_bfloat16>(a, b, st);
}

}  // namespace hymoe
