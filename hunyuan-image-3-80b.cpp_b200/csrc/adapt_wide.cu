// adapt_wide.cu — the adapters' wide product with its epilogue:
//   out[token of row] = base[token of row] + W_a low[row].
//
// A CTA takes a tile of 64 sorted rows of one adapter and a run of columns, 64 at a time: the
// weights and the base's rows of the next columns are copied while the present ones are multiplied;
// the result is added to the base in its shared-memory tile, rounded once, and leaves in rows of
// whole 16-byte pieces.  The intermediate rows are read once per CTA into registers, as 16-bit parts
// (two for a 16-bit result, enough to hold fp32 for an fp32 one), so the products run on the
// 16-bit matrix pipe.  Bound by reading and writing out's rows: 77 tokens to 4096 columns, rank 16,
// take 5 us; 8192 bf16 rows to 6144 off 16-byte boundaries, rank 64, 261 us, by their copies of 2 bytes
// (300 with the weights off them too; 124 with the weights alone).
#include "adapt.cuh"
#include "kernels.h"

namespace hymoe {
namespace {

constexpr int kWideCols = 64;
constexpr int kWideStages = 3;

template <typename Y, int RP, bool TRANS>
struct WideTile {
    static constexpr bool kF32 = sizeof(Y) == 4;
    static constexpr int kYRow = kF32 ? kWideCols * 4 + 32 : kWideCols * 2 + 16;
    static constexpr int kWRow = TRANS ? kWideCols * 2 + 16 : ad_pad16(RP * 2);
    static constexpr int kYBytes = kAdRows * kYRow;
    static constexpr int kWBytes = (TRANS ? RP : kWideCols) * kWRow;
    static constexpr int kStage = kYBytes + kWBytes;
    static constexpr int kSmem = kStage * kWideStages;
    static constexpr int kPerSm = 226 * 1024 / (kSmem + 1024) < 4 ? 226 * 1024 / (kSmem + 1024) : 4;  // CTAs on an SM
};

// The 16-bit parts of a pair of fp32 values; bf16 has fp32's range, fp16 rows are scaled before.
template <typename W, int NP>
__device__ __forceinline__ void split16(float x, float y, uint32_t (&p)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        p[i] = AdType<W>::pack(x, y);
        const float2 b = AdType<W>::unpack(p[i]);
        x = part_rest(x, b.x);
        y = part_rest(y, b.y);
    }
}

template <typename Y, typename W, int RP, bool TRANS>
__global__ __launch_bounds__(kAdThreads, WideTile<Y, RP, TRANS>::kPerSm) void wide_kernel(
    const __grid_constant__ AdaptWide a, int cols_per_cta) {
    using L = WideTile<Y, RP, TRANS>;
    constexpr bool kScaled = AdType<W>::kScaled;
    constexpr int NP = L::kF32 && !kScaled ? 3 : 2;  // bf16 parts of 8 bits, fp16 parts of 11
    extern __shared__ __align__(128) char smem[];
    griddep_wait();
    griddep_launch_dependents();
    const int4 tile = ad_part_tile(a.plan, blockIdx.x);
    if (tile.z == 0) return;
    const bool mul = tile.x >= 0;
    if (!mul && a.in_place) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int c_lo = blockIdx.y * cols_per_cta, c_hi = min(a.N, c_lo + cols_per_cta);
    const int n_blk = (c_hi - c_lo + kWideCols - 1) / kWideCols;

    constexpr int P = 16 / static_cast<int>(sizeof(Y));
    constexpr int kYPieces = kWideCols / P;                // pieces of a row
    constexpr int kYRows = 32 / kYPieces;                  // rows that a warp covers at once
    constexpr int kYIter = 16 / kYRows;                    // a warp loads and stores its own 16 rows
    const int yc = lane % kYPieces, yr0 = warp * 16 + lane / kYPieces;
    const char* bp[kYIter];  // this thread's pieces of the base's and the result's rows, in column 0
    char* op[kYIter];
    int yn[kYIter];          // bytes of a whole piece: none where the row does not exist
#pragma unroll
    for (int i = 0; i < kYIter; ++i) {
        const int r = yr0 + i * kYRows;
        const bool ok = r < tile.z;
        const int tok = ok ? __ldg(a.plan.perm + tile.y + r) : 0;
        yn[i] = ok ? 16 : 0;
        bp[i] = static_cast<const char*>(a.base) + (static_cast<size_t>(tok) * a.ldb + (ok ? yc * P : 0)) * sizeof(Y);
        op[i] = static_cast<char*>(a.out) + (static_cast<size_t>(tok) * a.ldo + yc * P) * sizeof(Y);
    }
    constexpr int kWPieces = TRANS ? kWideCols / 8 : RP / 8, kWAll = (TRANS ? RP : kWideCols) * kWPieces;
    constexpr int kWIter = kWAll / kAdThreads;
    static_assert(kWAll % kAdThreads == 0, "whole rounds of pieces");
    const char* wbase = static_cast<const char*>(a.w) + static_cast<size_t>(mul ? tile.x : 0) * a.R * a.N * 2;
    const char* wp[kWIter];
    int wn[kWIter];
#pragma unroll
    for (int i = 0; i < kWIter; ++i) {
        const int p = tid + i * kAdThreads, r = p / kWPieces, c = p % kWPieces * 8;
        const bool ok = TRANS ? r < a.R : c < a.R;  // trans: row = rank, columns = out; else row = out, columns = rank
        wp[i] = ok ? wbase + (static_cast<size_t>(r) * (TRANS ? a.N : a.R) + c) * 2 : wbase;
        wn[i] = !ok ? 0 : TRANS ? 16 : min(16, (a.R - c) * 2);
    }
    auto load = [&](int stage, int blk) {
        char* ys = smem + stage * L::kStage;
        char* ws = ys + L::kYBytes;
        const int c0 = c_lo + blk * kWideCols;
        const bool whole = c0 + kWideCols <= c_hi;
        if (a.base != nullptr) {
            if (whole && a.vec_b) {
#pragma unroll
                for (int i = 0; i < kYIter; ++i)
                    cp_async16_part(ys + (yr0 + i * kYRows) * L::kYRow + yc * 16, yn[i] ? bp[i] + static_cast<size_t>(c0) * sizeof(Y) : bp[i], yn[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kYIter; ++i) {
                    const int n = yn[i] ? c_hi - (c0 + yc * P) : 0;
                    ad_copy_piece<sizeof(Y)>(ys + (yr0 + i * kYRows) * L::kYRow + yc * 16,
                                             n > 0 ? bp[i] + static_cast<size_t>(c0) * sizeof(Y) : static_cast<const char*>(a.base), n, a.vec_b);
                }
            }
        }
        if (mul) {
            const size_t adv = static_cast<size_t>(c0) * (TRANS ? 1 : a.R) * 2;
            if (whole && a.vec_w) {
#pragma unroll
                for (int i = 0; i < kWIter; ++i) {
                    const int p = tid + i * kAdThreads;
                    cp_async16_part(ws + p / kWPieces * L::kWRow + p % kWPieces * 16, wn[i] ? wp[i] + adv : wbase, wn[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kWIter; ++i) {
                    const int p = tid + i * kAdThreads, r = p / kWPieces, c = p % kWPieces;
                    const int n = wn[i] == 0 ? 0 : TRANS ? a.N - (c0 + c * 8) : (c0 + r < a.N ? a.R - c * 8 : 0);
                    ad_copy_piece<2>(ws + r * L::kWRow + c * 16, n > 0 ? wp[i] + adv : wbase, n, a.vec_w);
                }
            }
        }
    };
#pragma unroll
    for (int s = 0; s < kWideStages - 1; ++s) {
        if (s < n_blk) load(s, s);
        cp_async_commit();
    }

    // this warp's 16 rows of low, as fragments of NP 16-bit parts
    uint32_t af[RP / 16][NP][4];
    float back[2] = {1.f, 1.f};
    if (mul) {
        float2 v[RP / 16][4];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int r = warp * 16 + g + 8 * q;
            const float* row = a.low + static_cast<size_t>(tile.y + min(r, tile.z - 1)) * RP;
#pragma unroll
            for (int k = 0; k < RP / 16; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    v[k][2 * h + q] = r < tile.z ? *reinterpret_cast<const float2*>(row + k * 16 + h * 8 + 2 * t) : make_float2(0.f, 0.f);
        }
        if constexpr (kScaled) {
            // fp16 parts: every row times a power of two that brings its largest value into [1, 2)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float m = 0.f;
#pragma unroll
                for (int k = 0; k < RP / 16; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) m = fmaxf(m, fmaxf(fabsf(v[k][2 * h + q].x), fabsf(v[k][2 * h + q].y)));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const int e = max(1, min(253, static_cast<int>(__float_as_uint(m) >> 23)));
                const float f = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
                back[q] = __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
                for (int k = 0; k < RP / 16; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        v[k][2 * h + q].x *= f;
                        v[k][2 * h + q].y *= f;
                    }
            }
        }
#pragma unroll
        for (int k = 0; k < RP / 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t p[NP];
                split16<W, NP>(v[k][i].x, v[k][i].y, p);
#pragma unroll
                for (int j = 0; j < NP; ++j) af[k][j][i] = p[j];
            }
    }

    for (int blk = 0; blk < n_blk; ++blk) {
        const int stage = blk % kWideStages;
        cp_async_wait<kWideStages - 2>();
        __syncthreads();
        const int nxt = blk + kWideStages - 1;
        if (nxt < n_blk) load(nxt % kWideStages, nxt);
        cp_async_commit();
        char* ys = smem + stage * L::kStage;
        if (mul || a.base == nullptr) {
            float acc[kWideCols / 8][4];
#pragma unroll
            for (int i = 0; i < kWideCols / 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
            if (mul) {
                const uint32_t wa = smem_u32(ys + L::kYBytes);
#pragma unroll
                for (int k = 0; k < RP / 16; ++k) {
#pragma unroll
                    for (int j = 0; j < kWideCols / 16; ++j) {
                        uint32_t bf[4];
                        if (TRANS)
                            ldsm4_t(bf, wa + (k * 16 + (lane & 15)) * L::kWRow + (j * 16 + (lane >> 4) * 8) * 2);
                        else
                            ldsm4(bf, wa + (j * 16 + (lane >> 4) * 8 + (lane & 7)) * L::kWRow + (k * 16 + (lane >> 3 & 1) * 8) * 2);
#pragma unroll
                        for (int p = NP - 1; p >= 0; --p) {
                            AdType<W>::mma(acc[2 * j], af[k][p], bf[0], bf[1]);
                            AdType<W>::mma(acc[2 * j + 1], af[k][p], bf[2], bf[3]);
                        }
                    }
                }
            }
            // base + result, in the base's tile
#pragma unroll
            for (int j = 0; j < kWideCols / 8; ++j)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    char* at = ys + (warp * 16 + g + 8 * q) * L::kYRow + (j * 8 + 2 * t) * static_cast<int>(sizeof(Y));
                    float x = acc[j][2 * q], y = acc[j][2 * q + 1];
                    if (kScaled) {
                        x *= back[q];
                        y *= back[q];
                    }
                    if constexpr (L::kF32) {
                        if (a.base != nullptr) {
                            const float2 b = *reinterpret_cast<const float2*>(at);
                            x += b.x;
                            y += b.y;
                        }
                        *reinterpret_cast<float2*>(at) = make_float2(x, y);
                    } else {
                        if (a.base != nullptr) {
                            const float2 b = AdType<W>::unpack(*reinterpret_cast<const uint32_t*>(at));
                            x += b.x;
                            y += b.y;
                        }
                        *reinterpret_cast<uint32_t*>(at) = AdType<W>::pack(x, y);
                    }
                }
            __syncwarp();
        }
        const int c0 = c_lo + blk * kWideCols;
        if (c0 + kWideCols <= c_hi && a.vec_o) {
#pragma unroll
            for (int i = 0; i < kYIter; ++i)
                if (yn[i])
                    *reinterpret_cast<uint4*>(op[i] + static_cast<size_t>(c0) * sizeof(Y)) =
                        *reinterpret_cast<const uint4*>(ys + (yr0 + i * kYRows) * L::kYRow + yc * 16);
        } else {
#pragma unroll
            for (int i = 0; i < kYIter; ++i) {
                const Y* src = reinterpret_cast<const Y*>(ys + (yr0 + i * kYRows) * L::kYRow + yc * 16);
                Y* dst = reinterpret_cast<Y*>(op[i]) + c0;
                if (yn[i])
                    for (int j = 0; j < P && c0 + yc * P + j < c_hi; ++j) dst[j] = src[j];
            }
        }
    }
    cp_async_wait<0>();
}

template <typename Y, typename W, int RP, bool TRANS>
cudaError_t launch_t(const AdaptWide& a, int n_sms, cudaStream_t st) {
    using L = WideTile<Y, RP, TRANS>;
    auto kern = wide_kernel<Y, W, RP, TRANS>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    // runs of columns: as many as fill the GPU once
    const int blks = (a.N + kWideCols - 1) / kWideCols, tiles = a.plan.max_tiles * (a.plan.tile_rows / kAdRows);
    const int fit = L::kPerSm * n_sms / tiles;
    const int parts = fit < 1 ? 1 : fit < blks ? fit : blks;
    const int cols = (blks + parts - 1) / parts * kWideCols;
    return launch_kernel(true, kern, dim3(tiles, (a.N + cols - 1) / cols), dim3(kAdThreads), L::kSmem, st, a, cols);
}

template <typename Y, typename W>
cudaError_t launch_y(const AdaptWide& a, bool trans, int n_sms, cudaStream_t st) {
    switch (adapt_rp(a.R)) {
        case 16: return trans ? launch_t<Y, W, 16, true>(a, n_sms, st) : launch_t<Y, W, 16, false>(a, n_sms, st);
        case 32: return trans ? launch_t<Y, W, 32, true>(a, n_sms, st) : launch_t<Y, W, 32, false>(a, n_sms, st);
        case 64: return trans ? launch_t<Y, W, 64, true>(a, n_sms, st) : launch_t<Y, W, 64, false>(a, n_sms, st);
        default: return trans ? launch_t<Y, W, 128, true>(a, n_sms, st) : launch_t<Y, W, 128, false>(a, n_sms, st);
    }
}

}  // namespace

cudaError_t launch_adapt_wide(const AdaptWide& a, int type_y, int type_w, bool trans, int n_sms, cudaStream_t st) {
    if (type_w == HYMOE_TYPE_F16)
        return type_y == HYMOE_TYPE_F32 ? launch_y<float, __half>(a, trans, n_sms, st)
                                        : launch_y<__half, __half>(a, trans, n_sms, st);
    return type_y == HYMOE_TYPE_F32 ? launch_y<float, __nv_bfloat16>(a, trans, n_sms, st)
                                    : launch_y<__nv_bfloat16, __nv_bfloat16>(a, trans, n_sms, st);
}

}  // namespace hymoe
