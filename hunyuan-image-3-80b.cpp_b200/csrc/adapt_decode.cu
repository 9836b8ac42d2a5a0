// adapt_decode.cu — hymoe_adapt for a few tokens, in one launch without a plan or a workspace.
//
// One cluster of CTAs per token, each thread block over a part of the long dimensions:
//   1. its part of the columns of A_a x: four rank rows at a time per warp, fp32 sums,
//   2. the CTAs' partial results [rank] are added in distributed shared memory, in their order,
//   3. its part of the rows of B_a: one output per thread, added to the base.
// The weights of step 3 are asked for (into L2) before step 1 begins.  Tokens of the same adapter
// read its weights from L2 again.  Four CTAs fit an SM, so 64 tokens' 512 run at once (with three,
// rank 32 went from 9.1 us at 48 tokens to 16.2 at 64).  Bound by the latency of its two passes over the weights
// (about 5 us with the launch) up to some 20 MB of distinct adapters, then by reading them:
// 64 tokens of 32 adapters, 4096 to 6144, rank 32 (21 MB), 10.5 us with them in L2, 15 without.
#include "adapt.cuh"
#include "kernels.h"

namespace hymoe {
namespace {

constexpr int kDecThreads = 256, kDecWarps = kDecThreads / 32;
constexpr int kDecRows = 4;  // rank rows per warp and pass

__device__ __forceinline__ float dec_f(float v) { return v; }
__device__ __forceinline__ float dec_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float dec_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void dec_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void dec_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void dec_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Eight consecutive values from an address aligned to 16 bytes.
__device__ __forceinline__ void dec_load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void dec_unpack8(uint4 q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = AdType<T>::unpack(w[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename T>
__device__ __forceinline__ void dec_load8(const T* p, float (&v)[8]) {
    dec_unpack8<T>(*reinterpret_cast<const uint4*>(p), v);
}

template <typename X, typename W, typename Y>
__global__ __launch_bounds__(kDecThreads, 4) void decode_adapt_kernel(const __grid_constant__ AdaptDecode d) {
    __shared__ float part[kDecWarps][HYMOE_ADAPT_MAX_RANK];
    __shared__ float mine[HYMOE_ADAPT_MAX_RANK];    // this CTA's partial result, read by the others
    __shared__ __align__(16) float low[HYMOE_ADAPT_MAX_RANK];
    const int C = d.ctas, t = blockIdx.x / C, rank = blockIdx.x % C;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int a = d.ids != nullptr ? __ldg(d.ids + t) : 0;
    const bool has = a >= 0 && a < d.n;
    if (!has && d.in_place) return;  // the whole cluster: nothing to add
    const int R = d.R, K = d.K, N = d.N;
    const X* x = static_cast<const X*>(d.x) + static_cast<size_t>(t) * d.ldx;
    const W* wa = static_cast<const W*>(d.a) + static_cast<size_t>(has ? a : 0) * R * K;
    const W* wb = static_cast<const W*>(d.b) + static_cast<size_t>(has ? a : 0) * N * R;
    const int n_per = (N + C - 1) / C, n_lo = min(N, rank * n_per), n_hi = min(N, n_lo + n_per);
    if (has) {
        // step 3's rows into L2
        const char* p0 = reinterpret_cast<const char*>(wb + static_cast<size_t>(n_lo) * R);
        const size_t bytes = static_cast<size_t>(n_hi - n_lo) * R * sizeof(W);
        for (size_t o = static_cast<size_t>(tid) * 128; o < bytes; o += kDecThreads * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(p0 + o));
        // step 1: columns [k_lo, k_hi) in whole pieces of 8
        const int k_per = ((K + C - 1) / C + 7) / 8 * 8, k_lo = min(K, rank * k_per), k_hi = min(K, k_lo + k_per);
        const int groups = (R + kDecRows - 1) / kDecRows;
        // few rank rows: the warps share the columns too
        const int kparts = groups >= kDecWarps ? 1 : kDecWarps / groups, gstep = groups >= kDecWarps ? kDecWarps : groups;
        const int kp = warp / gstep;
        if (kp < kparts) {
            for (int g = warp % gstep; g < groups; g += gstep) {
                float s[kDecRows] = {};
                const W* row[kDecRows];
#pragma unroll
                for (int i = 0; i < kDecRows; ++i) row[i] = wa + static_cast<size_t>(min(g * kDecRows + i, R - 1)) * K;
                if (d.vec_x && d.vec_a) {  // (K and k_lo .. k_hi are whole pieces of 8 then)
#pragma unroll 2
                    for (int k = k_lo + (kp * 32 + lane) * 8; k + 8 <= k_hi; k += kparts * 256) {
                        float xv[8];
                        dec_load8(x + k, xv);
#pragma unroll
                        for (int i = 0; i < kDecRows; ++i) {
                            float wv[8];
                            dec_load8(row[i] + k, wv);
#pragma unroll
                            for (int j = 0; j < 8; ++j) s[i] = fmaf(xv[j], wv[j], s[i]);
                        }
                    }
                } else {
                    for (int k = k_lo + kp * 32 + lane; k < k_hi; k += kparts * 32) {
                        const float xv = dec_f(x[k]);
#pragma unroll
                        for (int i = 0; i < kDecRows; ++i) s[i] = fmaf(xv, dec_f(row[i][k]), s[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < kDecRows; ++i) {
#pragma unroll
                    for (int o = 16; o; o >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
                    if (lane == 0 && g * kDecRows + i < R) part[kp][g * kDecRows + i] = s[i];
                }
            }
        }
        __syncthreads();
        for (int j = tid; j < R; j += kDecThreads) {
            float s = 0.f;
            for (int q = 0; q < kparts; ++q) s += part[q][j];
            mine[j] = s;
        }
        cluster_sync();
        const float f = d.scale != nullptr ? __ldg(d.scale + a) : 1.f;
        for (int j = tid; j < R; j += kDecThreads) {
            float s = 0.f;
            for (int q = 0; q < C; ++q) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(mine + j, q)) : "memory");
                s += v;
            }
            low[j] = s * f;
        }
        __syncthreads();
    }
    const Y* base = static_cast<const Y*>(d.base);
    Y* out = static_cast<Y*>(d.out) + static_cast<size_t>(t) * d.ldo;
    for (int o = n_lo + tid; o < n_hi; o += kDecThreads) {
        float s = 0.f;
        if (has) {
            const W* row = wb + static_cast<size_t>(o) * R;
            if (d.vec_b) {
#pragma unroll 4
                for (int j = 0; j < R; j += 8) {
                    float wv[8];
                    dec_load8(row + j, wv);
                    const float4 l0 = *reinterpret_cast<const float4*>(low + j), l1 = *reinterpret_cast<const float4*>(low + j + 4);
                    s = fmaf(l0.x, wv[0], s);
                    s = fmaf(l0.y, wv[1], s);
                    s = fmaf(l0.z, wv[2], s);
                    s = fmaf(l0.w, wv[3], s);
                    s = fmaf(l1.x, wv[4], s);
                    s = fmaf(l1.y, wv[5], s);
                    s = fmaf(l1.z, wv[6], s);
                    s = fmaf(l1.w, wv[7], s);
                }
            } else {
                for (int j = 0; j < R; ++j) s = fmaf(low[j], dec_f(row[j]), s);
            }
        }
        Y v;
        dec_store(&v, 0.f);
        if (base != nullptr) v = base[static_cast<size_t>(t) * d.ldb + o];
        if (has) dec_store(&v, s + dec_f(v));  // else the base's value as it is (0 + -0 would be 0)
        out[o] = v;
    }
    if (has) cluster_sync();  // no CTA leaves while another reads its partial result
}

template <typename X, typename W, typename Y>
cudaError_t launch_t(const AdaptDecode& d, int T, cudaStream_t st) {
    auto kern = decode_adapt_kernel<X, W, Y>;
    if (d.ctas > 8) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(T) * d.ctas);
    cfg.blockDim = dim3(kDecThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = d.ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, d);
}

template <typename W>
cudaError_t launch_w(const AdaptDecode& d, bool x_f32, bool y_f32, int T, cudaStream_t st) {
    if (x_f32) return y_f32 ? launch_t<float, W, float>(d, T, st) : launch_t<float, W, W>(d, T, st);
    return y_f32 ? launch_t<W, W, float>(d, T, st) : launch_t<W, W, W>(d, T, st);
}

}  // namespace

cudaError_t launch_adapt_decode(const AdaptDecode& d, int type_x, int type_w, int type_y, int T, cudaStream_t st) {
    const bool xf = type_x == HYMOE_TYPE_F32, yf = type_y == HYMOE_TYPE_F32;
    return type_w == HYMOE_TYPE_F16 ? launch_w<__half>(d, xf, yf, T, st) : launch_w<__nv_bfloat16>(d, xf, yf, T, st);
}

}  // namespace hymoe
