// adapt_tc.cuh — what the adapters' tcgen05 kernels share: matrix descriptors for both operand
// orders and the tensor maps.
//
// Operand tiles are 128-byte rows in the 128B swizzle.  K-major: a row is one M (or N) index, 64
// values along K; rows of 8 are 1024 bytes apart.  MN-major: a row is one K index, 64 values along
// M (or N); blocks of 64 along M are `block` bytes apart, groups of 8 K indexes 1024 bytes.
//
// Token rows come in sorted order.  Where a tile's tokens are consecutive (a request's) tiled loads
// take them; else warps copy them.
#pragma once

#include <type_traits>

#include "adapt.cuh"
#include "kernels.h"

namespace hymoe {

constexpr int kTcRows = 128;  // token rows of a tile

// TMA maps of one adapter product, made on the host for every call.
struct AdaptMaps {
    CUtensorMap rows;    // token rows, box {128 bytes, tile rows}
    CUtensorMap w;       // weights [n][rows][columns], box {64 columns, rows of a stage, 1}
};
cudaError_t launch_adapt_low_tc(const AdaptMaps& maps, const AdaptLow& a, int type_w, bool trans, int n_sms, cudaStream_t st);
cudaError_t launch_adapt_wide_tc(const AdaptMaps& maps, const AdaptWide& a, int type_y, int type_w, bool trans, int n_sms,
                                 cudaStream_t st);

// 16-bit values of a row of low in three parts: the first, in whole panels of 64, and the other two
// from adapt_rest on.
__host__ __device__ constexpr int adapt_rest(int rp) { return rp < 64 ? 64 : rp; }
__host__ __device__ constexpr int adapt_parts(int rp) { return adapt_rest(rp) + (rp < 32 ? 64 : 2 * rp); }

// Both gradients of a call (either may be absent: g[i].g == nullptr; plan, R and n are always set).
struct AdaptGradPair {
    AdaptGrad g[2];
    CUtensorMap rows[2];  // their long rows, box {64 values, 64 rows}
    CUtensorMap lows[2];  // low in parts, the same box
    void* parts[2];       // [T, adapt_parts(RP)] 16-bit values: low's parts, in sorted order
    int groups0;          // column groups of the first (set by the launcher)
};
cudaError_t launch_adapt_grad_tc(AdaptGradPair p, int type_w, cudaStream_t st);

#ifdef __CUDACC__

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// Whether a tile's tokens (ascending) are consecutive, and the first one.
__device__ __forceinline__ bool tile_run(const AdaptPlan& p, const int4& tile, int* first) {
    *first = __ldg(p.perm + tile.y);
    return __ldg(p.perm + tile.y + tile.z - 1) - *first == tile.z - 1;
}

// Arrives on `bar` (counted in its expected arrivals) when this thread's cp.async copies so far have
// landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// All threads of the cluster, in two halves.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// 32 lanes x 16 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// The same lanes and columns written.
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MN-major operand in the 128B swizzle (see above).
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t saddr, uint32_t block) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(block >> 4) << 16;        // leading offset: next 64 values along M or N
    d |= static_cast<uint64_t>(1024 >> 4) << 32;         // stride offset: next 8 K indexes
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// Instruction descriptor, kind::f16 with W operands: fp32 D, M = 128; mn_a / mn_b: that operand is
// MN-major.
template <typename W>
__host__ __device__ constexpr uint32_t ad_idesc(int N, bool mn_a, bool mn_b) {
    const uint32_t f = std::is_same<W, __nv_bfloat16>::value ? 1u : 0u;
    return idesc_f16_f32(128, N) | (f << 7) | (f << 10) | (mn_a ? 1u << 15 : 0u) | (mn_b ? 1u << 16 : 0u);
}

#endif

}  // namespace hymoe
