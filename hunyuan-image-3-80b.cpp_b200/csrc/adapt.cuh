// adapt.cuh — shared by the adapter kernels (adapt.cu, adapt_low.cu, adapt_wide.cu,
// adapt_grad.cu): the plan's lists, shared-memory tiles, mma.sync wrappers and the splitting of
// fp32 operands.
//
// Tiles in shared memory have rows padded so that a row is an odd number of 16-byte pieces (fp32
// tiles read in 8-byte pairs: 32 bytes of padding): the eight rows of an ldmatrix, and the rows of
// a fragment access, fall into different banks.
//
// Fragment layouts are those of mma.sync (thread g = lane / 4, t = lane % 4).  An m16n8k16
// fragment of 16-bit values holds k = 2t, 2t+1 in one register; taken as the k = t and t + 4 of an
// m16n8k8 tf32 fragment on both operands, the same registers feed a tf32 product: the sum over k
// does not mind the order.  Every 16-bit value is exact in tf32, and an fp32 value is the sum of two
// tf32 parts to 2^-22.
#pragma once

#include "common.cuh"
#include "entry.h"

namespace hymoe {

constexpr int kAdRows = 64;         // token rows of a tile
constexpr int kAdThreads = 128;     // four warps of 16 rows
constexpr int kAdGradCols = 128;    // columns of a gradient tile

// Rank padded to the kernels' sizes.
__host__ __device__ constexpr int adapt_rp(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

// Tokens of one gradient item.  An adapter of up to twice the average length, and of up to a fifth of
// all tokens, stays whole (with fewer than ten adapters the fifth decides), as does one of up to 512
// tokens; a longer one is cut into pieces that run side by side (their sums are added in order by a
// second kernel), five where it has all the tokens, at most eight.
constexpr int kAdMinChunk = 512, kAdMaxPieces = 8;
__host__ __device__ constexpr int adapt_chunk(int T, int n) {
    const int avg = static_cast<int>(static_cast<int64_t>(T) * 2 / n), fifth = T / 5;
    int c = avg < fifth ? avg : fifth;
    const int least = (T + kAdMaxPieces - 1) / kAdMaxPieces;
    c = c < least ? least : c;
    c = c < kAdMinChunk ? kAdMinChunk : c;
    return (c + 63) / 64 * 64;
}

// CTAs that share a tile of the narrow product over K columns: as many as the `slots` of the GPU
// leave for each of `tiles` tiles, each with two blocks of 64 columns at least.
constexpr int kAdMaxSplits = 16;
constexpr int kAdMaxSlots = 640;  // CTAs that a GPU is taken to hold at most (four on each of 160 SMs)
__host__ __device__ constexpr int adapt_splits(int tiles, int K, int slots) {
    const int nk = (K + 63) / 64;
    int s = slots / tiles < nk / 2 ? slots / tiles : nk / 2;
    s = s < kAdMaxSplits ? s : kAdMaxSplits;
    return s < 1 ? 1 : s;
}

// Whether hymoe_adapt runs as clusters per token: the weights are read once per token, so up to 64
// tokens and fewer where the rank is high.
__host__ __device__ constexpr bool adapt_decodes(size_t T, int R) { return T <= 64 && T * adapt_rp(R) <= 4096; }

// What the plan kernel writes: tokens in the order of their adapters (stable; those without one
// last) and the work lists over that order.
struct AdaptPlan {
    int* perm;       // [T] token of each sorted row
    int4* tiles;     // {adapter or -1, first row, rows, 0} of at most tile_rows rows
    int4* items;     // gradients: {adapter, first row, rows, partial slot or -1}; every adapter has one
    int* pieces;     // gradients: [n + 1] first item of each adapter (items are adapter-major)
    int* err;        // DevErr bits of a bounded wait that expired: n_lists, or the caller's word
    int* n_lists;    // [0] status, [1] tiles, [2] items,
                     // [3] tiles that have an adapter (the first ones)
    int tile_rows;   // 64 or 128
    unsigned* amax;  // gradients of fp16 rows: [2 n] largest |low| of every adapter (bits), of dy's then of x's
    unsigned* counters;  // [max_tiles] (backward: twice) CTAs of a tile that have left their partial sums (0 between launches)
    int max_tiles, max_items;
    int spare_tiles; // of max_tiles, those for adapters' last, part-filled tiles
};

struct AdaptLow {      // low[row, j] = scale[a] * sum_k X[perm[row], k] W_a(j, k), rows in sorted order
    AdaptPlan plan;
    const void* x;
    size_t ldx;        // elements
    const void* w;     // [n] matrices of R x K (trans: K x R)
    const float* scale;
    float* low;        // [T, RP]
    float* part;       // [max_tiles * S] partial sums of 64 x RP
    unsigned* amax;    // [n] largest |low| of every adapter, or nullptr
    int K, R;
    int vec_x, vec_w;  // rows start on 16-byte boundaries
};
struct AdaptWide {     // out[t, o] = base[t, o] + sum_j low[row, j] W_a(o, j)
    AdaptPlan plan;
    const float* low;
    const void* w;     // [n] matrices of N x R (trans: R x N)
    const void* base;  // nullptr: zeros
    void* out;
    size_t ldb, ldo;
    int N, R;
    int vec_w, vec_b, vec_o;
    int in_place;      // base is out: rows without an adapter need no copy
};
struct AdaptGrad {     // G_a(m, j) = sum over a's rows of X[perm[row], m] low[row, j]
    AdaptPlan plan;
    const float* low;  // [T, RP]
    const void* x;
    size_t ldx;
    float* g;          // [n] matrices: element (m, j) at m * gm + j * gj
    float* part;       // partial slots of M * R
    int M, R, gm, gj, n;
    int vec_x;
};

struct AdaptDecode {   // hymoe_adapt for a few tokens: clusters of `ctas` CTAs per token
    const void* x;
    const void* base;  // nullptr: zeros
    void* out;
    const int* ids;
    const void* a;
    const void* b;
    const float* scale;
    size_t ldx, ldb, ldo;
    int n, R, K, N, ctas;
    int vec_x, vec_a, vec_b;  // rows start on 16-byte boundaries
    int in_place;
};
cudaError_t launch_adapt_decode(const AdaptDecode& d, int type_x, int type_w, int type_y, int T, cudaStream_t st);

// type_x: HYMOE_TYPE_F32 or type_w; trans: the weight matrix has the rank as its fast dimension
// (low) or the columns as its fast dimension (wide).
cudaError_t launch_adapt_low(const AdaptLow& a, int type_x, int type_w, bool trans, int n_sms, cudaStream_t st);
// Two narrow products as one launch: trans and then not, x of one type.
cudaError_t launch_adapt_lows(const AdaptLow& a, const AdaptLow& b, int type_x, int type_w, int n_sms, cudaStream_t st);
cudaError_t launch_adapt_wide(const AdaptWide& a, int type_y, int type_w, bool trans, int n_sms, cudaStream_t st);
// One or two gradients over long rows of one type (g == nullptr: none).
cudaError_t launch_adapt_grad(const AdaptGrad& a, const AdaptGrad& b, int type_x, cudaStream_t st);
// Adds the pieces of long adapters in one or two gradients (g == nullptr: none).
cudaError_t launch_adapt_join(const AdaptGrad& a, const AdaptGrad& b, cudaStream_t st);

#ifdef __CUDACC__

// The 64 rows that a CTA of the mma.sync kernels takes: part of a tile; rows 0: none.
__device__ __forceinline__ int4 ad_part_tile(const AdaptPlan& p, int id) {
    const int sub = p.tile_rows / kAdRows;
    if (id / sub >= p.n_lists[1]) return make_int4(-1, 0, 0, 0);
    int4 t = p.tiles[id / sub];
    const int off = id % sub * kAdRows;
    t.y += off;
    t.z = min(kAdRows, t.z - off);
    return t.z > 0 ? t : make_int4(-1, 0, 0, 0);
}

// The warp's largest |value| (never negative) into an adapter's entry: maxima commute, so any order
// gives the same.
__device__ __forceinline__ void ad_amax(unsigned* amax, float v) {
    const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
    if ((threadIdx.x & 31) == 0) atomicMax(amax, m);
}

constexpr int ad_pad16(int bytes) { return (bytes / 16 % 2 == 0) ? bytes + 16 : bytes; }  // odd number of pieces

__device__ __forceinline__ void cp_async16_part(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// One 16-byte piece of a row into shared memory: `n` of its elements exist (the rest become 0).
// src must be a valid address also where n == 0.
template <int ES>
__device__ __forceinline__ void ad_copy_piece(char* dst, const char* src, int n, bool vec) {
    constexpr int P = 16 / ES;
    n = n < 0 ? 0 : n > P ? P : n;
    if (vec) {
        cp_async16_part(dst, src, n * ES);
    } else {
        uint32_t v[4] = {0u, 0u, 0u, 0u};
        if constexpr (ES == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < n) v[i] = reinterpret_cast<const uint32_t*>(src)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(src)[i]) << (16 * (i & 1));
        }
        *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename W>
struct AdType;
template <>
struct AdType<__half> {
    static constexpr bool kScaled = true;  // a row of fp32 values needs a power of two before it is split
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // the two values of a register as fp32
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct AdType<__nv_bfloat16> {
    static constexpr bool kScaled = false;
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// v = hi + lo, both tf32 (their low 13 bits are 0, or ignored by the product): lo is exact in fp32.
__device__ __forceinline__ void split_tf32(float v, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(v) & 0xffffe000u;
    lo = __float_as_uint(v - __uint_as_float(hi));
}
// What is left of v beside its first part: nothing of an infinity (inf - inf would make the row NaN).
__device__ __forceinline__ float part_rest(float v, float part) { return fabsf(v) == INFINITY ? 0.f : v - part; }

#endif  // __CUDACC__

}  // namespace hymoe
