// adapt_wide_tc.cu — the adapters' wide product on the 5th-generation tensor cores with its
// epilogue: out[token of row] = base[token of row] + W_a low[row], for rows and weights on 16-byte
// boundaries.
//
// Persistent: the work is (tile of 128 sorted rows, 256 bytes of its columns), tile-major, and every
// CTA takes an equal run of it, so that a few tiles of unequal adapters still fill the GPU.
//   warp 0     brings in each unit's weights (TMA), up to the ring's stages ahead, and its base rows
//              where the tile's tokens are consecutive
//   warps 10-13 copy the base rows of other tiles, 16 lanes to a row (gather4 loads of
//              four rows were tried: they top out at 3.1 TB/s, and one such tile among consecutive
//              ones held the whole call up)
//   warp 1     issues the products: M = 128 rows, N = 128 (16-bit results) or 64 columns, into one of
//              four accumulators in tensor memory
//   warps 2-9  at a tile's start turn its fp32 rows of low into 16-bit parts in shared memory (two
//              for a 16-bit result; enough to hold fp32 for an fp32 one), which then are the A operand
//              of all its units; for every unit add the sums to the base in its shared-memory tile,
//              round once and write pieces of 128 bytes.  Two warps share 32 rows (a quarter of the
//              accumulator's lanes), each with half of the columns.
// One lane owns one row, so fp16 parts can carry a power of two per row.  Bound by reading and
// writing the rows of out: 4160 tokens of requests to 4096 F32 columns, rank 16, 26.5 us (5.1 TB/s);
// 8192 tokens in any order to 6144 bf16 columns, rank 64, 52 us (3.9 TB/s, in pieces of 256 bytes).
#include "adapt_tc.cuh"

namespace hymoe {
namespace {

constexpr int kWtcThreads = 448;
constexpr int kWtcAccs = 4;
constexpr int kWtcPanel = kTcRows * 128;      // 128 bytes of every row
constexpr int kWtcBase = 2 * kWtcPanel;       // a unit's rows

template <typename Y, typename W, int RP, bool TRANS>
struct WtcTile {
    static constexpr bool kF32 = sizeof(Y) == 4;
    static constexpr int kCols = kF32 ? 64 : 128;             // columns of a unit
    static constexpr int kParts = kF32 && !AdType<W>::kScaled ? 3 : 2;
    static constexpr int kKBlocks = (RP + 63) / 64;           // 64-wide blocks of the rank
    static constexpr int kA = kParts * kKBlocks * kWtcPanel;
    // weights of a unit: K-major [kCols][RP in blocks of 64]; MN-major [columns in blocks of 64][RP rows]
    static constexpr int kW = TRANS ? kCols / 64 * RP * 128 : kKBlocks * kCols * 128;
    static constexpr int kStage = kWtcBase + (kW + 1023) / 1024 * 1024;
    static constexpr int kStages = (225 * 1024 - kA) / kStage < 4 ? (225 * 1024 - kA) / kStage : 4;
    static constexpr int kSmem = 1024 + kA + kStages * kStage;
    static_assert(kStages >= 2, "a ring");
};

// Bounded wait of a whole warp until a counter in shared memory reaches n.
__device__ __forceinline__ bool count_wait(const uint32_t* count, int n, int* err) {
    int ok = 1;
    if (n > 0 && (threadIdx.x & 31) == 0) {
        const uint64_t t0 = globaltimer_ns();
        while (ok && static_cast<int>(ld_acquire_cta_u32(count)) < n) {
            __nanosleep(40);
            if (globaltimer_ns() - t0 > kWaitBudgetNs || *(volatile int*)err != 0) {
                atomicOr(err, DEVERR_TIMEOUT_PRODUCER);
                ok = 0;
            }
        }
    }
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

template <typename Y, typename W, int RP, bool TRANS>
__global__ __launch_bounds__(kWtcThreads, 1) void wide_tc_kernel(const __grid_constant__ AdaptMaps maps,
                                                                 const __grid_constant__ AdaptWide a) {
    using L = WtcTile<Y, W, RP, TRANS>;
    extern __shared__ uint8_t raw[];
    uint8_t* sA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* ring = sA + L::kA;
    __shared__ uint64_t full[L::kStages], copied[L::kStages], empty[L::kStages], acc_full[kWtcAccs], acc_empty[kWtcAccs], a_full, mma_end;
    __shared__ uint32_t tmem_s, armed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&copied[s], 128);
            mbar_init(&empty[s], 9);  // the products' completion and eight epilogue warps
        }
        for (int b = 0; b < kWtcAccs; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 8);
        }
        mbar_init(&a_full, 8);
        mbar_init(&mma_end, 1);
        armed = 0u;
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
    // The plan was complete before the narrow product began (which let this grid be scheduled), and
    // whatever wrote the base and the weights before the plan began: their loads need not wait for the
    // narrow product, only its readers do.
    if (warp >= 2 && warp < 10) griddep_wait();
    griddep_launch_dependents();
    int* err = a.plan.err;
    const int n_blk = (a.N + L::kCols - 1) / L::kCols;
    const int n_tiles = a.plan.n_lists[a.in_place ? 3 : 1];  // in place, rows without an adapter stay
    const int64_t units = static_cast<int64_t>(n_tiles) * n_blk;
    const int64_t u_lo = units * blockIdx.x / gridDim.x;
    const int n_units = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x - u_lo);
    // this CTA's first unit; every role steps on from it by itself (a division per unit and role cost
    // 0.8 us a unit)
    const int ti0 = static_cast<int>(u_lo / n_blk), blk0 = static_cast<int>(u_lo % n_blk);

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            int it = 0, at = -1, first = 0;
            int4 tile = make_int4(-1, 0, 0, 0);
            bool run = false;
            for (int ti = ti0, blk = blk0; it < n_units; ++it, ++blk) {
                if (blk == n_blk) {
                    blk = 0;
                    ++ti;
                }
                const int c0 = blk * L::kCols;
                if (ti != at) {
                    at = ti;
                    tile = a.plan.tiles[ti];
                    run = a.base != nullptr && tile_run(a.plan, tile, &first);
                }
                const int s = it % L::kStages;
                uint8_t* sb = ring + s * L::kStage;
                if (!mbar_wait(&empty[s], ((it / L::kStages) & 1) ^ 1, err, DEVERR_TIMEOUT_PRODUCER)) break;
                red_release_cta_add(&armed, 1u);
                mbar_arrive_expect_tx(&full[s], (tile.x >= 0 ? L::kW : 0) + (run ? kWtcBase : 0));
                if (tile.x >= 0) {
                    uint8_t* sw = sb + kWtcBase;
                    if (TRANS) {  // [RP rows][64 columns] per block of columns
#pragma unroll
                        for (int n = 0; n < L::kCols / 64; ++n)
                            tma_load_3d(sw + n * RP * 128, &maps.w, &full[s], c0 + n * 64, 0, tile.x);
                    } else {      // [columns][64 of the rank] per block of the rank
#pragma unroll
                        for (int k = 0; k < L::kKBlocks; ++k)
                            tma_load_3d(sw + k * L::kCols * 128, &maps.w, &full[s], k * 64, c0, tile.x);
                    }
                }
                if (run) {
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        tma_load_2d(sb + p * kWtcPanel, &maps.rows, &full[s], c0 + p * (L::kCols / 2), first);
                }
            }
            for (int j = it > L::kStages ? it - L::kStages : 0; j < it; ++j) mbar_drain(&full[j % L::kStages], (j / L::kStages) & 1);
        }
        __syncwarp();
    } else if (warp >= 10) {
        // ------------------------------------------------------------ base rows in any order
        constexpr int kPer = 16 / static_cast<int>(sizeof(Y));
        const int ct = tid - 320, piece = ct & 15, row0 = ct >> 4;  // rows row0 + 8 i of the tile
        const char* src[16];
        int it = 0, at = -1, n_copied = 0;
        bool copy = false;
        for (int ti = ti0, blk = blk0; it < n_units; ++it, ++blk) {
            if (blk == n_blk) {
                blk = 0;
                ++ti;
            }
            const int c0 = blk * L::kCols;
            if (ti != at) {
                at = ti;
                const int4 tile = a.plan.tiles[ti];
                int first;
                copy = a.base != nullptr && !tile_run(a.plan, tile, &first);
                if (copy) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        src[i] = static_cast<const char*>(a.base) +
                                 (static_cast<size_t>(__ldg(a.plan.perm + tile.y + min(row0 + 8 * i, tile.z - 1))) * a.ldb + piece * kPer) * sizeof(Y);
                }
            }
            if (!copy) continue;
            // Units between copied ones pass without these warps, so they follow the producer's count of
            // slots that it found free (a barrier's parity tells phases apart only for a warp that
            // takes part in each).  The barriers `copied` are taken in turn.
            const int s = it % L::kStages;
            if (!count_wait(&armed, it + 1, err)) break;
            uint8_t* dst = ring + s * L::kStage + piece / 8 * kWtcPanel;
            const int bytes = c0 + piece * kPer < a.N ? 16 : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                cp_async16_part(dst + sw128_offset(row0 + 8 * i, piece % 8),
                                bytes ? src[i] + static_cast<size_t>(c0) * sizeof(Y) : static_cast<const char*>(a.base), bytes);
            cp_async_arrive(&copied[n_copied % L::kStages]);
            ++n_copied;
        }
        cp_async_wait_all();
    } else if (warp == 1) {
        // ------------------------------------------------------------ products
        if (lane == 0) {
            constexpr uint32_t idesc = ad_idesc<W>(L::kCols, false, TRANS);
            int it = 0, at = -1, tiles_done = 0, accs = 0;
            bool mul = false, ok = true;
            for (int ti = ti0, blk = blk0; ok && it < n_units; ++it, ++blk) {
                if (blk == n_blk) {
                    blk = 0;
                    ++ti;
                }
                const int s = it % L::kStages;
                if (ti != at) {
                    at = ti;
                    mul = a.plan.tiles[ti].x >= 0;
                    if (mul) {
                        ok = mbar_wait(&a_full, tiles_done & 1, err, DEVERR_TIMEOUT_MMA);
                        ++tiles_done;
                    }
                }
                ok = ok && mbar_wait(&full[s], (it / L::kStages) & 1, err, DEVERR_TIMEOUT_MMA);
                if (!ok) break;
                if (!mul) {
                    mbar_arrive(&empty[s]);
                    continue;
                }
                const int b = accs % kWtcAccs;
                ok = mbar_wait(&acc_empty[b], ((accs / kWtcAccs) & 1) ^ 1, err, DEVERR_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after();
                const uint32_t sa = smem_u32(sA), sw = smem_u32(ring + s * L::kStage + kWtcBase);
                uint32_t more = 0;
#pragma unroll
                for (int p = L::kParts - 1; p >= 0; --p)  // small parts first
#pragma unroll
                    for (int k = 0; k < RP / 16; ++k) {
                        const uint64_t da = sw128_kmajor_desc(sa + (p * L::kKBlocks + k / 4) * kWtcPanel + (k % 4) * 32);
                        const uint64_t db = TRANS ? sw128_mnmajor_desc(sw + k * 2048, RP * 128)
                                                  : sw128_kmajor_desc(sw + (k / 4) * L::kCols * 128 + (k % 4) * 32);
                        mma_f16_ss(tmem + b * 128, da, db, idesc, more);
                        more = 1;
                    }
                mma_commit(&empty[s]);
                mma_commit(&acc_full[b]);
                ++accs;
            }
            mma_commit(&mma_end);
            mbar_drain(&mma_end, 0);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ epilogue
        const int q = warp & 3, half = (warp - 2) >> 2, r = q * 32 + lane;
        int it = 0, at = -1, accs = 0, n_copied = 0;
        int4 tile = make_int4(-1, 0, 0, 0);
        bool copy = false;
        char* op[8];       // rows 4 i + lane / 8 of the quarter, at this lane's piece; nullptr: no such row
        float back = 1.f;
        constexpr int kPer = 16 / static_cast<int>(sizeof(Y));  // values of a piece
        constexpr int kHalf = L::kCols / 2;                     // this warp's columns: one panel
        const int col_off = half * kHalf + (lane & 7) * kPer;
        bool ok = true;
        for (int ti = ti0, blk = blk0; ok && it < n_units; ++it, ++blk) {
            if (blk == n_blk) {
                blk = 0;
                ++ti;
            }
            const int c0 = blk * L::kCols;
            const int s = it % L::kStages;
            if (ti != at) {
                // the previous tile's products have ended: their sums were waited for
                at = ti;
                tile = a.plan.tiles[ti];
                int first;
                copy = a.base != nullptr && !tile_run(a.plan, tile, &first);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int row = q * 32 + 4 * i + (lane >> 3);
                    op[i] = row < tile.z ? static_cast<char*>(a.out) +
                                               (static_cast<size_t>(__ldg(a.plan.perm + tile.y + row)) * a.ldo + col_off) * sizeof(Y)
                                         : nullptr;
                }
                if (tile.x >= 0) {
                    const bool real = r < tile.z;
                    const float4* row = reinterpret_cast<const float4*>(a.low + static_cast<size_t>(tile.y + (real ? r : 0)) * RP);
                    float f = 1.f;
                    if constexpr (AdType<W>::kScaled) {  // a power of two that brings the row into [1, 2)
                        float m = 0.f;
                        for (int c = 0; c < RP / 4; ++c) {
                            const float4 v = row[c];
                            m = fmaxf(m, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                        }
                        const int e = max(1, min(253, static_cast<int>(__float_as_uint(m) >> 23)));
                        f = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
                        back = __uint_as_float(static_cast<uint32_t>(e) << 23);
                    }
#pragma unroll 2
                    for (int c = half * (RP / 16); c < (half + 1) * (RP / 16); ++c) {
                        float v[8];
                        *reinterpret_cast<float4*>(v) = row[2 * c];
                        *reinterpret_cast<float4*>(v + 4) = row[2 * c + 1];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = real ? v[j] * f : 0.f;
#pragma unroll
                        for (int p = 0; p < L::kParts; ++p) {
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                w[j] = AdType<W>::pack(v[2 * j], v[2 * j + 1]);
                                const float2 b = AdType<W>::unpack(w[j]);
                                v[2 * j] = part_rest(v[2 * j], b.x);
                                v[2 * j + 1] = part_rest(v[2 * j + 1], b.y);
                            }
                            *reinterpret_cast<uint4*>(sA + (p * L::kKBlocks + c / 8) * kWtcPanel + sw128_offset(r, c % 8)) =
                                make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&a_full);
                }
            }
            const bool mul = tile.x >= 0;
            uint8_t* sb = ring + s * L::kStage;
            const int b = accs % kWtcAccs;
            if (mul) ok = mbar_wait(&acc_full[b], (accs / kWtcAccs) & 1, err, DEVERR_TIMEOUT_EPILOGUE);
            // the base rows, however they came (`full` in any case: see the copying warps)
            ok = ok && mbar_wait(&full[s], (it / L::kStages) & 1, err, DEVERR_TIMEOUT_EPILOGUE);
            if (ok && copy) ok = mbar_wait(&copied[n_copied % L::kStages], (n_copied / L::kStages) & 1, err, DEVERR_TIMEOUT_EPILOGUE);
            ok = __all_sync(0xffffffffu, ok);
            n_copied += copy;
            if (!ok) break;
            if (mul || a.base == nullptr) {
                tc_fence_after();
                uint8_t* panel = sb + half * kWtcPanel + r * 128;
                const uint32_t flip = static_cast<uint32_t>(r & 7) << 4;
                uint4 o[8];  // the row's 128 bytes of this panel, all loaded before any is stored
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    o[j] = a.base != nullptr ? *reinterpret_cast<const uint4*>(panel + ((static_cast<uint32_t>(j) << 4) ^ flip))
                                             : make_uint4(0u, 0u, 0u, 0u);
                if (mul) {
                    constexpr int kPieces = 32 / kPer;  // pieces of 32 columns
#pragma unroll
                    for (int h = 0; h < kHalf / 32; ++h) {
                        uint32_t v[32];
                        tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(q * 32) << 16) + b * 128 + half * kHalf + h * 32, v);
                        tmem_ld_wait();
                        if (AdType<W>::kScaled) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * back);
                        }
#pragma unroll
                        for (int j = 0; j < kPieces; ++j) {
                            uint32_t* ow = reinterpret_cast<uint32_t*>(&o[h * kPieces + j]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if constexpr (L::kF32) {
                                    ow[i] = __float_as_uint(__uint_as_float(ow[i]) + __uint_as_float(v[4 * j + i]));
                                } else {
                                    const float2 f2 = AdType<W>::unpack(ow[i]);
                                    ow[i] = AdType<W>::pack(f2.x + __uint_as_float(v[8 * j + 2 * i]), f2.y + __uint_as_float(v[8 * j + 2 * i + 1]));
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(panel + ((static_cast<uint32_t>(j) << 4) ^ flip)) = o[j];
                if (mul) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_empty[b]);
                    ++accs;
                }
                __syncwarp();
            }
            // the warp's 32 rows of 128 bytes, four rows per store
            {
                const uint8_t* from = sb + half * kWtcPanel + (q * 32 + (lane >> 3)) * 128;
                uint4 o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    o[i] = *reinterpret_cast<const uint4*>(from + i * 512 + (((lane & 7) ^ ((4 * i + (lane >> 3)) & 7)) << 4));
                if (c0 + col_off < a.N) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (op[i] != nullptr) *reinterpret_cast<uint4*>(op[i] + static_cast<size_t>(c0) * sizeof(Y)) = o[i];
                }
            }
            fence_proxy_async_smem();  // the slot was written here and is TMA's next
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename Y, typename W, int RP, bool TRANS>
cudaError_t launch_t(const AdaptMaps& maps, const AdaptWide& a, int n_sms, cudaStream_t st) {
    using L = WtcTile<Y, W, RP, TRANS>;
    auto kern = wide_tc_kernel<Y, W, RP, TRANS>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    return launch_kernel(true, kern, dim3(n_sms), dim3(kWtcThreads), L::kSmem, st, maps, a);
}

template <typename Y, typename W>
cudaError_t launch_y(const AdaptMaps& maps, const AdaptWide& a, bool trans, int n_sms, cudaStream_t st) {
    switch (adapt_rp(a.R)) {
        case 16: return trans ? launch_t<Y, W, 16, true>(maps, a, n_sms, st) : launch_t<Y, W, 16, false>(maps, a, n_sms, st);
        case 32: return trans ? launch_t<Y, W, 32, true>(maps, a, n_sms, st) : launch_t<Y, W, 32, false>(maps, a, n_sms, st);
        case 64: return trans ? launch_t<Y, W, 64, true>(maps, a, n_sms, st) : launch_t<Y, W, 64, false>(maps, a, n_sms, st);
        default: return trans ? launch_t<Y, W, 128, true>(maps, a, n_sms, st) : launch_t<Y, W, 128, false>(maps, a, n_sms, st);
    }
}

}  // namespace

cudaError_t launch_adapt_wide_tc(const AdaptMaps& maps, const AdaptWide& a, int type_y, int type_w, bool trans, int n_sms,
                                 cudaStream_t st) {
    if (type_w == HYMOE_TYPE_F16)
        return type_y == HYMOE_TYPE_F32 ? launch_y<float, __half>(maps, a, trans, n_sms, st)
                                        : launch_y<__half, __half>(maps, a, trans, n_sms, st);
    return type_y == HYMOE_TYPE_F32 ? launch_y<float, __nv_bfloat16>(maps, a, trans, n_sms, st)
                                    : launch_y<__nv_bfloat16, __nv_bfloat16>(maps, a, trans, n_sms, st);
}

}  // namespace hymoe
