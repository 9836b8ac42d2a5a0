// adapt_low_tc.cu — the adapters' narrow product on the 5th-generation tensor cores, for rows of the
// weights' 16-bit type on 16-byte boundaries: low[row] = scale[a] * W_a x[token of row].
//
// A tile of 128 sorted rows of one adapter is a cluster of S CTAs (1, 2, 4 or 8), each over a part
// of the long dimension.  64 columns of the rows and of the weights make a stage: one thread brings
// the weights in by TMA, and the rows too where their tokens are consecutive; rows in any order are
// copied by the four later epilogue warps, eight lanes to a row (gather4 loads of four rows were
// tried: they top out at 2.5 TB/s).  One thread issues the products (M = 128 rows, N = RP) into
// tensor memory.  The parts are added in distributed shared memory, every CTA taking its share of
// the rows, in the order of the parts.
//
// The pipe truncates what it adds, up to 1.4 times 2^-23 of the running sum each time (terms of one
// sign; some 4e-8 of it on average over terms of both), so a CTA's
// columns take turns in four accumulators (two at rank 128), as long as that makes 64 stages at most:
// 64 additions each (128).  Longer rows (LONG) go in segments of 8 stages, 32 additions to one
// accumulator, which the epilogue's warps add in fp32 to totals in tensor memory while the next
// segment goes to another (at rank 128 there is room for one and the totals: the next segment's loads
// go on, its products wait).  Without segments 2^20 columns lost 1.5e-4 of low (rank 128: 3.4e-4).
//
// Bound by reading x: 8192 tokens of 4096 columns, rank 64, in
// any order 21 us (3.2 TB/s; some 8 us pass before the loads are in full flow and after they end).
#include "adapt_tc.cuh"

namespace hymoe {
namespace {

constexpr int kLtcRows = kTcRows;
constexpr int kLtcThreads = 192;  // TMA, MMA, four copying and epilogue warps
constexpr int kLtcMostStages = 64;  // of a CTA without segments
constexpr int kLtcSegment = 8;      // stages of a segment

// N: columns of the product; an MN-major weight tile has whole blocks of 64.
template <int RP, bool TRANS>
struct LtcTile {
    static constexpr int kN = TRANS && RP < 64 ? 64 : RP;
    static constexpr int kA = kLtcRows * 128, kB = kN * 128;
    static constexpr int kStages = kN == 128 ? 3 : 4;
    static constexpr int kSmem = 1024 + kStages * (kA + kB);
    static_assert(kStages * (kA + kB) >= kLtcRows * (RP + 4) * 4, "the stages hold the partial sums");
    static constexpr int kAccs = kN == 128 ? 2 : 4;  // accumulators
    static constexpr int kSet = kN < 32 ? 32 : kN;   // columns of one
    static constexpr int kCols = kAccs * kSet;       // two CTAs share the 512 of an SM
    static constexpr int kBufs = kAccs / 2;          // LONG: those of segments, and behind them the totals
};

template <typename W, int RP, bool TRANS, bool LONG>
__global__ __launch_bounds__(kLtcThreads, 2) void low_tc_kernel(const __grid_constant__ AdaptMaps maps,
                                                                const __grid_constant__ AdaptLow a, int S) {
    using L = LtcTile<RP, TRANS>;
    constexpr int kSets = LONG ? 1 : L::kAccs;  // accumulators that a stage's products take in turn
    static_assert(L::kStages < kLtcSegment, "the copying warps add up a segment amid the next");
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full[L::kStages], empty[L::kStages], done, seg_done[L::kBufs], seg_free[L::kBufs];
    __shared__ uint32_t tmem_s;
    __shared__ int tok[kLtcRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();
    griddep_launch_dependents();
    const int tile_id = blockIdx.x / S, rank = blockIdx.x % S;
    int4 tile = make_int4(-1, 0, 0, 0);
    if (tile_id < a.plan.n_lists[1]) tile = a.plan.tiles[tile_id];
    if (tile.x < 0) return;  // the whole cluster: no such tile, or rows without an adapter
    int first;
    const bool run = tile_run(a.plan, tile, &first);
    if (tid < kLtcRows) tok[tid] = __ldg(a.plan.perm + tile.y + min(tid, tile.z - 1));
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full[s], run ? 1 : 129);  // TMA, and the copying threads
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        if (LONG) {
            for (int b = 0; b < L::kBufs; ++b) {
                mbar_init(&seg_done[b], 1);
                mbar_init(&seg_free[b], 4);  // the epilogue's warps
            }
        }
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_s, L::kCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    const int nk = (a.K + 63) / 64;
    const int k_lo = static_cast<int>(static_cast<int64_t>(nk) * rank / S);
    const int k_hi = static_cast<int>(static_cast<int64_t>(nk) * (rank + 1) / S);
    const int n_seg = (k_hi - k_lo + kLtcSegment - 1) / kLtcSegment;
    int* err = a.plan.err;  // the status word

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
                const int s = it % L::kStages;
                if (!mbar_wait(&empty[s], ((it / L::kStages) & 1) ^ 1, err, DEVERR_TIMEOUT_PRODUCER)) break;
                uint8_t* sa = smem + s * (L::kA + L::kB);
                mbar_arrive_expect_tx(&full[s], L::kB + (run ? L::kA : 0));
                if (run) tma_load_2d(sa, &maps.rows, &full[s], kb * 64, first);
                if (TRANS) {
                    // weights [K][R]: 64 K rows, in blocks of 64 along the rank
#pragma unroll
                    for (int n = 0; n < L::kN / 64; ++n)
                        tma_load_3d(sa + L::kA + n * 8192, &maps.w, &full[s], n * 64, kb * 64, tile.x);
                } else {
                    tma_load_3d(sa + L::kA, &maps.w, &full[s], kb * 64, 0, tile.x);
                }
            }
            // (a stage whose rows are copied completes only if the copying warps went on as well)
            for (int j = it > L::kStages ? it - L::kStages : 0; j < it; ++j) mbar_drain(&full[j % L::kStages], (j / L::kStages) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = ad_idesc<W>(L::kN, false, TRANS);
            int it = 0;
            for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
                const int s = it % L::kStages;
                const int seg = it / kLtcSegment, b = LONG ? seg % L::kBufs : 0, seg_it = LONG ? it % kLtcSegment : it;
                if (LONG && seg_it == 0 && seg >= L::kBufs && !mbar_wait(&seg_free[b], (seg / L::kBufs - 1) & 1, err, DEVERR_TIMEOUT_MMA)) break;
                if (!mbar_wait(&full[s], (it / L::kStages) & 1, err, DEVERR_TIMEOUT_MMA)) break;
                if (!run) fence_proxy_async_smem();  // the copied rows, before the tensor core reads them
                tc_fence_after();
                const uint32_t sa = smem_u32(smem + s * (L::kA + L::kB)), sb = sa + L::kA;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    mma_f16_ss(tmem + (b + kk % kSets) * L::kSet, sw128_kmajor_desc(sa + kk * 32),
                               TRANS ? sw128_mnmajor_desc(sb + kk * 2048, 8192) : sw128_kmajor_desc(sb + kk * 32), idesc,
                               seg_it != 0 || kk >= kSets ? 1u : 0u);
                mma_commit(&empty[s]);
                if (LONG && seg_it == kLtcSegment - 1 && seg + 1 < n_seg) mma_commit(&seg_done[b]);
            }
            mma_commit(&done);
            mbar_drain(&done, 0);  // every product has ended before tensor memory is freed
        }
        __syncwarp();
    } else {
        const int q = warp & 3, et = tid - 64;
        const uint32_t mine = tmem + (static_cast<uint32_t>(q * 32) << 16);  // this warp's rows
        // Sixteen columns of accumulators b .. b + kSets and, with `more`, of the totals.
        const auto gather = [&](int b, int c, bool more, float (&sum)[16]) {
            uint32_t v[kSets + LONG][16];
#pragma unroll
            for (int set = 0; set < kSets; ++set) tmem_ld_32x32b_x16(mine + (b + set) * L::kSet + c, v[set]);
            if (LONG && more) tmem_ld_32x32b_x16(mine + L::kBufs * L::kSet + c, v[kSets - 1 + LONG]);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                sum[j] = __uint_as_float(v[0][j]);
#pragma unroll
                for (int set = 1; set < kSets; ++set) sum[j] += __uint_as_float(v[set][j]);
                if (LONG && more) sum[j] += __uint_as_float(v[kSets - 1 + LONG][j]);
            }
        };
        // The sums of the next segment but the last, when it has ended, into the totals.
        int folded = 0;
        const auto fold = [&]() {
            const int b = folded % L::kBufs;
            if (!__all_sync(0xffffffffu, mbar_wait(&seg_done[b], (folded / L::kBufs) & 1, err, DEVERR_TIMEOUT_EPILOGUE))) return false;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < RP; c += 16) {
                float sum[16];
                gather(b, c, folded > 0, sum);
                uint32_t v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(sum[j]);
                tmem_st_32x32b_x16(mine + L::kBufs * L::kSet + c, v);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&seg_free[b]);
            ++folded;
            return true;
        };
        bool ok = true;
        if (!run) {
            // this thread's piece of rows et / 8 + 16 i
            const int piece = et & 7;
            const char* src[8];
            uint32_t dst[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = (et >> 3) + 16 * i;
                src[i] = static_cast<const char*>(a.x) + (static_cast<size_t>(tok[r]) * a.ldx + piece * 8) * 2;
                dst[i] = sw128_offset(r, piece);
            }
            int it = 0;
            for (int kb = k_lo; ok && kb < k_hi; ++kb, ++it) {
                const int s = it % L::kStages;
                // the ring is full of the next segment's stages (which may wait for this): time for the last one's sums
                if (LONG && it >= kLtcSegment && it % kLtcSegment == L::kStages && !(ok = fold())) break;
                if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ((it / L::kStages) & 1) ^ 1, err, DEVERR_TIMEOUT_PRODUCER))) break;
                uint8_t* sa = smem + s * (L::kA + L::kB);
                const int left = a.K - kb * 64 - piece * 8;
                const int bytes = left >= 8 ? 16 : 0;  // K is a multiple of 8
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    cp_async16_part(sa + dst[i], bytes ? src[i] + static_cast<size_t>(kb) * 128 : static_cast<const char*>(a.x), bytes);
                cp_async_arrive(&full[s]);
            }
            ok = ok && it == k_hi - k_lo;
            cp_async_wait_all();
        }
        if (LONG)
            while (ok && folded + 1 < n_seg) ok = fold();
        // on an expired wait the status word says that the results are not valid
        mbar_wait(&done, 0, err, DEVERR_TIMEOUT_EPILOGUE);
        tc_fence_after();
        const int r = q * 32 + lane;
        const float f = a.scale != nullptr ? __ldg(a.scale + tile.x) : 1.f;
        // the sums through shared memory (the stages are free): rows padded by four floats
        float* red = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int c = 0; c < RP; c += 16) {
            float sum[16];
            gather(LONG ? (n_seg - 1) % L::kBufs : 0, c, n_seg > 1, sum);
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *reinterpret_cast<float4*>(red + r * (RP + 4) + c + j) = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
        }
        tc_fence_before();
        if (S == 1) {
            named_bar_sync(1, 128);
        } else {
            cluster_arrive();
            cluster_wait();
        }
        const int rows = kLtcRows / S;
        float top = 0.f;
        for (int p = et; p < rows * (RP / 4); p += 128) {
            const int row = rank * rows + p / (RP / 4), c = p % (RP / 4) * 4;
            if (row >= tile.z) break;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < S; ++i) {
                const float4 v = ld_cluster4(mapa_shared(red + row * (RP + 4) + c, i));
                s.x += v.x;
                s.y += v.y;
                s.z += v.z;
                s.w += v.w;
            }
            // (columns behind the rank: 0 times an infinity is none of the result's)
            s = make_float4(c < a.R ? s.x * f : 0.f, c + 1 < a.R ? s.y * f : 0.f, c + 2 < a.R ? s.z * f : 0.f, c + 3 < a.R ? s.w * f : 0.f);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(s.x), fabsf(s.y)), fmaxf(fabsf(s.z), fabsf(s.w))));
            *reinterpret_cast<float4*>(a.low + static_cast<size_t>(tile.y + row) * RP + c) = s;
        }
        __syncwarp();
        if (a.amax != nullptr) ad_amax(a.amax + tile.x, top);
    }
    if (S > 1) {  // every thread arrives once before the sums are read and once after
        if (warp < 2) {
            cluster_arrive();
            cluster_wait();
        }
        cluster_arrive();
        cluster_wait();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, L::kCols);
    }
}

template <typename W, int RP, bool TRANS>
cudaError_t launch_t(const AdaptMaps& maps, const AdaptLow& a, int n_sms, cudaStream_t st) {
    using L = LtcTile<RP, TRANS>;
    // as many CTAs as two to an SM allow (for the tiles that are likely: half of the adapters' last
    // ones are short of the bound), each with two stages of columns at least
    const int nk = (a.K + 63) / 64, tiles = a.plan.max_tiles - a.plan.spare_tiles / 2;
    int S = 1;
    while (S < 8 && tiles * 2 * S <= 2 * n_sms && nk >= 4 * S) S *= 2;
    auto kern = (nk + S - 1) / S > kLtcMostStages ? low_tc_kernel<W, RP, TRANS, true> : low_tc_kernel<W, RP, TRANS, false>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.plan.max_tiles) * S);
    cfg.blockDim = dim3(kLtcThreads);
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
    return cudaLaunchKernelEx(&cfg, kern, maps, a, S);
}

template <typename W>
cudaError_t launch_w(const AdaptMaps& maps, const AdaptLow& a, bool trans, int n_sms, cudaStream_t st) {
    switch (adapt_rp(a.R)) {
        case 16: return trans ? launch_t<W, 16, true>(maps, a, n_sms, st) : launch_t<W, 16, false>(maps, a, n_sms, st);
        case 32: return trans ? launch_t<W, 32, true>(maps, a, n_sms, st) : launch_t<W, 32, false>(maps, a, n_sms, st);
        case 64: return trans ? launch_t<W, 64, true>(maps, a, n_sms, st) : launch_t<W, 64, false>(maps, a, n_sms, st);
        default: return trans ? launch_t<W, 128, true>(maps, a, n_sms, st) : launch_t<W, 128, false>(maps, a, n_sms, st);
    }
}

}  // namespace

cudaError_t launch_adapt_low_tc(const AdaptMaps& maps, const AdaptLow& a, int type_w, bool trans, int n_sms, cudaStream_t st) {
    return type_w == HYMOE_TYPE_F16 ? launch_w<__half>(maps, a, trans, n_sms, st) : launch_w<__nv_bfloat16>(maps, a, trans, n_sms, st);
}

}  // namespace hymoe
