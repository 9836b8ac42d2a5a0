// adapt.cu — hymoe_adapt and hymoe_adapt_backward: low-rank adapters of many requests beside a
// projection they share, and their gradients.
//
//   low[t]  = scale[a] * A_a x[t]          (a = ids[t]; backward also scale[a] * B_a^T dy[t])
//   out[t]  = base[t] + B_a low[t]         (backward: dx[t] = base[t] + A_a^T low_dy[t])
//   dA_a    = sum_t low_dy[t] x[t]^T,  dB_a = sum_t dy[t] low_x[t]^T
//
// This file: the plan (tokens sorted by adapter, tiles of 64 or 128 rows of one adapter, gradient
// items), the checks and the order of the launches.  adapt_low.cu, adapt_wide.cu and
// adapt_grad.cu hold the three products, adapt_*_tc.cu the same on tcgen05, adapt_decode.cu all of
// hymoe_adapt for a few tokens.
#include <initializer_list>

#include <cudaTypedefs.h>

#include "adapt_tc.cuh"

namespace hymoe {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kPlanThreads = 1024;
constexpr int kPlanSmem = 220 * 1024;

// Warps of the plan that count and place tokens: one row of counters each, beside five lists.
__host__ __device__ constexpr int plan_rows(int n) {
    const int fit = (kPlanSmem / 4 - 5 * (n + 2)) / (n + 1);
    return fit < 32 ? fit : 32;
}

// Exclusive prefix sum of v[0, n) in place, v[n] = the sum; one warp.
__device__ void warp_scan(int* v, int n) {
    const int lane = threadIdx.x & 31;
    int run = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int x = i0 + lane < n ? v[i0 + lane] : 0;
        int inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kAll, inc, o);
            if (lane >= o) inc += u;
        }
        if (i0 + lane < n) v[i0 + lane] = run + inc - x;
        run += __shfl_sync(kAll, inc, 31);
    }
    if (lane == 0) v[n] = run;
}

// Largest b with pre[b] <= i, of pre[0..n] ascending, pre[n] > i.
__device__ __forceinline__ int bucket_of(const int* pre, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Stable counting sort of the tokens by adapter and the lists over the sorted rows, by one CTA:
// each counting warp owns a run of tokens (in order) and a row of counters, 32 tokens a step; the
// lanes of equal adapters find one another by a ballot for every bit of the adapter's number (a
// warp match takes a step for every distinct adapter: 16 us instead of 6 at 8192 tokens of 16).
// Up to 8192 tokens the adapters stay in registers between counting and placing.  Latency: 6 us for
// 77 tokens, 10 for 8192 of 16 adapters.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const int* __restrict__ ids, int T, int n, AdaptPlan p,
                                                            int chunk) {
    extern __shared__ int sm[];
    griddep_launch_dependents();
    const int nb = n + 1;  // the last bucket: no adapter
    int *off = sm, *tpre = off + n + 2, *ipre = tpre + n + 2, *spre = ipre + n + 2, *tot = spre + n + 2;
    int* cnt = tot + n + 2;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, W = plan_rows(n);
    const int per = ((T + W - 1) / W + 31) / 32 * 32;
    const int64_t lo64 = static_cast<int64_t>(warp) * per;
    const int t_lo = lo64 < T ? static_cast<int>(lo64) : T, t_hi = warp < W ? min(T, t_lo + per) : t_lo;
    const int bits = 32 - __clz(n);
    int b[8], rank[8], peers[8];  // adapter, place among the step's tokens of that adapter, their number
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = t0 + 32 * i + lane;
            int v = ids != nullptr && t < t_hi ? __ldg(ids + t) : 0;
            if (v < 0 || v >= n) v = n;
            b[i] = t < t_hi ? v : -1;
        }
    };
    auto equals = [&](int v) {  // lanes with the same v
        unsigned same = __ballot_sync(kAll, v >= 0);
        if (v < 0) same = ~same;
        for (int k = 0; k < bits; ++k) {
            const unsigned one = __ballot_sync(kAll, v >> k & 1);
            same &= v >> k & 1 ? one : ~one;
        }
        return same;
    };
    fetch(t_lo);
    for (int i = tid; i < W * nb; i += kPlanThreads) cnt[i] = 0;
    for (int i = tid; i < (p.items ? 2 : 1) * p.max_tiles * (p.tile_rows / kAdRows); i += kPlanThreads) p.counters[i] = 0u;
    __syncthreads();
    int* mine = cnt + (warp < W ? warp : 0) * nb;
    auto rate = [&](int i) {
        const unsigned same = equals(b[i]);
        rank[i] = __popc(same & ((1u << lane) - 1u));
        peers[i] = __popc(same);
    };
    for (int t0 = t_lo; t0 < t_hi; t0 += 256) {
        if (t0 > t_lo) fetch(t0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (t0 + 32 * i >= t_hi) break;
            rate(i);
            if (b[i] >= 0 && rank[i] == 0) mine[b[i]] += peers[i];
            __syncwarp();
        }
    }
    __syncthreads();
    for (int a = warp; a < nb; a += kPlanThreads / 32) {  // every run's start among the adapter's tokens
        const int c = lane < W ? cnt[lane * nb + a] : 0;
        int inc = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kAll, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane < W) cnt[lane * nb + a] = inc - c;
        if (lane == 31) {
            tot[a] = inc;
            off[a] = inc;
            tpre[a] = (inc + p.tile_rows - 1) / p.tile_rows;
            const int pieces = a < n ? max(1, (inc + chunk - 1) / chunk) : 0;
            ipre[a] = pieces;
            spre[a] = pieces > 1 ? pieces : 0;
        }
    }
    __syncthreads();
    if (warp == 0) warp_scan(off, nb);
    if (warp == 1) warp_scan(tpre, nb);
    if (warp == 2) warp_scan(ipre, n);
    if (warp == 3) warp_scan(spre, n);
    __syncthreads();
    const bool again = t_hi - t_lo > 256;  // more tokens than the registers held
    for (int t0 = t_lo; t0 < t_hi; t0 += 256) {
        if (again) fetch(t0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (t0 + 32 * i >= t_hi) break;
            if (again) rate(i);
            const int at = b[i] >= 0 ? mine[b[i]] : 0;
            __syncwarp();
            if (b[i] >= 0) {
                p.perm[off[b[i]] + at + rank[i]] = t0 + 32 * i + lane;
                if (rank[i] == 0) mine[b[i]] = at + peers[i];
            }
            __syncwarp();
        }
    }
    const int n_tiles = tpre[nb];
    for (int i = tid; i < n_tiles; i += kPlanThreads) {
        const int a = bucket_of(tpre, nb, i), r = (i - tpre[a]) * p.tile_rows;
        p.tiles[i] = make_int4(a < n ? a : -1, off[a] + r, min(p.tile_rows, tot[a] - r), 0);
    }
    if (p.items != nullptr) {
        const int n_items = ipre[n];
        for (int i = tid; i < n_items; i += kPlanThreads) {
            // equal pieces of whole 64s: none is empty, as chunk >= 512 makes tot > 512 (pieces - 1)
            // and pieces <= 8
            const int a = bucket_of(ipre, n, i), q = i - ipre[a], pieces = ipre[a + 1] - ipre[a];
            const int len = ((tot[a] + pieces - 1) / pieces + 63) / 64 * 64, r = q * len;
            p.items[i] = make_int4(a, off[a] + r, min(len, tot[a] - r), pieces > 1 ? spre[a] + q : -1);
        }
        for (int a = tid; a <= n; a += kPlanThreads) p.pieces[a] = ipre[a];
        for (int a = tid; a < 2 * n; a += kPlanThreads) p.amax[a] = 0u;
        if (tid == 0) p.n_lists[2] = n_items;
    }
    if (tid == 0) {
        p.n_lists[0] = 0;
        p.n_lists[1] = n_tiles;
        p.n_lists[3] = tpre[n];
    }
}

cudaError_t launch_plan_adapt(const int* ids, int T, int n, const AdaptPlan& p, cudaStream_t st) {
    const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanSmem);
    if (e != cudaSuccess) return e;
    const size_t smem = sizeof(int) * (5 * (static_cast<size_t>(n) + 2) + static_cast<size_t>(plan_rows(n)) * (n + 1));
    plan_kernel<<<1, kPlanThreads, smem, st>>>(ids, T, n, p, adapt_chunk(T, n));
    return cudaGetLastError();
}

// The workspace: every part starts on 256 bytes.
struct AdaptLayout {
    size_t perm, tiles, items, pieces, amax, lists, counters, low, low2, low_part, low_part2, part[2], slots, low16[2], bytes;
    int tile_rows, max_tiles, spare_tiles, max_items;
};
// (the sizes do not depend on tile_rows)
AdaptLayout adapt_layout(const hymoe_adapters* ad, size_t T, bool backward, int tile_rows = kAdRows) {
    AdaptLayout l{};
    const size_t n = ad->n_adapters;
    auto take = [&](size_t bytes) {
        const size_t at = l.bytes;
        l.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    if (T == 0 || (!backward && adapt_decodes(T, static_cast<int>(ad->rank)))) return l;
    const size_t long_pieces = T / kAdMinChunk < kAdMaxPieces ? T / kAdMinChunk : kAdMaxPieces;  // T / adapt_chunk at most
    const size_t buckets = n + 1 < T ? n + 1 : T;                   // adapters that have tokens, at most
    const size_t tiles64 = T / kAdRows + buckets, half_tiles = tiles64 + buckets;  // also twice the tiles of 128
    l.tile_rows = tile_rows;
    l.max_tiles = static_cast<int>(T / tile_rows + buckets);
    l.spare_tiles = static_cast<int>(buckets);
    l.max_items = static_cast<int>(n + long_pieces);
    l.lists = take(4 * sizeof(int));
    l.perm = take(T * sizeof(int));
    l.tiles = take(tiles64 * sizeof(int4));
    l.counters = take((backward ? 2 : 1) * half_tiles * sizeof(unsigned));
    l.low = take(T * adapt_rp(ad->rank) * sizeof(float));
    const size_t shared_tiles = half_tiles * kAdMaxSplits;
    const size_t low_part = (shared_tiles < kAdMaxSlots ? shared_tiles : kAdMaxSlots) * kAdRows * adapt_rp(ad->rank) * sizeof(float);
    l.low_part = take(low_part);
    if (backward) {
        l.items = take(static_cast<size_t>(l.max_items) * sizeof(int4));
        l.pieces = take((n + 1) * sizeof(int));
        l.amax = take(2 * n * sizeof(unsigned));
        l.low_part2 = take(low_part);
        l.low2 = take(T * adapt_rp(ad->rank) * sizeof(float));
        for (size_t& at : l.low16) at = take(T > kTcRows ? T * adapt_parts(adapt_rp(ad->rank)) * 2 : 0);
        l.slots = 2 * long_pieces;  // an adapter of c tokens in p > 1 pieces: p < 2 c / chunk
        // one part each: behind da's odd number of pieces' elements db's would not be on 16 bytes, as the join loads them
        l.part[0] = take(l.slots * ad->rank * ad->in_features * sizeof(float));
        l.part[1] = take(l.slots * ad->rank * ad->out_features * sizeof(float));
    }
    return l;
}
AdaptPlan plan_in(const AdaptLayout& l, char* ws, bool backward) {
    AdaptPlan p{};
    p.perm = reinterpret_cast<int*>(ws + l.perm);
    p.tiles = reinterpret_cast<int4*>(ws + l.tiles);
    p.items = backward ? reinterpret_cast<int4*>(ws + l.items) : nullptr;
    p.pieces = backward ? reinterpret_cast<int*>(ws + l.pieces) : nullptr;
    p.amax = backward ? reinterpret_cast<unsigned*>(ws + l.amax) : nullptr;
    p.err = p.n_lists = reinterpret_cast<int*>(ws + l.lists);  // the workspace's first word
    p.counters = reinterpret_cast<unsigned*>(ws + l.counters);
    p.tile_rows = l.tile_rows;
    p.max_tiles = l.max_tiles;
    p.spare_tiles = l.spare_tiles;
    p.max_items = l.max_items;
    return p;
}

// Rows of `ld` elements of `es` bytes that all start on 16-byte boundaries.
bool rows_vec(const void* p, size_t ld, size_t es) { return entry_aligned(p, 16) && ld * es % 16 == 0; }

const char* adapters_problem(const hymoe_adapters* ad) {
    if (!ad) return "null adapters";
    if (ad->n_adapters == 0 || ad->n_adapters > HYMOE_ADAPT_MAX_ADAPTERS) return "n_adapters must be 1..4096";
    if (ad->rank == 0 || ad->rank > HYMOE_ADAPT_MAX_RANK) return "rank must be 1..128";
    if (ad->in_features == 0 || ad->in_features > HYMOE_ADAPT_MAX_FEATURES || ad->out_features == 0 ||
        ad->out_features > HYMOE_ADAPT_MAX_FEATURES)
        return "in_features and out_features must be 1..1048576";
    if (ad->type != HYMOE_TYPE_F16 && ad->type != HYMOE_TYPE_BF16) return "adapters must be F16 or BF16";
    return nullptr;
}

const char* weights_problem(const hymoe_adapters* ad) {
    if (!ad->a || !ad->b) return "null adapter weights";
    if (!entry_aligned(ad->a, 2) || !entry_aligned(ad->b, 2) || !entry_aligned(ad->scale, 4))
        return "adapter pointers must be aligned to their elements";
    return nullptr;
}

// A matrix of the adapters' type or F32.
bool rows_ok(const hymoe_mat* m, uint32_t cols, int32_t type) {
    return entry_mat_ok(m, cols) && (m->type == type || m->type == HYMOE_TYPE_F32);
}

bool same_rows(const hymoe_mat* a, const hymoe_mat* b) { return a->data == b->data && a->ld == b->ld; }

}  // namespace
}  // namespace hymoe

using namespace hymoe;

extern "C" hymoe_status hymoe_adapt_workspace(const hymoe_adapters* ad, uint32_t n_tokens, int backward, size_t* bytes) {
    set_thread_error("");
    if (const char* why = adapters_problem(ad)) return entry_fail(HYMOE_ERR_INVALID_ARG, why);
    if (!bytes) return entry_fail(HYMOE_ERR_INVALID_ARG, "null bytes");
    if (n_tokens > HYMOE_ADAPT_MAX_TOKENS) return entry_fail(HYMOE_ERR_INVALID_ARG, "n_tokens must be at most 16777216");
    *bytes = adapt_layout(ad, n_tokens, backward != 0).bytes;
    return HYMOE_OK;
}

namespace {

// The checks that both calls share: sizes, workspace, device.
const char* common_problem(const hymoe_adapters* ad, const int32_t* ids, uint32_t T, const void* ws, size_t ws_bytes,
                           size_t need) {
    if (T > HYMOE_ADAPT_MAX_TOKENS) return "n_tokens must be at most 16777216";
    if (const char* why = weights_problem(ad)) return why;
    if (!entry_aligned(ids, 4)) return "ids must be 4-byte aligned";
    if (need > 0 && (!ws || ws_bytes < need || !entry_aligned(ws, 256)))
        return "workspace must be 256-byte aligned and of hymoe_adapt_workspace bytes";
    return nullptr;
}

hymoe_status current_device(int* dev) {
    if (cudaGetDevice(dev) == cudaSuccess) return HYMOE_OK;
    cudaGetLastError();
    return entry_fail(HYMOE_ERR_CUDA, "cudaGetDevice failed");
}

// SMs that the launches are sized for (the workspace's bound on partial sums assumes at most this).
int sm_count(int dev) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n < 1 ? 1 : n < kAdMaxSlots / 4 ? n : kAdMaxSlots / 4;
}

// ---- tensor maps of the tcgen05 kernels

using EncodeFn = PFN_cuTensorMapEncodeTiled_v12000;
EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

bool encode(CUtensorMap* m, int type, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
    const EncodeFn fn = encode_fn();
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUtensorMapDataType t = type == HYMOE_TYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : type == HYMOE_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return fn && fn(m, t, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Token rows [T, cols], boxes of 128 bytes of `rows` rows.
bool encode_rows(CUtensorMap* m, const hymoe_mat& x, int T, int cols, int rows) {
    const size_t es = elem_bytes(x.type);
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(T)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(T > 1 ? x.ld : cols) * es};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / es), static_cast<cuuint32_t>(rows)};
    return encode(m, x.type, 2, x.data, dims, strides, box);
}

// Weights [n][rows][cols], boxes of 64 columns and `box_rows` rows of one adapter.
bool encode_weights(AdaptMaps* m, const void* w, int type, int n, int rows, int cols, int box_rows) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(n)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 2, static_cast<cuuint64_t>(cols) * rows * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
    return encode(&m->w, type, 3, w, dims, strides, box);
}

// Rows that TMA can load in pieces of 128 bytes.
bool rows_tma(const hymoe_mat* m, uint32_t cols) {
    const size_t es = elem_bytes(m->type);
    return rows_vec(m->data, static_cast<size_t>(m->ld), es) && static_cast<size_t>(m->ld) * es < (size_t(1) << 40) &&
           cols * es % 16 == 0 && cols >= 64;
}
bool weights_tma(const hymoe_adapters* ad) {
    return ad->rank % 8 == 0 && ad->in_features % 8 == 0 && ad->out_features % 8 == 0 && entry_aligned(ad->a, 16) &&
           entry_aligned(ad->b, 16);
}

AdaptLow low_args(const AdaptPlan& plan, const hymoe_mat& x, const void* w, bool trans, const float* scale, float* low,
                  float* part, unsigned* amax, int R, int K) {
    AdaptLow a{};
    a.plan = plan;
    a.x = x.data;
    a.ldx = static_cast<size_t>(x.ld);
    a.w = w;
    a.scale = scale;
    a.low = low;
    a.part = part;
    a.amax = amax;
    a.K = K;
    a.R = R;
    a.vec_x = rows_vec(x.data, a.ldx, elem_bytes(x.type));
    a.vec_w = rows_vec(w, trans ? R : K, 2);
    return a;
}

cudaError_t run_low(const AdaptLow& a, const hymoe_mat& x, int type_w, bool trans, int T, int n, bool tc, int n_sms, cudaStream_t st) {
    if (!tc) return launch_adapt_low(a, x.type, type_w, trans, n_sms, st);
    AdaptMaps m;
    if (!encode_rows(&m.rows, x, T, a.K, kTcRows) ||
        !(trans ? encode_weights(&m, a.w, type_w, n, a.K, a.R, 64) : encode_weights(&m, a.w, type_w, n, a.R, a.K, adapt_rp(a.R))))
        return cudaErrorInvalidValue;
    return launch_adapt_low_tc(m, a, type_w, trans, n_sms, st);
}

cudaError_t run_wide(const AdaptPlan& plan, const float* low, const void* w, int type_w, bool trans, const hymoe_mat* base,
                     const hymoe_mat& out, int R, int N, int T, int n, bool tc, int n_sms, cudaStream_t st) {
    const size_t es = elem_bytes(out.type);
    AdaptWide a{};
    a.plan = plan;
    a.low = low;
    a.w = w;
    a.base = base ? base->data : nullptr;
    a.out = out.data;
    a.ldb = base ? static_cast<size_t>(base->ld) : 0;
    a.ldo = static_cast<size_t>(out.ld);
    a.N = N;
    a.R = R;
    a.in_place = base && base->data == out.data;
    if (tc) {
        AdaptMaps m;
        if (!encode_rows(&m.rows, base ? *base : out, T, N, kTcRows) ||
            !(trans ? encode_weights(&m, w, type_w, n, R, N, adapt_rp(R))
                    : encode_weights(&m, w, type_w, n, N, R, out.type == HYMOE_TYPE_F32 ? 64 : 128)))
            return cudaErrorInvalidValue;
        return launch_adapt_wide_tc(m, a, out.type, type_w, trans, n_sms, st);
    }
    a.vec_w = rows_vec(w, trans ? N : R, 2);
    a.vec_b = base ? rows_vec(base->data, a.ldb, es) : 0;
    a.vec_o = rows_vec(out.data, a.ldo, es);
    return launch_adapt_wide(a, out.type, type_w, trans, n_sms, st);
}

AdaptGrad grad_args(const AdaptPlan& plan, const float* low, const hymoe_mat& x, float* g, float* part, int n, int R, int M,
                    int gm, int gj) {
    AdaptGrad a{};
    a.plan = plan;
    a.low = low;
    a.x = x.data;
    a.ldx = static_cast<size_t>(x.ld);
    a.g = g;
    a.part = part;
    a.M = M;
    a.R = R;
    a.gm = gm;
    a.gj = gj;
    a.n = n;
    a.vec_x = rows_vec(x.data, a.ldx, elem_bytes(x.type));
    return a;
}

bool all_on(int dev, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (p && !entry_on_device(p, dev)) return false;
    return true;
}

}  // namespace

extern "C" hymoe_status hymoe_adapt(const hymoe_adapters* ad, const hymoe_mat* x, const int32_t* ids, uint32_t n_tokens,
                                    const hymoe_mat* base, const hymoe_mat* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    return adapt_call(ad, x, ids, n_tokens, base, out, workspace, workspace_bytes, stream, nullptr);
}

hymoe_status hymoe::adapt_call(const hymoe_adapters* ad, const hymoe_mat* x, const int32_t* ids, uint32_t n_tokens,
                               const hymoe_mat* base, const hymoe_mat* out, void* workspace, size_t workspace_bytes,
                               void* stream, int* err) {
    set_thread_error("");
    if (const char* why = adapters_problem(ad)) return entry_fail(HYMOE_ERR_INVALID_ARG, why);
    if (n_tokens == 0) return HYMOE_OK;
    if (const char* why = common_problem(ad, ids, n_tokens, workspace, workspace_bytes,
                                         adapt_layout(ad, n_tokens, false).bytes))
        return entry_fail(HYMOE_ERR_INVALID_ARG, why);
    const uint32_t T = n_tokens, I = ad->in_features, O = ad->out_features;
    if (!rows_ok(x, I, ad->type) || !rows_ok(out, O, ad->type) || (base && (!rows_ok(base, O, ad->type) || base->type != out->type)))
        return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_adapt: x and out must be matrices of the adapters' type or F32 "
                                                 "with ld >= their columns, base like out");
    const EntrySpan so = entry_span(out, T, O), sw = entry_span(workspace, workspace_bytes);
    const size_t wa = static_cast<size_t>(ad->n_adapters) * ad->rank * 2;
    const EntrySpan in[6] = {entry_span(x, T, I),
                             entry_span(ids, ids ? size_t(T) * 4 : 0),
                             entry_span(ad->a, wa * I),
                             entry_span(ad->b, wa * O),
                             entry_span(ad->scale, ad->scale ? size_t(ad->n_adapters) * 4 : 0),
                             base ? entry_span(base, T, O) : EntrySpan{0, 0}};
    for (int i = 0; i < 6; ++i)
        if ((entry_overlap(so, in[i]) && !(i == 5 && same_rows(base, out))) || entry_overlap(sw, in[i]) || entry_overlap(so, sw))
            return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_adapt: out or the workspace overlaps an argument");
    int dev = -1;
    if (current_device(&dev) != HYMOE_OK) return HYMOE_ERR_CUDA;
    if (!all_on(dev, {x->data, ids, ad->a, ad->b, ad->scale, base ? base->data : nullptr, out->data, workspace}))
        return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_adapt: every pointer must be memory of the current device");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int n = static_cast<int>(ad->n_adapters), R = static_cast<int>(ad->rank), t = static_cast<int>(T);
    const int n_sms = sm_count(dev);
    if (adapt_decodes(T, R)) {
        AdaptDecode d{};
        d.x = x->data;
        d.base = base ? base->data : nullptr;
        d.out = out->data;
        d.ids = ids;
        d.a = ad->a;
        d.b = ad->b;
        d.scale = ad->scale;
        d.ldx = static_cast<size_t>(x->ld);
        d.ldb = base ? static_cast<size_t>(base->ld) : 0;
        d.ldo = static_cast<size_t>(out->ld);
        d.n = n;
        d.R = R;
        d.K = static_cast<int>(I);
        d.N = static_cast<int>(O);
        d.ctas = T <= 16 ? 16 : 8;
        d.vec_x = rows_vec(x->data, 0, elem_bytes(x->type)) && (T == 1 || rows_vec(x->data, d.ldx, elem_bytes(x->type)));
        d.vec_a = rows_vec(ad->a, I, 2);
        d.vec_b = rows_vec(ad->b, R, 2);
        d.in_place = base && base->data == out->data;
        if (launch_adapt_decode(d, x->type, ad->type, out->type, t, st) != cudaSuccess)
            return entry_fail(HYMOE_ERR_CUDA, "hymoe_adapt: kernel launch failed");
        return HYMOE_OK;
    }
    // The tensor cores' kernels need TMA's alignment; mma.sync takes any rows, and fp32 ones of x.
    const bool aligned = T > kTcRows && weights_tma(ad);
    const bool tc_low = aligned && x->type == ad->type && rows_tma(x, I);
    const bool tc_wide = aligned && rows_tma(out, O) && (!base || rows_tma(base, O));
    const AdaptLayout l = adapt_layout(ad, T, false, tc_low || tc_wide ? kTcRows : kAdRows);
    char* ws = static_cast<char*>(workspace);
    AdaptPlan plan = plan_in(l, ws, false);
    if (err) plan.err = err;
    float* low = reinterpret_cast<float*>(ws + l.low);
    float* low_part = reinterpret_cast<float*>(ws + l.low_part);
    cudaError_t e = launch_plan_adapt(ids, t, n, plan, st);
    if (e == cudaSuccess) e = run_low(low_args(plan, *x, ad->a, false, ad->scale, low, low_part, nullptr, R, static_cast<int>(I)), *x, ad->type, false, t, n, tc_low, n_sms, st);
    if (e == cudaSuccess) e = run_wide(plan, low, ad->b, ad->type, false, base, *out, R, static_cast<int>(O), t, n, tc_wide, n_sms, st);
    if (e != cudaSuccess) return entry_fail(HYMOE_ERR_CUDA, "hymoe_adapt: kernel launch failed");
    return HYMOE_OK;
}

extern "C" hymoe_status hymoe_adapt_backward(const hymoe_adapters* ad, const hymoe_mat* x, const hymoe_mat* dy,
                                             const int32_t* ids, uint32_t n_tokens, const hymoe_mat* base,
                                             const hymoe_mat* dx, float* da, float* db, void* workspace,
                                             size_t workspace_bytes, void* stream) {
    set_thread_error("");
    if (const char* why = adapters_problem(ad)) return entry_fail(HYMOE_ERR_INVALID_ARG, why);
    const uint32_t T = n_tokens, I = ad->in_features, O = ad->out_features;
    const size_t wa = static_cast<size_t>(ad->n_adapters) * ad->rank;
    if (!entry_aligned(da, 4) || !entry_aligned(db, 4))
        return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_adapt_backward: da and db must be 4-byte aligned");
    if (T > 0) {
        if (const char* why = common_problem(ad, ids, T, workspace, workspace_bytes, adapt_layout(ad, T, true).bytes))
            return entry_fail(HYMOE_ERR_INVALID_ARG, why);
        if (!rows_ok(x, I, ad->type) || !rows_ok(dy, O, ad->type) || (dx && (!rows_ok(dx, I, ad->type) || dx->type != x->type)) ||
            (base && (!dx || !rows_ok(base, I, ad->type) || base->type != dx->type)))
            return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_adapt_backward: x and dy must be matrices of the adapters' "
                                                     "type or F32 with ld >= their columns, dx and base like x");
    }
    const EntrySpan outs[4] = {T > 0 && dx ? entry_span(dx, T, I) : EntrySpan{0, 0}, entry_span(da, da ? wa * I * 4 : 0),
                               entry_span(db, db ? wa * O * 4 : 0), entry_span(workspace, T > 0 ? workspace_bytes : 0)};
    const EntrySpan in[7] = {T > 0 ? entry_span(x, T, I) : EntrySpan{0, 0},
                             T > 0 ? entry_span(dy, T, O) : EntrySpan{0, 0},
                             entry_span(ids, ids ? size_t(T) * 4 : 0),
                             entry_span(ad->a, wa * I * 2),
                             entry_span(ad->b, wa * O * 2),
                             entry_span(ad->scale, ad->scale ? size_t(ad->n_adapters) * 4 : 0),
                             T > 0 && base ? entry_span(base, T, I) : EntrySpan{0, 0}};
    for (int i = 0; i < 4; ++i) {
        for (int j = i + 1; j < 4; ++j)
            if (entry_overlap(outs[i], outs[j]))
                return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_adapt_backward: outputs overlap");
        for (int j = 0; j < 7; ++j)
            if (entry_overlap(outs[i], in[j]) && !(i == 0 && j == 6 && same_rows(base, dx)))
                return entry_fail(HYMOE_ERR_INVALID_ARG, "hymoe_adapt_backward: an output overlaps an input");
    }
    int dev = -1;
    if (current_device(&dev) != HYMOE_OK) return HYMOE_ERR_CUDA;
    if (!all_on(dev, {T > 0 ? x->data : nullptr, T > 0 ? dy->data : nullptr, ids, ad->a, ad->b, ad->scale,
                      T > 0 && base ? base->data : nullptr, T > 0 && dx ? dx->data : nullptr, da, db, T > 0 ? workspace : nullptr}))
        return entry_fail(HYMOE_ERR_INVALID_ARG,
                          "hymoe_adapt_backward: every pointer must be memory of the current device");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int n = static_cast<int>(ad->n_adapters), R = static_cast<int>(ad->rank), t = static_cast<int>(T);
    if (T == 0) {
        if ((da && cudaMemsetAsync(da, 0, wa * I * 4, st) != cudaSuccess) ||
            (db && cudaMemsetAsync(db, 0, wa * O * 4, st) != cudaSuccess)) {
            cudaGetLastError();
            return entry_fail(HYMOE_ERR_CUDA, "hymoe_adapt_backward: cudaMemsetAsync failed");
        }
        return HYMOE_OK;
    }
    const int n_sms = sm_count(dev);
    const bool aligned = T > kTcRows && weights_tma(ad);
    const bool tc_x = aligned && x->type == ad->type && rows_tma(x, I), tc_dy = aligned && dy->type == ad->type && rows_tma(dy, O);
    const bool tc_grad = (!da || tc_x) && (!db || (tc_dy && entry_aligned(db, 16)));
    const bool tc_dx = aligned && dx && rows_tma(dx, I) && (!base || rows_tma(base, I));
    const AdaptLayout l = adapt_layout(ad, T, true, tc_x || tc_dy || tc_dx ? kTcRows : kAdRows);
    char* ws = static_cast<char*>(workspace);
    const AdaptPlan plan = plan_in(l, ws, true);
    float* low_dy = reinterpret_cast<float*>(ws + l.low);
    float* low_x = reinterpret_cast<float*>(ws + l.low2);
    float *low_part = reinterpret_cast<float*>(ws + l.low_part), *low_part2 = reinterpret_cast<float*>(ws + l.low_part2);
    float *part_a = reinterpret_cast<float*>(ws + l.part[0]), *part_b = reinterpret_cast<float*>(ws + l.part[1]);
    const int i = static_cast<int>(I), o = static_cast<int>(O);
    unsigned* amax = tc_grad && ad->type == HYMOE_TYPE_F16 ? plan.amax : nullptr;
    cudaError_t e = launch_plan_adapt(ids, t, n, plan, st);
    // the narrow products, dy's for dx and da and x's for db; as one launch where both are mma.sync's
    const AdaptLow by_dy = low_args(plan, *dy, ad->b, true, ad->scale, low_dy, low_part, amax, R, o);
    AdaptLow by_x = low_args(plan, *x, ad->a, false, ad->scale, low_x, low_part2, amax ? amax + n : nullptr, R, i);
    by_x.plan.counters += l.max_tiles * (l.tile_rows / kAdRows);
    const bool pair = (dx || da) && db && !tc_dy && !tc_x && x->type == dy->type;
    if (e == cudaSuccess && pair) e = launch_adapt_lows(by_dy, by_x, x->type, ad->type, n_sms, st);
    if (e == cudaSuccess && !pair && (dx || da)) e = run_low(by_dy, *dy, ad->type, true, t, n, tc_dy, n_sms, st);
    if (e == cudaSuccess && dx) e = run_wide(plan, low_dy, ad->a, ad->type, true, base, *dx, R, i, t, n, tc_dx, n_sms, st);
    if (e == cudaSuccess && !pair && db) e = run_low(by_x, *x, ad->type, false, t, n, tc_x, n_sms, st);
    // dA from x and dy's narrow rows, dB from dy and x's; long adapters in pieces
    AdaptGradPair grads;
    grads.g[0] = grad_args(plan, low_dy, *x, da, part_a, n, R, i, 1, i);
    grads.g[1] = grad_args(plan, low_x, *dy, db, part_b, n, R, o, R, 1);
    if (tc_grad) {
        const int wide = adapt_parts(adapt_rp(R));
        for (int k = 0; k < 2; ++k) {
            const hymoe_mat rows = k == 0 ? *x : *dy, low = {ws + l.low16[k], ad->type, wide};
            grads.parts[k] = low.data;
            if (grads.g[k].g && (!encode_rows(&grads.rows[k], rows, t, k == 0 ? i : o, 64) || !encode_rows(&grads.lows[k], low, t, wide, 64)))
                e = cudaErrorInvalidValue;
        }
        if (e == cudaSuccess && (da || db)) e = launch_adapt_grad_tc(grads, ad->type, st);
    } else if (x->type == dy->type) {
        if (e == cudaSuccess && (da || db)) e = launch_adapt_grad(grads.g[0], grads.g[1], x->type, st);
    } else {
        const AdaptGrad none{};
        if (e == cudaSuccess && da) e = launch_adapt_grad(grads.g[0], none, x->type, st);
        if (e == cudaSuccess && db) e = launch_adapt_grad(grads.g[1], none, dy->type, st);
    }
    if (e == cudaSuccess && (da || db) && t > adapt_chunk(t, n)) e = launch_adapt_join(grads.g[0], grads.g[1], st);
    if (e != cudaSuccess) return entry_fail(HYMOE_ERR_CUDA, "hymoe_adapt_backward: kernel launch failed");
    return HYMOE_OK;
}
