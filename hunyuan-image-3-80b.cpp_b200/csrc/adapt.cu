// adapt.cu — hymoe_adapt and hymoe_adapt_backward: low-rank adapters of many requests beside a
// projection they share, and their gradients.
//
//   low[t]  = scale[a] * A_a x[t]          (a = ids[t]; backward also scale[a] * B_a^T dy[t])
//   out[t]  = base[t] + B_a low[t]         (backward: dx[t] = base[t] + A_a^T low_dy[t])
//   dA_a    = sum_t low_dy[t] x[t]^T,  dB_a = sum_t dy[t] low_x[t]^T
#include <initializer_list>

#include "common.cuh"
#include "entry.h"

namespace hymoe {
namespace {

constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

__device__ __forceinline__ int adapter_of(const int* ids, int t, int n) {
    const int a = ids != nullptr ? __ldg(ids + t) : 0;
    return a >= 0 && a < n ? a : -1;
}

// low[t, j] = scale * sum_i x[t, i] W[a][j * wj + i * wi]; one warp per (token, j).
template <typename TX, typename TW>
__global__ void low_kernel(const TX* __restrict__ x, size_t ldx, const int* __restrict__ ids, int T, int n, int R,
                           int K, const TW* __restrict__ w, size_t wj, size_t wi, const float* __restrict__ scale,
                           float* __restrict__ low) {
    const size_t id = (static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
    const int t = static_cast<int>(id / R), j = static_cast<int>(id % R), lane = threadIdx.x & 31;
    if (t >= T) return;
    const int a = adapter_of(ids, t, n);
    float s = 0.f;
    if (a >= 0) {
        const TW* wr = w + static_cast<size_t>(a) * R * K + j * wj;
        for (int i = lane; i < K; i += 32) s = fmaf(to_f(x[t * ldx + i]), to_f(wr[i * wi]), s);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
        if (scale != nullptr) s *= __ldg(scale + a);
    }
    if (lane == 0) low[static_cast<size_t>(t) * R + j] = s;
}

// out[t, o] = base[t, o] + sum_j low[t, j] W[a][j * wj + o * wo]; one thread per element.
template <typename TY, typename TW>
__global__ void wide_kernel(const float* __restrict__ low, const int* __restrict__ ids, int T, int n, int R, int N,
                            const TW* __restrict__ w, size_t wj, size_t wo, const TY* base, size_t ldb, TY* out,
                            size_t ldo) {
    const size_t id = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int t = static_cast<int>(id / N), o = static_cast<int>(id % N);
    if (t >= T) return;
    const int a = adapter_of(ids, t, n);
    float s = 0.f;
    if (a >= 0) {
        const TW* wr = w + static_cast<size_t>(a) * R * N + o * wo;
        for (int j = 0; j < R; ++j) s = fmaf(low[static_cast<size_t>(t) * R + j], to_f(wr[j * wj]), s);
    }
    if (base != nullptr) s += to_f(base[t * ldb + o]);
    from_f(out[t * ldo + o], s);
}

// g[a][j * gj + m * gm] = sum over a's tokens of low[t, j] x[t, m]; one thread per element.
template <typename TX>
__global__ void outer_kernel(const float* __restrict__ low, const TX* __restrict__ x, size_t ldx,
                             const int* __restrict__ ids, int T, int n, int R, int M, float* __restrict__ g, size_t gj,
                             size_t gm) {
    const size_t id = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int m = static_cast<int>(id % M), j = static_cast<int>(id / M % R), a = static_cast<int>(id / M / R);
    if (a >= n) return;
    float s = 0.f;
    for (int t = 0; t < T; ++t)
        if (adapter_of(ids, t, n) == a) s = fmaf(low[static_cast<size_t>(t) * R + j], to_f(x[t * ldx + m]), s);
    g[static_cast<size_t>(a) * R * M + j * gj + m * gm] = s;
}

unsigned blocks(size_t threads) { return static_cast<unsigned>((threads + 255) / 256); }

template <typename TW>
cudaError_t run_low(const hymoe_mat& x, const int* ids, int T, int n, int R, int K, const void* w, size_t wj, size_t wi,
                    const float* scale, float* low, cudaStream_t st) {
    const TW* wp = static_cast<const TW*>(w);
    const unsigned g = blocks(static_cast<size_t>(T) * R * 32);
    if (x.type == HYMOE_TYPE_F32)
        low_kernel<float, TW><<<g, 256, 0, st>>>(static_cast<const float*>(x.data), x.ld, ids, T, n, R, K, wp, wj, wi, scale, low);
    else
        low_kernel<TW, TW><<<g, 256, 0, st>>>(static_cast<const TW*>(x.data), x.ld, ids, T, n, R, K, wp, wj, wi, scale, low);
    return cudaGetLastError();
}

template <typename TW>
cudaError_t run_wide(const float* low, const int* ids, int T, int n, int R, int N, const void* w, size_t wj, size_t wo,
                     const hymoe_mat* base, const hymoe_mat& out, cudaStream_t st) {
    const TW* wp = static_cast<const TW*>(w);
    const unsigned g = blocks(static_cast<size_t>(T) * N);
    const void* bp = base ? base->data : nullptr;
    const size_t ldb = base ? base->ld : 0;
    if (out.type == HYMOE_TYPE_F32)
        wide_kernel<float, TW><<<g, 256, 0, st>>>(low, ids, T, n, R, N, wp, wj, wo, static_cast<const float*>(bp), ldb,
                                                  static_cast<float*>(out.data), out.ld);
    else
        wide_kernel<TW, TW><<<g, 256, 0, st>>>(low, ids, T, n, R, N, wp, wj, wo, static_cast<const TW*>(bp), ldb,
                                               static_cast<TW*>(out.data), out.ld);
    return cudaGetLastError();
}

template <typename TW>
cudaError_t run_outer(const float* low, const hymoe_mat& x, const int* ids, int T, int n, int R, int M, float* g,
                      size_t gj, size_t gm, cudaStream_t st) {
    const unsigned b = blocks(static_cast<size_t>(n) * R * M);
    if (x.type == HYMOE_TYPE_F32)
        outer_kernel<float><<<b, 256, 0, st>>>(low, static_cast<const float*>(x.data), x.ld, ids, T, n, R, M, g, gj, gm);
    else
        outer_kernel<TW><<<b, 256, 0, st>>>(low, static_cast<const TW*>(x.data), x.ld, ids, T, n, R, M, g, gj, gm);
    return cudaGetLastError();
}

size_t low_bytes(const hymoe_adapters* ad, size_t T) { return (T * ad->rank * 4 + 255) / 256 * 256; }

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
    *bytes = low_bytes(ad, n_tokens) * (backward ? 2 : 1);
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

bool all_on(int dev, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (p && !entry_on_device(p, dev)) return false;
    return true;
}

}  // namespace

extern "C" hymoe_status hymoe_adapt(const hymoe_adapters* ad, const hymoe_mat* x, const int32_t* ids, uint32_t n_tokens,
                                    const hymoe_mat* base, const hymoe_mat* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    set_thread_error("");
    if (const char* why = adapters_problem(ad)) return entry_fail(HYMOE_ERR_INVALID_ARG, why);
    if (n_tokens == 0) return HYMOE_OK;
    if (const char* why = common_problem(ad, ids, n_tokens, workspace, workspace_bytes, low_bytes(ad, n_tokens)))
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
    float* low = static_cast<float*>(workspace);
    auto go = [&](auto tag) {
        using TW = decltype(tag);
        cudaError_t e = run_low<TW>(*x, ids, t, n, R, static_cast<int>(I), ad->a, I, 1, ad->scale, low, st);
        if (e == cudaSuccess) e = run_wide<TW>(low, ids, t, n, R, static_cast<int>(O), ad->b, 1, R, base, *out, st);
        return e;
    };
    const cudaError_t e = ad->type == HYMOE_TYPE_F16 ? go(__half{}) : go(__nv_bfloat16{});
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
        if (const char* why = common_problem(ad, ids, T, workspace, workspace_bytes, 2 * low_bytes(ad, T)))
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
    float* low_x = static_cast<float*>(workspace);
    float* low_dy = low_x + low_bytes(ad, T) / 4;
    const int i = static_cast<int>(I), o = static_cast<int>(O);
    auto go = [&](auto tag) {
        using TW = decltype(tag);
        cudaError_t e = cudaSuccess;
        if (db) e = run_low<TW>(*x, ids, t, n, R, i, ad->a, I, 1, ad->scale, low_x, st);
        if (e == cudaSuccess && (dx || da)) e = run_low<TW>(*dy, ids, t, n, R, o, ad->b, 1, R, ad->scale, low_dy, st);
        if (e == cudaSuccess && dx) e = run_wide<TW>(low_dy, ids, t, n, R, i, ad->a, I, 1, base, *dx, st);
        if (e == cudaSuccess && da) e = run_outer<TW>(low_dy, *x, ids, t, n, R, i, da, I, 1, st);
        if (e == cudaSuccess && db) e = run_outer<TW>(low_x, *dy, ids, t, n, R, o, db, 1, R, st);
        return e;
    };
    const cudaError_t e = ad->type == HYMOE_TYPE_F16 ? go(__half{}) : go(__nv_bfloat16{});
    if (e != cudaSuccess) return entry_fail(HYMOE_ERR_CUDA, "hymoe_adapt_backward: kernel launch failed");
    return HYMOE_OK;
}
