// entry.h — argument checks shared by the entry points that work on the caller's device
// buffers without a context (gate.cu, adapt.cu): no allocation, no device state.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/hymoe.h"

namespace hymoe {

// Thread-local message slot read by hymoe_last_error(NULL) (hymoe_api.cu).
void set_thread_error(const char* msg);

inline hymoe_status entry_fail(hymoe_status st, const char* msg) {
    set_thread_error(msg);
    return st;
}

// Bytes of one element of a plain (unblocked) type, 0 for any other.
inline size_t elem_bytes(int32_t type) {
    return type == HYMOE_TYPE_F32 ? 4 : type == HYMOE_TYPE_F16 || type == HYMOE_TYPE_BF16 ? 2 : 0;
}

// Memory the kernels, which run on the current device `dev`, may read and write directly:
// device memory of that device, or managed memory.
inline bool entry_on_device(const void* p, int dev) {
    cudaPointerAttributes a{};
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == dev);
}

inline bool entry_aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A row-major matrix argument of `cols` columns whose rows do not overlap.
inline bool entry_mat_ok(const hymoe_mat* m, uint32_t cols) {
    return m && m->data && elem_bytes(m->type) != 0 && m->ld >= static_cast<int64_t>(cols) &&
           m->ld < (int64_t(1) << 40) && entry_aligned(m->data, elem_bytes(m->type));
}

// Byte range [first, last) of a matrix of `rows` rows; used to refuse overlapping outputs.
struct EntrySpan {
    uintptr_t lo, hi;
};
inline EntrySpan entry_span(const void* p, size_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return {a, a + bytes};
}
inline EntrySpan entry_span(const hymoe_mat* m, uint32_t rows, uint32_t cols) {
    const size_t es = elem_bytes(m->type);
    return entry_span(m->data, rows == 0 ? 0 : (static_cast<size_t>(rows - 1) * m->ld + cols) * es);
}
inline bool entry_overlap(EntrySpan a, EntrySpan b) { return a.lo < b.hi && b.lo < a.hi; }

// hymoe_adapt with the word that an expired device-side wait sets (nullptr: the workspace's first).
hymoe_status adapt_call(const hymoe_adapters* ad, const hymoe_mat* x, const int32_t* ids, uint32_t n_tokens,
                        const hymoe_mat* base, const hymoe_mat* out, void* workspace, size_t workspace_bytes,
                        void* stream, int* err);

}  // namespace hymoe
