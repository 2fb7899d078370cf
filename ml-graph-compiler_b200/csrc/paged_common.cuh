// What the paged-cache operators share: element conversions, the batch description on the device,
// argument checks (the layout is described at mgc_cuda_paged in mgc_cuda.h).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mgc {
namespace paged {

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// V consecutive elements moved in the widest accesses their bytes allow (up to 16).
template <int BYTES> struct Raw;
template <> struct Raw<2> { using t = unsigned short; };
template <> struct Raw<4> { using t = uint32_t; };
template <> struct Raw<8> { using t = uint2; };
template <> struct Raw<16> { using t = uint4; };

template <int V, typename T> struct Pack {
    static constexpr int BYTES = V * (int)sizeof(T) > 16 ? 16 : V * (int)sizeof(T);
    static constexpr int N = V * (int)sizeof(T) / BYTES;
    using R = typename Raw<BYTES>::t;
    union {
        R raw[N];
        T e[V];
    };
    __device__ __forceinline__ Pack() {}
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int k = 0; k < N; ++k) raw[k] = reinterpret_cast<const R *>(p)[k];
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int k = 0; k < N; ++k) reinterpret_cast<R *>(p)[k] = raw[k];
    }
};

// The batch description as the kernels take it.
struct Batch {
    const int32_t *table, *kv_lens, *q_starts;
    long long table_stride;
    int table_pages, pages, page_size, batch;
    int *status;
};

// Sequence of packed token t: the last b with q_starts[b] <= t (sequences without tokens share
// their successor's start). One warp counts the starts at or below t, 32 at a time.
__device__ __forceinline__ int sequence_of(const Batch &d, int t) {
    int b = -1;
    for (int base = 0; base < d.batch; base += 32) {
        const int i = base + (int)(threadIdx.x & 31);
        const unsigned below = __ballot_sync(0xFFFFFFFFu, i < d.batch && __ldg(d.q_starts + i) <= t);
        b += __popc(below);
        if (below != 0xFFFFFFFFu) break;
    }
    return b;
}

// Page that holds position p of sequence b, or -1 (and the status word set) if the table has none.
__device__ __forceinline__ int page_of(const Batch &d, int b, int slot) {
    int page = -1;
    if (slot >= 0 && slot < d.table_pages) page = __ldg(d.table + (long long)b * d.table_stride + slot);
    if (page < 0 || page >= d.pages) {
        if (d.status) *d.status = MGC_CUDA_GATHER_OOB;
        page = -1;
    }
    return page;
}

inline bool dtype_ok(int64_t dt) { return dt == MGC_F32 || dt == MGC_F16 || dt == MGC_BF16; }
inline int elem_size(int64_t dt) { return dt == MGC_F32 ? 4 : 2; }
inline bool aligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (unsigned)bytes == 0; }

// Checks of the fields both operators read; `what` names the entry point.
inline int check_paged(const mgc_cuda_paged &a, const char *what) {
    if (!a.k || !a.v || (a.batch > 0 && ((a.table_pages > 0 && !a.block_table) || !a.kv_lens || !a.q_starts)))
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: a cache or batch pointer is NULL", what);
    if (!dtype_ok(a.dtype)) return fail(MGC_CUDA_UNSUPPORTED, "%s: pages of type %d", what, (int)a.dtype);
    if (a.kv_heads < 1 || a.head_dim < 1 || a.page_size < 1 || a.pages < 1 || a.batch < 0 || a.tokens < 0 ||
        a.table_pages < 0 || a.table_stride < 0)
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: a size is negative or zero", what);
    const int64_t most = 0x7FFFFFFF;
    if (a.pages > most || a.page_size > most || a.batch > most - 1 || a.tokens > most || a.kv_heads > 65535 ||
        a.table_pages > most / a.page_size)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: a size does not fit 32 bits", what);
    if (a.page_stride < 0 || a.token_stride < 0 || a.head_stride < 0)
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: a cache stride is negative", what);
    return MGC_CUDA_OK;
}

inline Batch batch_of(const mgc_cuda_paged &a) {
    Batch d;
    d.table = a.block_table;
    d.kv_lens = a.kv_lens;
    d.q_starts = a.q_starts;
    d.table_stride = a.table_stride;
    d.table_pages = (int)a.table_pages;
    d.pages = (int)a.pages;
    d.page_size = (int)a.page_size;
    d.batch = (int)a.batch;
    d.status = a.status_dev;
    return d;
}

}  // namespace paged
}  // namespace mgc
