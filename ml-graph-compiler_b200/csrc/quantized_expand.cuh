// The values of a batch's visible positions as plain pages in a workspace: what calls with many query rows a
// key head attend over with the kernels for plain pages.
//
// A chunk's products (4 D operations a row and key) outweigh its keys' conversion, and the tensor cores take
// operands from shared memory or TMEM in 16 bits: converting each tile once a row tile of 256 would repeat it
// for every one of them. Once for all is a read of the codes and a write and a read of D values.
//
// Pages of `page` positions (the cache's page size or a divisor), one head's rows side by side; sequence b's
// positions from page * s on are page b * slots + s. Rows that no token sees are zero, so that whatever the cache
// holds there is not met again; a missing page stays missing. Values are fp32, rounded once to the pages' type:
// fp32, or half for 16-bit queries, held within its range.
#pragma once

#include "kv_read.cuh"
#include "quantized_mma.cuh"

namespace mgc {
namespace paged {

struct ExpandParams {
    QuantAttend a;
    Quantized z;
    void *k, *v;        // [batch * slots][heads][page][head_dim]
    int32_t *table;     // [batch][slots]
    int32_t *kv_lens;   // [batch]: 0 for sequences that are left to the kernels for codes
    int slots, page, h0, heads;
};

template <typename T> __device__ __forceinline__ T held(float x) { return from_f<T>(x); }
template <> __device__ __forceinline__ __half held(float x) { return from_f<__half>(x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x); }

// Block (slot, head, sequence).
template <typename T, int BITS>
__global__ void __launch_bounds__(256) quantized_expand_kernel(const __grid_constant__ ExpandParams p) {
    const int slot = (int)blockIdx.x, h = (int)blockIdx.y, b = (int)blockIdx.z;
    const Sequence seq = load_sequence(static_cast<const AttendParams &>(p.a), b);
    const bool mine = seq.nq > 0 && left_out(p.a, seq);
    if (threadIdx.x == 0 && slot == 0 && h == 0 && p.h0 == 0) p.kv_lens[b] = mine ? __ldg(p.a.batch.kv_lens + b) : 0;
    int lo = 0, hi = 0, top, bottom;
    if (mine) {
        visible(p.a, seq.n, seq.base, lo, top);
        visible(p.a, seq.n, seq.base + seq.nq - 1, bottom, hi);
    }
    const int j0 = slot * p.page;
    int page = -1;
    const int ps = p.a.batch.page_size;
    if (j0 < hi && j0 + p.page > lo) {
        page = __ldg(p.a.batch.table + (long long)b * p.a.batch.table_stride + j0 / ps);
        if (page < 0 || page >= p.a.batch.pages) page = -1;
    }
    const long long to = (long long)b * p.slots + slot;
    if (threadIdx.x == 0 && h == 0 && p.h0 == 0) p.table[to] = page < 0 ? -1 : (int)to;
    if (page < 0) return;
    const int first = j0 % ps, kh = p.h0 + h, chunks = p.a.head_dim / 8;
    const long long codes = (long long)page * p.a.page_stride + kh * p.a.head_stride;
    const long long pairs = (long long)page * p.z.page_stride + kh * p.z.head_stride;
    const long long row0 = (to * p.heads + h) * p.page;
    for (int x = (int)threadIdx.x; x < p.page * chunks; x += 256) {
        const int r = x / chunks, c = x - r * chunks, j = j0 + r;
        const bool seen = j >= lo && j < hi;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            Pack<8, T> y;
            if (seen) {
                float code[8];
                eight_codes<BITS>(static_cast<const uint8_t *>(kv ? p.a.v_pages : p.a.k_pages) + codes + (first + r) * p.a.token_stride + c * BITS, code);
                const float2 so = __half22float2((kv ? p.z.v_scales : p.z.k_scales)[pairs + (first + r) * p.z.token_stride + 8 * c / p.z.group]);
#pragma unroll
                for (int i = 0; i < 8; ++i) y.e[i] = held<T>(fmaf(so.x, code[i], so.y));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y.e[i] = from_f<T>(0.0f);
            }
            y.store(static_cast<T *>(kv ? p.v : p.k) + (row0 + r) * p.a.head_dim + c * 8);
        }
    }
}

}  // namespace paged
}  // namespace mgc
