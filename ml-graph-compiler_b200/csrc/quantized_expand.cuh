// The values of a batch's visible positions as plain pages in a workspace: what calls with many query rows a
// key head attend over with the kernels for plain pages.
//
// A chunk's products (4 D operations a row and key) outweigh its keys' conversion, and the tensor cores take
// operands from shared memory or TMEM in 16 bits: converting each tile once a row tile of 256 would repeat it
// for every one of them. Once for all is a read of the codes and a write and a read of D values.
//
// Pages of `page` positions (the cache's page size or a divisor), one head's rows side by side; sequence b's
// positions from page * s on are page b * slots + s. Rows that no token sees are zero, so that whatever the cache
// holds there is not met again; a missing page stays missing. Values are halves, rounded once and held within
// half's range. 8 x 8192 positions of 8 heads x 128 in 4 bits (36 MB read, 268 MB written): 65 us, 4.7 TB/s.
#pragma once

#include "kv_read.cuh"
#include "quantized_mma.cuh"

namespace mgc {
namespace paged {

struct ExpandParams {
    QuantAttend a;
    Quantized z;
    __half *k, *v;      // [batch * slots][heads][page][head_dim]
    int32_t *table;     // [batch][slots]
    int32_t *kv_lens;   // [batch]: 0 for sequences that are left to the kernels for codes
    int slots, page, h0, heads;
    uint32_t code_page, code_token, pair_page, pair_token;  // QuantParams's
    int per_page;                        // pages of `page` positions in one of the cache's
    uint32_t per_magic, page_magic;      // x / per_page = x * per_magic >> per_shift; r / page = r * page_magic >> 16, r < 256
    int per_shift;
};

// Eight codes' values in order, by one fused operation each (rounded once), held within half's range.
template <int BITS> __device__ __forceinline__ void expand_eight(const EightCodes<BITS> &c, __half2 so, __half *dst) {
    const __half2 s = __low2half2(so), o = __high2half2(so), most = __float2half2_rn(65504.0f), least = __float2half2_rn(-65504.0f);
    auto value = [&](uint32_t code, uint32_t bias) {  // of a pair of codes in the mantissas of 1024 or 64
        const __half2 v = __hfma2(s, __hsub2(*reinterpret_cast<__half2 *>(&code), *reinterpret_cast<__half2 *>(&bias)), o);
        const __half2 h = __hmax2_nan(__hmin2_nan(v, most), least);
        return *reinterpret_cast<const uint32_t *>(&h);
    };
    uint4 y;
    if constexpr (BITS == 4) {
        const uint32_t a = value(and_or(c.w, 0x000F000Fu, 0x64006400u), 0x64006400u);       // channels 0, 4
        const uint32_t b = value(and_or(c.w, 0x00F000F0u, 0x54005400u), 0x54005400u);       // 1, 5
        const uint32_t d = value(and_or(c.w >> 8, 0x000F000Fu, 0x64006400u), 0x64006400u);  // 2, 6
        const uint32_t e = value(and_or(c.w >> 8, 0x00F000F0u, 0x54005400u), 0x54005400u);  // 3, 7
        y = make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(d, e, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(d, e, 0x7632));
    } else {
        const uint32_t bias = 0x64006400u;
        y = make_uint4(value(__byte_perm(c.w.x, 0x64646464u, 0x4140), bias), value(__byte_perm(c.w.x, 0x64646464u, 0x4342), bias),
                       value(__byte_perm(c.w.y, 0x64646464u, 0x4140), bias), value(__byte_perm(c.w.y, 0x64646464u, 0x4342), bias));
    }
    *reinterpret_cast<uint4 *>(dst) = y;
}

constexpr int EXPAND_ROWS = 4;  // of a thread, in flight together

// Block (64 positions, or one page of more; head; sequence): a thread takes eight channels of every few rows.
template <int BITS>
__global__ void __launch_bounds__(256) quantized_expand_kernel(const __grid_constant__ ExpandParams p) {
    const int h = (int)blockIdx.y, b = (int)blockIdx.z, tid = (int)threadIdx.x, kh = p.h0 + h;
    const Sequence seq = load_sequence(static_cast<const AttendParams &>(p.a), b);
    const bool mine = seq.nq > 0 && left_out(p.a, seq);
    if (tid == 0 && blockIdx.x == 0 && h == 0 && p.h0 == 0) p.kv_lens[b] = mine ? __ldg(p.a.batch.kv_lens + b) : 0;
    int lo = 0, hi = 0, other;
    if (mine) {
        visible(p.a, seq.n, seq.base, lo, other);
        visible(p.a, seq.n, seq.base + seq.nq - 1, other, hi);
    }
    const int rows = p.page < 64 ? 64 / p.page * p.page : p.page, s0 = (int)blockIdx.x * (rows / p.page);
    const int32_t *table = p.a.batch.table + (long long)b * p.a.batch.table_stride;
    // source page of slot s, -1 if it is missing or no row sees it
    auto source = [&](int s) {
        const int j = s * p.page;
        if (s >= p.slots || j >= hi || j + p.page <= lo) return -1;
        const int page = __ldg(table + (int)((unsigned long long)(unsigned)s * p.per_magic >> p.per_shift));
        return page < 0 || page >= p.a.batch.pages ? -1 : page;
    };
    if (h == 0 && p.h0 == 0 && tid < rows / p.page && s0 + tid < p.slots)
        p.table[(long long)b * p.slots + s0 + tid] = source(s0 + tid) < 0 ? -1 : b * p.slots + s0 + tid;
    const int j0 = s0 * p.page;
    if (j0 >= hi || j0 + rows <= lo) return;
    const int chunks = p.a.head_dim / 8, at_once = 256 / chunks, c = tid % chunks, group = 8 * c / p.z.group;
    if (tid >= at_once * chunks) return;
    const uint8_t *k_pages = static_cast<const uint8_t *>(p.a.k_pages) + kh * p.a.head_stride + c * BITS;
    const uint8_t *v_pages = static_cast<const uint8_t *>(p.a.v_pages) + kh * p.a.head_stride + c * BITS;
    const __half2 *k_pairs = p.z.k_scales + kh * p.z.head_stride + group, *v_pairs = p.z.v_scales + kh * p.z.head_stride + group;
    for (int r0 = tid / chunks; r0 < rows; r0 += EXPAND_ROWS * at_once) {
        EightCodes<BITS> code[EXPAND_ROWS][2];
        __half2 so[EXPAND_ROWS][2];
        int to[EXPAND_ROWS];  // row of the plain pages, counted from the block's first; -1: none
#pragma unroll
        for (int i = 0; i < EXPAND_ROWS; ++i) {
            const int r = r0 + i * at_once, ds = (int)((uint32_t)r * p.page_magic >> 16), row = r - ds * p.page, slot = s0 + ds, j = j0 + r;
            const int page = r < rows ? source(slot) : -1;
            to[i] = page < 0 ? -1 : ds * p.heads * p.page + row;
            code[i][0] = code[i][1] = EightCodes<BITS>{};
            so[i][0] = so[i][1] = __floats2half2_rn(0.0f, 0.0f);
            if (page >= 0 && j >= lo && j < hi) {
                const int in_page = row + (slot - (int)((unsigned long long)(unsigned)slot * p.per_magic >> p.per_shift) * p.per_page) * p.page;
                const unsigned long long at = (unsigned long long)(unsigned)page * p.code_page + (uint32_t)in_page * p.code_token;
                const unsigned long long pair = (unsigned long long)(unsigned)page * p.pair_page + (uint32_t)in_page * p.pair_token;
                code[i][0].load(k_pages + at);
                code[i][1].load(v_pages + at);
                so[i][0] = __ldg(k_pairs + pair);
                so[i][1] = __ldg(v_pairs + pair);
            }
        }
        const long long first = (((long long)b * p.slots + s0) * p.heads + h) * p.page;
#pragma unroll
        for (int i = 0; i < EXPAND_ROWS; ++i) {
            if (to[i] < 0) continue;
            expand_eight<BITS>(code[i][0], so[i][0], p.k + (first + to[i]) * p.a.head_dim + c * 8);
            expand_eight<BITS>(code[i][1], so[i][1], p.v + (first + to[i]) * p.a.head_dim + c * 8);
        }
    }
}

}  // namespace paged
}  // namespace mgc
