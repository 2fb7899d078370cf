// Attention of new tokens over quantised pages (quantized_common.cuh): paged_attention_params.cuh's
// definition with k_j and v_j the values that the codes stand for. The choice of kernels and the launch.
//
// Few query rows a key head attend over the codes (quantized_mma.cuh), and fp32 ones always. Of 16-bit calls with
// many, the values of sequences with many rows are written to plain half pages in the workspace first
// (quantized_expand.cuh) and the kernels for plain pages attend over them; key heads some at a time where the
// workspace would be large.
#pragma once

#include "quantized_expand.cuh"

namespace mgc {
namespace paged {

inline int check_attend_quantized(const mgc_cuda_paged_attention_quantized_args &a, const char *what) {
    const mgc_cuda_paged &c = a.attention.paged;
    MGC_CHECK(check_attend(a.attention, what));
    MGC_CHECK(check_quantized(a.quantized, c, what));
    // the kernel multiplies strides by page numbers and rows in 32 bits
    const int64_t most = 0xFFFFFFFFll;
    auto fits = [&](int64_t page, int64_t token) { return page <= most && token <= most / c.page_size; };
    if (!fits(c.page_stride, c.token_stride) || !fits(a.quantized.page_stride, a.quantized.token_stride))
        return fail(MGC_CUDA_UNSUPPORTED, "%s: a page does not fit 32 bits", what);
    return MGC_CUDA_OK;
}

// How a call runs.
struct QuantPlan {
    int nb = 1;          // eights of query rows of a unit
    int row_tiles = 1, splits = 1;  // CTAs of a cluster that share a unit's keys
    bool even = false, interleaved = false;
    int ctas = 0, live_rows = 1;
    int64_t workspace = 0;  // of the part over codes
    // the part over plain pages: 0 heads if there is none
    int heads = 0;          // key heads at a time
    int page = 0, slots = 0;
    int rows_left = 0;      // sequences of more query rows a key head are its
    int64_t pages_bytes = 0, inner = 0;  // of k or v; of the attention over them
    bool rest = true;       // the part over codes may have sequences
    int64_t index_bytes = 0;  // of block table and lengths
    int64_t total() const { return heads ? 2 * pages_bytes + index_bytes + inner + workspace : workspace; }
};

// Sequences with more query rows a key head than this take the way over plain pages, where a call has one.
constexpr int64_t DIRECT_ROWS = 64;
constexpr int64_t EXPANDED_BYTES = 1ll << 30;  // of plain pages at a time

inline int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

// The call of the attention over plain pages for key heads [h0, h0 + heads).
inline mgc_cuda_paged_attention_args expanded_args(const mgc_cuda_paged_attention_args &a, const QuantPlan &s, int h0, int heads, char *at) {
    mgc_cuda_paged_attention_args x = a;
    mgc_cuda_paged &c = x.paged;
    const int es = elem_size(c.dtype), group = (int)(a.q_heads / c.kv_heads);
    if (c.dtype == MGC_BF16) c.dtype = MGC_F16;
    c.k = at;
    c.v = at + s.pages_bytes;
    c.pages = c.batch * s.slots;
    c.kv_heads = heads;
    c.page_size = s.page;
    c.token_stride = c.head_dim;
    c.head_stride = c.head_dim * s.page;
    c.page_stride = c.head_stride * heads;
    c.block_table = reinterpret_cast<int32_t *>(at + 2 * s.pages_bytes);
    c.table_stride = c.table_pages = s.slots;
    c.kv_lens = c.block_table + c.batch * s.slots;
    x.q = static_cast<const char *>(a.q) + (int64_t)h0 * group * a.q_head_stride * es;
    x.out = static_cast<char *>(a.out) + (int64_t)h0 * group * a.o_head_stride * es;
    x.q_heads = (int64_t)heads * group;
    x.workspace = at + 2 * s.pages_bytes + s.index_bytes;
    x.workspace_bytes = s.inner;
    return x;
}

inline int width_of(int64_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Calls `go` with the configuration of a type, width, row tile and grouping.
template <int BITS, typename F> inline auto with_config(int64_t dtype, const mgc_cuda_quantized &z, int64_t head_dim, int nb, F go) {
    auto widths = [&](auto type) {
        using T = decltype(type);
        const int dp = width_of(head_dim);
        if (dp == 64) return nb > 1 ? go(QuantConfig<T, BITS, 64, 2, true>()) : go(QuantConfig<T, BITS, 64, 1, true>());
        const bool one = z.group == head_dim;
        if (dp == 256) return one ? go(QuantConfig<T, BITS, 256, 1, true>()) : go(QuantConfig<T, BITS, 256, 1, false>());
        if (one) return nb > 1 ? go(QuantConfig<T, BITS, 128, 2, true>()) : go(QuantConfig<T, BITS, 128, 1, true>());
        return nb > 1 ? go(QuantConfig<T, BITS, 128, 2, false>()) : go(QuantConfig<T, BITS, 128, 1, false>());
    };
    if (dtype == MGC_F32) return widths(float());
    return dtype == MGC_F16 ? widths(__half()) : widths(__nv_bfloat16());
}

inline QuantPlan quant_plan_of(const mgc_cuda_paged_attention_quantized_args &a) {
    const mgc_cuda_paged &c = a.attention.paged;
    QuantPlan s;
    const int64_t group = a.attention.q_heads / c.kv_heads;
    const int64_t max_q = a.attention.max_q < 1 ? 1 : a.attention.max_q > c.tokens ? c.tokens : a.attention.max_q;
    const int64_t rows = max_q * group;
    s.nb = rows <= 8 || c.head_dim > 128 ? 1 : 2;
    const int unit_rows = 8 * s.nb;
    s.row_tiles = (int)ceil_div(rows, unit_rows);
    s.live_rows = (int)(rows < unit_rows ? rows : unit_rows);
    const int64_t units = c.batch * c.kv_heads * s.row_tiles;
    const int64_t capacity = c.table_pages * c.page_size;
    int64_t most = a.attention.max_kv < capacity ? a.attention.max_kv : capacity;
    if (a.attention.window > 0 && a.attention.window + max_q < most) most = a.attention.window + max_q;
    // the kernel that adds pieces stores four elements at once
    const int es = elem_size(c.dtype);
    const bool wide = aligned(a.attention.out, 4 * es) && a.attention.o_token_stride % 4 == 0 && a.attention.o_head_stride % 4 == 0;
    auto held = [](auto config) { return decltype(config)::RESIDENT; };
    const int resident = a.quantized.bits == 4 ? with_config<4>(c.dtype, a.quantized, c.head_dim, s.nb, held)
                                               : with_config<8>(c.dtype, a.quantized, c.head_dim, s.nb, held);
    const int64_t slots = (int64_t)sm_count() * resident;
    // Few units: up to 8 CTAs of a cluster take equal parts of a unit's keys (one sequence of 1000 keys, 8 key heads of 128:
    // 8.7 us, even shares 11.4). From an eighth of the GPU's blocks on clusters wait for room on one part of the GPU
    // (16 x 500 keys of 12 key heads 15.9 us, a block a unit 9.7).
    int64_t splits = units * 8 <= slots ? MAX_CLUSTER : 1;
    if (splits > ceil_div(most, 128)) splits = most < 1 ? 1 : ceil_div(most, 128);
    s.splits = (int)splits;
    // Even shares leave no SM idle when sequences differ or 8 parts are too few; their second kernel and the pieces' way
    // through memory take some 500 keys' worth of time
    if (wide && most / splits > 512 + most * units / slots) {
        s.splits = 1;
        s.even = true;
        s.ctas = (int)slots;
        if (slots >= c.kv_heads && slots / c.kv_heads * c.kv_heads * 20 >= slots * 19) {
            s.interleaved = true;
            s.ctas = (int)(slots / c.kv_heads * c.kv_heads);
        }
        s.workspace = (int64_t)s.ctas * (2 * unit_rows * (c.head_dim * 4 + 8) + (int64_t)sizeof(CutUnit));
    }
    // Over plain pages: rows of 16 bytes are what those kernels take. bf16 queries go over half pages, in the tcgen05
    // kernel only: values rounded to bf16 once more left 0.5 % of error in the output of 4-bit pages, half 0.17 %, which is
    // bf16's own rounding of the output. fp32 codes take two products a value where plain fp32 pages take three of half
    // the depth: 96 rows over 8 x 2048 keys of 8 heads (8 bits) 97 and 349 us.
    auto rows16 = [&](const void *q, int64_t x, int64_t y) { return aligned(q, 16) && x * es % 16 == 0 && y * es % 16 == 0; };
    if (rows <= DIRECT_ROWS || c.dtype == MGC_F32 || !rows16(a.attention.q, a.attention.q_token_stride, a.attention.q_head_stride) ||
        !rows16(a.attention.out, a.attention.o_token_stride, a.attention.o_head_stride) ||
        (c.dtype == MGC_BF16 && (c.head_dim > 128 || c.page_size % 8)))
        return s;
    // In 10 ps at 128 channels, measured over 1 to 32 sequences of 500 to 8192 keys: a key of a key head takes 7 for 16 rows
    // over codes, 12 to be expanded and 18 for 256 rows over plain pages, whose four kernels take 25 us for a start.
    const double keys = (double)c.batch * (double)most * (double)c.kv_heads * width_of(c.head_dim) / 128;
    if (7 * keys * (double)ceil_div(rows, 16) < 2.5e6 + keys * (12 + 18 * (double)ceil_div(rows, 256))) return s;
    // Plain pages of the cache's size, or of a divisor that the tcgen05 kernel takes (paged_umma.cuh): 128, or a power of
    // two from 8 to 64
    int64_t page = c.page_size;
    if (page % 128 == 0) page = 128;
    else if (page % 8 == 0) page &= -page;
    const int64_t longest = a.attention.max_kv < capacity ? (a.attention.max_kv < 1 ? 1 : a.attention.max_kv) : capacity;
    const int64_t per_seq = ceil_div(longest, page);
    const int64_t head_bytes = c.batch * per_seq * page * c.head_dim * es;
    if (capacity == 0 || c.batch > 65535 || 2 * head_bytes > EXPANDED_BYTES || c.batch * per_seq > 0x7FFFFFFF) return s;
    int64_t heads = EXPANDED_BYTES / (2 * head_bytes);
    s.heads = (int)(heads > c.kv_heads ? c.kv_heads : heads);
    s.page = (int)page;
    s.slots = (int)per_seq;
    s.rows_left = c.batch > 1 ? (int)DIRECT_ROWS : 0;
    s.rest = c.batch > 1 || per_seq * page < capacity;
    s.pages_bytes = up256(head_bytes * s.heads);
    s.index_bytes = up256(4 * (c.batch * per_seq + c.batch));
    if (!s.rest) s.workspace = 0;
    // (the heads of the last pass may be fewer)
    for (int h0 = 0; h0 < c.kv_heads; h0 += s.heads) {
        const int n = (int)(c.kv_heads - h0 < s.heads ? c.kv_heads - h0 : s.heads);
        const mgc_cuda_paged_attention_args x = expanded_args(a.attention, s, h0, n, reinterpret_cast<char *>(256));
        const int64_t bytes = up256(mgc_cuda_paged_attention_workspace(&x));
        if (bytes > s.inner) s.inner = bytes;
    }
    return s;
}

inline int64_t attend_quantized_workspace(const mgc_cuda_paged_attention_quantized_args &a) {
    if (check_attend_quantized(a, "mgc_cuda_paged_attention_quantized_workspace") != MGC_CUDA_OK) return -1;
    return a.attention.paged.tokens == 0 || a.attention.paged.batch == 0 ? 0 : quant_plan_of(a).total();
}

// The kernels for codes of BITS bits, compiled in files of their own (quantized_4.cu, quantized_8.cu).
template <int BITS> int launch_codes(const QuantParams &p, const QuantPlan &s, int64_t dtype, const mgc_cuda_quantized &z, cudaStream_t stream);

// x / d = x * magic >> shift for 0 <= x < 2^31: with s = ceil(log2 d), ceil(2^(31 + s) / d) fits 32 bits and is exact.
inline void division(int64_t d, uint32_t &magic, int &shift) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    shift = 31 + s;
    magic = (uint32_t)(((1ull << shift) + (uint64_t)d - 1) / (uint64_t)d);
}

// The sequences that are expanded: values to plain pages, attention over them, some key heads at a time.
inline int attend_expanded(const mgc_cuda_paged_attention_args &a, const QuantParams &p, const QuantPlan &s, char *space, cudaStream_t stream) {
    const mgc_cuda_paged &c = a.paged;
    for (int h0 = 0; h0 < p.a.kv_heads; h0 += s.heads) {
        const int n = p.a.kv_heads - h0 < s.heads ? p.a.kv_heads - h0 : s.heads;
        const mgc_cuda_paged_attention_args x = expanded_args(a, s, h0, n, space);
        ExpandParams e;
        e.a = p.a;
        e.z = p.z;
        e.k = static_cast<__half *>(x.paged.k);
        e.v = static_cast<__half *>(x.paged.v);
        e.table = const_cast<int32_t *>(x.paged.block_table);
        e.kv_lens = const_cast<int32_t *>(x.paged.kv_lens);
        e.slots = s.slots;
        e.page = s.page;
        e.code_page = p.code_page;
        e.code_token = p.code_token;
        e.pair_page = p.pair_page;
        e.pair_token = p.pair_token;
        e.per_page = p.a.batch.page_size / s.page;
        division(e.per_page, e.per_magic, e.per_shift);
        e.page_magic = s.page > 128 ? 0 : (uint32_t)(65536 / s.page + (65536 % s.page != 0));
        e.h0 = h0;
        e.heads = n;
        const dim3 grid((unsigned)ceil_div(s.slots, s.page < 64 ? 64 / s.page : 1), (unsigned)n, (unsigned)c.batch);
        if (p.z.bits == 4) quantized_expand_kernel<4><<<grid, 256, 0, stream>>>(e);
        else quantized_expand_kernel<8><<<grid, 256, 0, stream>>>(e);
        MGC_CHECK(check_launch("quantized_expand_kernel"));
        MGC_CHECK(attend(x, c.dtype, stream));
    }
    return MGC_CUDA_OK;
}

inline int attend_quantized(const mgc_cuda_paged_attention_quantized_args &a, cudaStream_t stream) {
    const char *what = "mgc_cuda_paged_attention_quantized";
    const mgc_cuda_paged_attention_args &b = a.attention;
    const mgc_cuda_paged &c = b.paged;
    MGC_CHECK(check_attend_quantized(a, what));
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
    QuantParams p;
    static_cast<AttendParams &>(p.a) = attend_params(b);
    p.z = quantized_of(a.quantized, c);
    const QuantPlan s = quant_plan_of(a);
    if (c.tokens * p.a.group >= 0x80000000ll - 256 || c.batch * c.kv_heads * s.row_tiles > 0x7FFFFFFF)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: %lld tokens of %d heads a key head", what, (long long)c.tokens, p.a.group);
    p.a.row_tiles = s.row_tiles;
    p.a.interleaved = s.interleaved;
    p.a.splits = s.splits;
    if (s.total() && (!b.workspace || b.workspace_bytes < s.total() || !aligned(b.workspace, 16)))
        return fail(MGC_CUDA_NEEDS_WORKSPACE, "%s: needs %lld bytes of workspace (16-byte aligned), got %lld", what,
                    (long long)s.total(), (long long)(b.workspace ? b.workspace_bytes : 0));
    division(c.page_size, p.page_magic, p.page_shift);
    p.code_page = (uint32_t)c.page_stride;
    p.code_token = (uint32_t)c.token_stride;
    p.pair_page = (uint32_t)a.quantized.page_stride;
    p.pair_token = (uint32_t)a.quantized.token_stride;
    char *space = static_cast<char *>(b.workspace);
    p.a.rows_left = s.rows_left;
    p.a.kv_left = s.heads ? s.slots * s.page : 0;
    if (s.heads) {
        MGC_CHECK(attend_expanded(b, p, s, space, stream));
        if (!s.rest) return MGC_CUDA_OK;
        space += s.total() - s.workspace;
    }
    if (s.workspace) {
        const int64_t rows = (int64_t)s.ctas * 16 * s.nb;
        p.a.part = reinterpret_cast<float *>(space);
        p.a.part_ml = reinterpret_cast<float2 *>(p.a.part + rows * p.a.head_dim);
        p.a.cut = reinterpret_cast<CutUnit *>(p.a.part_ml + rows);
    }
    const int chunk = 16 / elem_size(c.dtype);
    p.slabs = (int)ceil_div(c.head_dim, 64);
    for (int x = 0; x < 4; ++x) p.group_of[x] = 64 * x < p.a.head_dim ? 64 * x / p.z.group : 0;
    p.pairs_wide = p.z.groups == 2 && c.head_dim == 128 && aligned(p.z.k_scales, 8) && aligned(p.z.v_scales, 8) &&
                   p.z.page_stride % 2 == 0 && p.z.token_stride % 2 == 0 && p.z.head_stride % 2 == 0;
    p.q_wide = aligned(b.q, 16) && b.q_token_stride % chunk == 0 && b.q_head_stride % chunk == 0;
    return a.quantized.bits == 4 ? launch_codes<4>(p, s, c.dtype, a.quantized, stream) : launch_codes<8>(p, s, c.dtype, a.quantized, stream);
}

}  // namespace paged
}  // namespace mgc
