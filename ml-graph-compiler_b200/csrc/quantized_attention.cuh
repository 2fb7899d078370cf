// Attention of new tokens over quantised pages (quantized_common.cuh): paged_attention_params.cuh's
// definition with k_j and v_j the values that the codes stand for.
#pragma once

#include "quantized_mma.cuh"

namespace mgc {
namespace paged {

inline int check_attend_quantized(const mgc_cuda_paged_attention_quantized_args &a, const char *what) {
    MGC_CHECK(check_attend(a.attention, what));
    return check_quantized(a.quantized, a.attention.paged, what);
}

// How a call runs.
struct QuantPlan {
    int nb = 1;          // eights of query rows of a unit
    int row_tiles = 1;
    bool even = false, interleaved = false;
    int ctas = 0, live_rows = 1;
    int64_t workspace = 0;
};

inline int width_of(int64_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Calls `go` with the configuration of a type, width and row tile.
template <typename F> inline auto with_config(int64_t dtype, int64_t bits, int64_t head_dim, int nb, F go) {
    auto widths = [&](auto type, auto b) {
        using T = decltype(type);
        constexpr int BITS = decltype(b)::value;
        const int dp = width_of(head_dim);
        if (dp == 64) return nb > 1 ? go(QuantConfig<T, BITS, 64, 2>()) : go(QuantConfig<T, BITS, 64, 1>());
        if (dp == 128) return nb > 1 ? go(QuantConfig<T, BITS, 128, 2>()) : go(QuantConfig<T, BITS, 128, 1>());
        return go(QuantConfig<T, BITS, 256, 1>());
    };
    auto types = [&](auto b) {
        if (dtype == MGC_F32) return widths(float(), b);
        return dtype == MGC_F16 ? widths(__half(), b) : widths(__nv_bfloat16(), b);
    };
    return bits == 4 ? types(std::integral_constant<int, 4>()) : types(std::integral_constant<int, 8>());
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
    int64_t most = a.attention.max_kv;
    if (a.attention.window > 0 && a.attention.window + max_q < most) most = a.attention.window + max_q;
    // the kernel that adds pieces stores four elements at once
    const int es = elem_size(c.dtype);
    const bool wide = aligned(a.attention.out, 4 * es) && a.attention.o_token_stride % 4 == 0 && a.attention.o_head_stride % 4 == 0;
    const int resident = with_config(c.dtype, a.quantized.bits, c.head_dim, s.nb, [](auto config) { return decltype(config)::RESIDENT; });
    const int64_t slots = (int64_t)sm_count() * resident;
    // Even shares cost a second kernel and the pieces' way through memory, some 500 keys' worth of time
    if (wide && most > 512 + most * units / slots) {
        s.even = true;
        s.ctas = (int)slots;
        if (slots >= c.kv_heads && slots / c.kv_heads * c.kv_heads * 20 >= slots * 19) {
            s.interleaved = true;
            s.ctas = (int)(slots / c.kv_heads * c.kv_heads);
        }
        s.workspace = (int64_t)s.ctas * (2 * unit_rows * (c.head_dim * 4 + 8) + (int64_t)sizeof(CutUnit));
    }
    return s;
}

inline int64_t attend_quantized_workspace(const mgc_cuda_paged_attention_quantized_args &a) {
    if (check_attend_quantized(a, "mgc_cuda_paged_attention_quantized_workspace") != MGC_CUDA_OK) return -1;
    return a.attention.paged.tokens == 0 || a.attention.paged.batch == 0 ? 0 : quant_plan_of(a).workspace;
}

template <typename T, int BITS, int DP, int NB>
inline int launch_quantized(const QuantParams &p, const QuantPlan &s, QuantConfig<T, BITS, DP, NB>, cudaStream_t stream) {
    using C = QuantConfig<T, BITS, DP, NB>;
    if (s.even) {
        auto kernel = quantized_attention_kernel<T, BITS, DP, NB, true>;
        MGC_CHECK(raise_smem_ceiling((const void *)kernel));
        kernel<<<(unsigned)s.ctas, C::THREADS, C::SMEM, stream>>>(p);
        MGC_CHECK(check_launch("quantized_attention_kernel"));
        return launch_after(paged_combine_units_kernel<T, C::R>, dim3((unsigned)s.ctas, (unsigned)s.live_rows), p.a,
                            s.interleaved ? p.a.kv_heads : 1, stream);
    }
    auto kernel = quantized_attention_kernel<T, BITS, DP, NB, false>;
    MGC_CHECK(raise_smem_ceiling((const void *)kernel));
    kernel<<<(unsigned)(p.a.batch.batch * p.a.kv_heads * s.row_tiles), C::THREADS, C::SMEM, stream>>>(p);
    return check_launch("quantized_attention_kernel");
}

inline int attend_quantized(const mgc_cuda_paged_attention_quantized_args &a, cudaStream_t stream) {
    const char *what = "mgc_cuda_paged_attention_quantized";
    const mgc_cuda_paged_attention_args &b = a.attention;
    const mgc_cuda_paged &c = b.paged;
    MGC_CHECK(check_attend_quantized(a, what));
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
    QuantParams p;
    p.a = attend_params(b);
    p.z = quantized_of(a.quantized, c);
    const QuantPlan s = quant_plan_of(a);
    if (c.tokens * p.a.group >= 0x80000000ll - 256 || c.batch * c.kv_heads * s.row_tiles > 0x7FFFFFFF)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: %lld tokens of %d heads a key head", what, (long long)c.tokens, p.a.group);
    p.a.row_tiles = s.row_tiles;
    p.a.interleaved = s.interleaved;
    if (s.workspace) {
        if (!b.workspace || b.workspace_bytes < s.workspace || !aligned(b.workspace, 16))
            return fail(MGC_CUDA_NEEDS_WORKSPACE, "%s: needs %lld bytes of workspace (16-byte aligned), got %lld", what,
                        (long long)s.workspace, (long long)(b.workspace ? b.workspace_bytes : 0));
        const int64_t rows = (int64_t)s.ctas * 16 * s.nb;
        p.a.part = static_cast<float *>(b.workspace);
        p.a.part_ml = reinterpret_cast<float2 *>(p.a.part + rows * p.a.head_dim);
        p.a.cut = reinterpret_cast<CutUnit *>(p.a.part_ml + rows);
    }
    // pairs of a row copied at once where their addresses allow it
    const int64_t all = 4 * p.z.groups;
    p.pair_bytes = (all == 8 || all == 16) && aligned(p.z.k_scales, (int)all) && aligned(p.z.v_scales, (int)all) &&
                           p.z.page_stride * 4 % all == 0 && p.z.token_stride * 4 % all == 0 && p.z.head_stride * 4 % all == 0
                       ? (int)all : 4;
    const int chunk = 16 / elem_size(c.dtype);
    p.q_wide = aligned(b.q, 16) && b.q_token_stride % chunk == 0 && b.q_head_stride % chunk == 0;
    return with_config(c.dtype, a.quantized.bits, c.head_dim, s.nb, [&](auto config) { return launch_quantized(p, s, config, stream); });
}

}  // namespace paged
}  // namespace mgc
