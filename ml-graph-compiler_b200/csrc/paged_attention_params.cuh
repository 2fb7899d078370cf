// Parameters of the paged attention kernels.
//
//   o_t[h] = sum_j w_j v_j,   w = softmax over the visible positions j of scale * q_t[h] . k_j
// computed in one pass over the keys with the running maximum m and sum l of the softmax:
//   m' = max(m, s_j),  l' = l e^(m - m') + e^(s_j - m'),  o' = o e^(m - m') + e^(s_j - m') v_j,
// exponentials in base 2 (scale carries log2 e), statistics and sums in fp32.
#pragma once

#include "paged_common.cuh"

namespace mgc {
namespace paged {

// A unit of rows whose first piece ended CTA c's stretch of work (one per CTA at most): its pieces
// are c's second slot of partial results and the first slots of the next pieces - 1 CTAs.
struct CutUnit {
    int h, b, t, pieces;
};

constexpr int MAX_HEAD_DIM = 256;

// Half has five exponent bits: a weight below 2^-14 of the largest would lose bits and one below 2^-25
// vanish from the products (not from the sum), and a long context can hold much of its mass there. So
// f16 weights are made 2^LIFT times as large; output and sum carry the factor and it cancels. The tcgen05
// kernel lets weights grow to 2^LAZY before it moves their reference: 2^15 at most in either kernel.
// What is left of the range: steps of 2^-38 of the largest weight, 2^-35 at least in the tcgen05 kernel.
template <typename T> struct Weight { static constexpr float LIFT = 0.0f, LAZY = 8.0f, LAZY_LIFT = 0.0f; };
template <> struct Weight<__half> { static constexpr float LIFT = 14.0f, LAZY = 4.0f, LAZY_LIFT = 11.0f; };

struct AttendParams {
    Batch batch;
    const void *k_pages, *v_pages;
    long long page_stride, token_stride, head_stride;
    const void *q;
    void *out;
    long long q_ts, q_hs, o_ts, o_hs;
    int tokens, q_heads, kv_heads, group, head_dim;
    int causal, window;
    float scale_log2;  // scale * log2 e
    int max_positions;  // positions a row of the block table can hold
    // clusters: row tiles per (sequence, key head) in the grid, CTAs that share a tile's keys
    int row_tiles, splits;
    // even shares: a stretch of every key head's units side by side (CTA c: key head c % kv_heads), or
    // the stretches key head by key head; partial results of the pieces
    int interleaved;
    float *part;        // [CTA][2][rows of a unit][head_dim], relative to the row's maximum
    float2 *part_ml;    // [CTA][2][rows of a unit]: maximum (scaled, base 2), sum
    CutUnit *cut;       // [CTA]
};

// Visible positions [lo, hi) of a token at position pos, of the n positions that can be read.
__device__ __forceinline__ void visible(const AttendParams &p, int n, int pos, int &lo, int &hi) {
    hi = p.causal ? min(n, pos + 1) : n;
    lo = p.window > 0 ? max(0, min(n, pos - p.window + 1)) : 0;
}

// ---- host side ---------------------------------------------------------------------------------
inline int check_attend(const mgc_cuda_paged_attention_args &a, const char *what) {
    const mgc_cuda_paged &c = a.paged;
    MGC_CHECK(check_paged(c, what));
    if (c.tokens > 0 && c.batch > 0 && (!a.q || !a.out)) return fail(MGC_CUDA_BAD_ARGUMENT, "%s: q or out is NULL", what);
    if (a.q_heads < 1 || a.q_heads % c.kv_heads)
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: %lld query heads over %lld key heads", what, (long long)a.q_heads,
                    (long long)c.kv_heads);
    if (c.head_dim > MAX_HEAD_DIM || a.q_heads > 65535)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: %lld heads of %lld channels (at most %d channels)", what,
                    (long long)a.q_heads, (long long)c.head_dim, MAX_HEAD_DIM);
    if (a.window < 0 || (a.window > 0 && !a.causal))
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: a window of %lld needs causal attention", what, (long long)a.window);
    if (!(a.scale > 0.0) || a.scale > 1e30) return fail(MGC_CUDA_BAD_ARGUMENT, "%s: scale %g", what, a.scale);
    if (a.max_q < 0 || a.max_kv < 0) return fail(MGC_CUDA_BAD_ARGUMENT, "%s: negative bound", what);
    return MGC_CUDA_OK;
}

// The call behind mgc_cuda_paged_attention (paged.cu). q_dtype: of q and out, where it is not the pages'
// (bf16 over half pages, in calls that take the tcgen05 kernel).
int attend(const mgc_cuda_paged_attention_args &a, int64_t q_dtype, cudaStream_t stream);

// The parameters that a call's arguments give; its plan adds the rest.
inline AttendParams attend_params(const mgc_cuda_paged_attention_args &a) {
    const mgc_cuda_paged &c = a.paged;
    AttendParams p;
    p.batch = batch_of(c);
    p.k_pages = c.k; p.v_pages = c.v;
    p.page_stride = c.page_stride; p.token_stride = c.token_stride; p.head_stride = c.head_stride;
    p.q = a.q; p.out = a.out;
    p.q_ts = a.q_token_stride; p.q_hs = a.q_head_stride; p.o_ts = a.o_token_stride; p.o_hs = a.o_head_stride;
    p.tokens = (int)c.tokens; p.q_heads = (int)a.q_heads; p.kv_heads = (int)c.kv_heads;
    p.group = p.q_heads / p.kv_heads; p.head_dim = (int)c.head_dim;
    p.causal = a.causal != 0;
    p.window = (int)(a.window > 0x3FFFFFFF ? 0x3FFFFFFF : a.window);
    p.scale_log2 = (float)(a.scale * 1.4426950408889634074);
    p.max_positions = (int)(c.table_pages * c.page_size);
    p.row_tiles = p.splits = 1;
    p.interleaved = 0;
    p.part = nullptr; p.part_ml = nullptr; p.cut = nullptr;
    return p;
}

}  // namespace paged
}  // namespace mgc
