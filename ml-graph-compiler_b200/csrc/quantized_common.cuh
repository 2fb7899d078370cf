// Pages of keys and values in 4 or 8 bits: the format, the place of a packed token, argument checks.
//
// The D channels of a token and key head are cut into groups of G. A group is D * bits / 8 / (D / G)
// bytes of codes (4 bits: the lower nibble is the earlier channel) and a pair of halves (scale,
// offset); channel c stands for scale * code + offset. Writing a group x takes
//   offset = half(min x),   scale = half((max x - offset) * (1 / L)),   L = 2^bits - 1,
//   code = (x - offset) / scale rounded to the nearest even whole number, within [0, L],
// each step rounded once to fp32, extremes held within +-65504 (half's range), scale 0 giving codes 0.
// Half has 11 significant bits: the codes are taken relative to the rounded pair, so a value is off by
// scale / 2 and, at the ends of the range, by what the pair's rounding cuts off, 2^-11 of the extremes.
// Halves rather than floats: 4 bytes a group of 64 channels in 4 bits are an eighth of its codes. A group
// with a value that is not finite gets the pair (NaN, NaN) and reads back as NaN.
#pragma once

#include "paged_common.cuh"

namespace mgc {
namespace paged {

// Two values of a 16-bit type at once.
template <typename T> __device__ __forceinline__ uint32_t two(float x, float y);
template <> __device__ __forceinline__ uint32_t two<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t two<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}
struct Quantized {
    const __half2 *k_scales, *v_scales;
    long long page_stride, token_stride, head_stride;  // pairs
    int bits, group, groups;
};

// Packed tokens one after the other: which sequence and position, and where its cache rows are. All
// lanes of a warp step together.
struct TokenWalk {
    int b, end, n;   // sequence, its end among the packed tokens, its cached positions
    int page, row;   // where the position is: page (-1: none), row in it
    int pos;         // position; negative: in no sequence, or no cached position
    int held;        // page of the sequence; -1: not looked up
    __device__ __forceinline__ void start(int t0) {
        b = -1;
        end = t0;
        n = 0;
        held = page = -1;
        row = 0;
    }
    __device__ __forceinline__ void step(const Batch &d, int t) {
        if (t >= end) {
            b = sequence_of(d, t);
            end = b < 0 ? t : __ldg(d.q_starts + b + 1);
            n = b < 0 ? 0 : __ldg(d.kv_lens + b);
            if (t >= end) {
                end = t + 1;
                n = 0;
            }
            held = -1;
        }
        pos = n - (end - t);
        if (pos < 0) {
            held = page = -1;
        } else if (held < 0) {
            held = pos / d.page_size;
            row = pos - held * d.page_size;
            page = page_of(d, b, held);
        } else if (++row == d.page_size) {
            row = 0;
            page = page_of(d, b, ++held);
        }
    }
    // Offset of the token's row in pages of these strides (page >= 0).
    __device__ __forceinline__ long long at(long long page_stride, long long token_stride) const {
        return (long long)page * page_stride + (long long)row * token_stride;
    }
};

// Warps of a launch over packed tokens: each takes a run of consecutive ones, and, when runs would be shorter than
// three tokens, a part of the tokens' heads, so that whole runs fill the GPU evenly.
struct TokenRuns {
    int run, parts;  // tokens of a run; parts of a token's heads
    unsigned blocks;
};
inline TokenRuns runs_of(int64_t tokens, int64_t most_parts, int warps, int resident) {
    const int64_t slots = (int64_t)sm_count() * resident * warps;
    int64_t parts = 1;
    while (parts < most_parts && ceil_div(tokens * parts, slots) < 3) parts = 2 * parts < most_parts ? 2 * parts : most_parts;
    TokenRuns r;
    r.parts = (int)parts;
    r.run = (int)ceil_div(tokens * parts, slots);
    r.blocks = (unsigned)ceil_div(ceil_div(tokens, r.run) * parts, warps);
    return r;
}

// Tells of rows of q_starts past the packed tokens (one thread of a launch).
__device__ __forceinline__ void check_rows(const Batch &d, int tokens) {
    if (d.status && __ldg(d.q_starts + d.batch) > tokens) *d.status = MGC_CUDA_GATHER_OOB;
}

inline int check_quantized(const mgc_cuda_quantized &z, const mgc_cuda_paged &c, const char *what) {
    if (z.bits != 4 && z.bits != 8) return fail(MGC_CUDA_UNSUPPORTED, "%s: pages of %lld bits", what, (long long)z.bits);
    if (!z.k_scales || !z.v_scales) return fail(MGC_CUDA_BAD_ARGUMENT, "%s: scales are NULL", what);
    if (c.head_dim % 16 || c.head_dim > 256)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: heads of %lld channels in %lld bits (a multiple of 16, at most 256)", what,
                    (long long)c.head_dim, (long long)z.bits);
    if (z.group < 1 || c.head_dim % z.group || (z.group != c.head_dim && z.group % 64))
        return fail(MGC_CUDA_UNSUPPORTED, "%s: groups of %lld of %lld channels (a multiple of 64, or all)", what, (long long)z.group,
                    (long long)c.head_dim);
    if (z.page_stride < 0 || z.token_stride < 0 || z.head_stride < 0)
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: a scale stride is negative", what);
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || c.page_stride % 16 || c.token_stride % 16 || c.head_stride % 16)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: rows of codes begin at multiples of 16 bytes", what);
    if (!aligned(z.k_scales, 4) || !aligned(z.v_scales, 4))
        return fail(MGC_CUDA_UNSUPPORTED, "%s: pairs of scales begin at multiples of 4 bytes", what);
    return MGC_CUDA_OK;
}

inline Quantized quantized_of(const mgc_cuda_quantized &z, const mgc_cuda_paged &c) {
    Quantized d;
    d.k_scales = static_cast<const __half2 *>(z.k_scales);
    d.v_scales = static_cast<const __half2 *>(z.v_scales);
    d.page_stride = z.page_stride;
    d.token_stride = z.token_stride;
    d.head_stride = z.head_stride;
    d.bits = (int)z.bits;
    d.group = (int)z.group;
    d.groups = (int)(c.head_dim / z.group);
    return d;
}

}  // namespace paged
}  // namespace mgc
