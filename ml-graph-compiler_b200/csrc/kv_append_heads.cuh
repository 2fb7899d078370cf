// Append of new keys and values to a paged cache with what a decoder does to each head on the way: the
// root-mean-square norm of queries and keys, the position rotation, and the quantisation of pages in 4
// or 8 bits.
//
//   x' = (x r) w,  r = fp32((sum x^2 / D + eps)^-1/2);   x'' = R_p x' (kv_append.cuh);   page or q_out row = x''
// The sum of squares and the root are in fp64, everything else in fp32 with one rounding a step and no
// contraction: a code falls on one side of its border whatever the order of the sum, so that a call
// repeats its bits and any computation of these steps gives the same codes.
//
// Memory bounds it. A head takes 8, 16 or 32 lanes of eight channels each, in two fours: a lane of the rotated
// channels holds the fours whose channels pair up, so that one lane turns a pair, and what a head needs of all
// its channels (the sum, a group's extremes) meets by shuffles. Pages of codes want a lane's eight channels side by
// side: where pairs lie rot / 2 apart, keys change lanes through shared memory. Each warp takes a run of consecutive
// tokens, all heads of one after the other, the next heads' loads ahead.
//
// Codes: the quotient by the group's scale is taken as a product with its inverse, and only where that lies next to
// the border between two codes (one value in some thousand) as the definition's division.
#pragma once

#include <type_traits>

#include "quantized_common.cuh"

namespace mgc {
namespace paged {

struct HeadsParams {
    Batch batch;
    Quantized z;
    void *k_pages, *v_pages;
    long long page_stride, token_stride, head_stride;
    const void *q, *k, *v;
    void *q_out;
    long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs;
    const float *cos, *sin, *q_norm, *k_norm;
    double eps;
    long long table_row;
    int positions, rot, interleaved;
    int q_heads, kv_heads, head_dim;
    int seg;  // lanes of a head
    int tokens, run, parts;
    double inv_dim;
};

constexpr int HEADS_WARPS = 4, HEADS_RESIDENT = 8;

// (mean + eps)^-1/2 as fp32. In fp32's range one Newton step from the hardware's root leaves 2^-43, so that
// the rounding to fp32 is the exact root's but for one case in 2^18.
__device__ __forceinline__ float inverse_root(double m) {
    if (!(m > 1e-30 && m < 1e30)) return (float)(1.0 / sqrt(m));
    const double r = (double)rsqrtf((float)m);
    return (float)(r * (1.5 - 0.5 * m * r * r));
}

// Group code of eight values side by side, next to each other in a lane.
template <int BITS> __device__ __forceinline__ uint2 encode(const float (&x)[8], float offset, float scale) {
    constexpr float TOP = (float)((1 << BITS) - 1), ROUND = 12582912.0f;  // 1.5 * 2^23: adding it rounds to whole numbers
    if (!(scale > 0.0f)) return make_uint2(0, 0);
    const float inv = __frcp_rn(scale);
    float q[8], far = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        // off by two roundings: 2^-22 of at most 255, below 1e-4
        q[s] = fminf(fmaxf(__fmul_rn(__fsub_rn(x[s], offset), inv), 0.0f), TOP);
        far = fmaxf(far, fabsf(q[s] - (__fadd_rn(q[s], ROUND) - ROUND)));
    }
    if (far > 0.4999f) {
#pragma unroll
        for (int s = 0; s < 8; ++s) q[s] = fminf(fmaxf(__fdiv_rn(__fsub_rn(x[s], offset), scale), 0.0f), TOP);
    }
    uint32_t code[2] = {0, 0};
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        const uint32_t c = __float_as_uint(__fadd_rn(q[s], ROUND)) & 255u;
        code[BITS == 4 ? 0 : s >> 2] |= c << (BITS == 4 ? 4 * s : 8 * (s & 3));
    }
    return make_uint2(code[0], code[1]);
}

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
// Four values in a row.
template <typename T> __device__ __forceinline__ void store_four(T *dst, const float *x) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2 *>(dst) = make_uint2(two<T>(x[0], x[1]), two<T>(x[2], x[3]));
}

// SEG: lanes of a head where D and rot are multiples of 8 and rows allow accesses of four elements; 0: any other
// case, p.seg lanes.
template <typename S, typename T, int BITS, int SEG>
__global__ void __launch_bounds__(32 * HEADS_WARPS, HEADS_RESIDENT) kv_append_heads_kernel(const __grid_constant__ HeadsParams p) {
    __shared__ __align__(16) float exchange[BITS ? HEADS_WARPS : 1][BITS ? 256 : 4];
    constexpr bool VEC = SEG > 0;
    const int lane = (int)(threadIdx.x & 31), warp = (int)(threadIdx.x >> 5), seg = VEC ? SEG : p.seg;
    const unsigned unit = blockIdx.x * HEADS_WARPS + warp;
    if (unit == 0 && lane == 0) check_rows(p.batch, p.tokens);
    const long long t_first = (long long)(unit / (unsigned)p.parts) * p.run;
    if (t_first >= p.tokens) return;
    const int t0 = (int)t_first, t1 = min(t0 + p.run, p.tokens);
    const int sl = lane & (seg - 1), at_once = 32 / seg, sub = lane / seg;
    // a token's heads, at_once of one kind at a time: queries, keys, values
    const int q_items = (p.q_heads + at_once - 1) / at_once, kv_items = (p.kv_heads + at_once - 1) / at_once;
    const int items = q_items + 2 * kv_items, part = (int)(unit % (unsigned)p.parts);
    const bool mine = 8 * sl < p.head_dim, turned = 2 * 4 * sl < p.rot;  // (VEC) this lane's channels exist, are rotated
    const bool apart = turned && !p.interleaved;                        // (VEC) pairs rot / 2 apart

    // Channels of value s of the lane. VEC: two fours side by side; else pair 4 sl + s / 2, first or second.
    const int first_turned = apart ? 4 * sl : 8 * sl, second_turned = apart ? 4 * sl + p.rot / 2 : 8 * sl + 4;
    auto channel = [&](int s, bool is_v) {
        const int i = 4 * sl + (s >> 1);
        return !is_v && !p.interleaved && i < p.rot / 2 ? i + (s & 1) * (p.rot / 2) : 2 * i + (s & 1);
    };
    struct Eight {
        Pack<4, S> a, b;
    };
    // the token's rows of q, k and v, this lane's heads first
    const S *q_row = nullptr, *k_row = nullptr, *v_row = nullptr;
    auto token = [&](int t) {
        q_row = static_cast<const S *>(p.q) + (long long)t * p.q_ts;
        k_row = static_cast<const S *>(p.k) + (long long)t * p.k_ts;
        v_row = static_cast<const S *>(p.v) + (long long)t * p.v_ts;
    };
    auto load = [&](Eight &e, int i) {
        const bool is_q = i < q_items, is_v = i >= q_items + kv_items;
        const int h = (i - (is_q ? 0 : is_v ? q_items + kv_items : q_items)) * at_once + sub;
        const S *src = (is_q ? q_row : is_v ? v_row : k_row) + (long long)h * (is_q ? p.q_hs : is_v ? p.v_hs : p.k_hs);
        const bool have = h < (is_q ? p.q_heads : p.kv_heads);
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < Pack<4, S>::N; ++k) e.a.raw[k] = e.b.raw[k] = typename Pack<4, S>::R{};
            if (!have || !mine) return;
            e.a.load(src + (is_v ? 8 * sl : first_turned));
            e.b.load(src + (is_v ? 8 * sl + 4 : second_turned));
        } else {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const int c = channel(s, is_v);
                (s < 4 ? e.a.e[s & 3] : e.b.e[s & 3]) = have && c < p.head_dim ? src[c] : from_f<S>(0.0f);
            }
        }
    };
    auto store_row = [&](T *dst, const float (&x)[8], bool is_v) {
        if constexpr (VEC) {
            if (!mine) return;
            store_four<T>(dst + (is_v ? 8 * sl : first_turned), x);
            store_four<T>(dst + (is_v ? 8 * sl + 4 : second_turned), x + 4);
        } else {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const int c = channel(s, is_v);
                if (c < p.head_dim) dst[c] = from_f<T>(x[s]);
            }
        }
    };

    TokenWalk walk;
    walk.start(t0);
    float cs[4], sn[4];
    bool turn = false;    // the token's heads are normalised and rotated
    bool cached = false;  // and its key and value written
    long long at = 0, pairs = 0;
    auto place = [&](int t) {
        walk.step(p.batch, t);
        turn = walk.pos >= 0;
        cached = walk.page >= 0;
        if (p.rot && walk.pos >= p.positions) {
            if (p.batch.status) *p.batch.status = MGC_CUDA_GATHER_OOB;
            turn = cached = false;
        }
        at = cached ? walk.at(p.page_stride, p.token_stride) : 0;
        if (BITS) pairs = cached ? walk.at(p.z.page_stride, p.z.token_stride) : 0;
        if (!turn || !p.rot) return;
        const float *c = p.cos + (long long)walk.pos * p.table_row, *s = p.sin + (long long)walk.pos * p.table_row;
        if constexpr (VEC) {
            if (!turned) return;
            Pack<4, float> x, y;
            x.load(c + 4 * sl);
            y.load(s + 4 * sl);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                cs[k] = x.e[k];
                sn[k] = y.e[k];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = 4 * sl + k;
                cs[k] = i < p.rot / 2 ? c[i] : 1.0f;
                sn[k] = i < p.rot / 2 ? s[i] : 0.0f;
            }
        }
    };
    auto rotate = [&](float &x1, float &x2, int k) {
        const float a = __fsub_rn(__fmul_rn(x1, cs[k]), __fmul_rn(x2, sn[k])), b = __fadd_rn(__fmul_rn(x2, cs[k]), __fmul_rn(x1, sn[k]));
        x1 = a;
        x2 = b;
    };
    // kind 0: queries, 1: keys, 2: values
    auto finish = [&](const Eight &e, int t, int i, auto kind) {
        constexpr bool IS_Q = decltype(kind)::value == 0, IS_V = decltype(kind)::value == 2;
        const int h = i * at_once + sub;
        const bool there = h < (IS_Q ? p.q_heads : p.kv_heads);
        float x[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) x[s] = to_f(s < 4 ? e.a.e[s & 3] : e.b.e[s & 3]);
        if constexpr (!IS_V) {
            const float *weight = IS_Q ? p.q_norm : p.k_norm;
            if (turn && weight) {
                double sum = 0.0;
#pragma unroll
                for (int s = 0; s < 8; ++s) sum = fma((double)x[s], (double)x[s], sum);
#pragma unroll
                for (int d = 1; d < (VEC ? SEG : 32); d <<= 1)
                    if (VEC || d < seg) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
                const float r = inverse_root(fma(sum, p.inv_dim, p.eps));
                if constexpr (VEC) {
                    if (mine) {
                        Pack<4, float> a, b;
                        a.load(weight + first_turned);
                        b.load(weight + second_turned);
#pragma unroll
                        for (int s = 0; s < 8; ++s) x[s] = __fmul_rn(__fmul_rn(x[s], r), s < 4 ? a.e[s & 3] : b.e[s & 3]);
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const int c = channel(s, false);
                        if (c < p.head_dim) x[s] = __fmul_rn(__fmul_rn(x[s], r), __ldg(weight + c));
                    }
                }
            }
            if (turn && p.rot) {
                if constexpr (VEC) {
                    if (apart) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) rotate(x[k], x[4 + k], k);
                    } else if (turned) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) rotate(x[2 * k], x[2 * k + 1], k);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (4 * sl + k < p.rot / 2) rotate(x[2 * k], x[2 * k + 1], k);
                }
            }
        }
        if constexpr (IS_Q) {
            if (there) store_row(static_cast<T *>(p.q_out) + t * p.qo_ts + h * p.qo_hs, x, false);
        } else if constexpr (BITS == 0) {
            if (there && cached) store_row(static_cast<T *>(IS_V ? p.v_pages : p.k_pages) + at + h * p.head_stride, x, IS_V);
        } else {
            if (!cached) return;
            // channels 8 sl .. 8 sl + 7 side by side
            if (!VEC || (!IS_V && p.rot && !p.interleaved)) {
                float *row = exchange[warp] + (lane - sl) * 8;
                __syncwarp();
                if constexpr (VEC) {
                    *reinterpret_cast<float4 *>(row + first_turned) = make_float4(x[0], x[1], x[2], x[3]);
                    *reinterpret_cast<float4 *>(row + second_turned) = make_float4(x[4], x[5], x[6], x[7]);
                } else {
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const int c = channel(s, IS_V);
                        if (c < p.head_dim) row[c] = x[s];
                    }
                }
                __syncwarp();
#pragma unroll
                for (int s = 0; s < 8; s += 4) {
                    const float4 y = *reinterpret_cast<const float4 *>(row + 8 * sl + s);
                    x[s] = y.x;
                    x[s + 1] = y.y;
                    x[s + 2] = y.z;
                    x[s + 3] = y.w;
                }
            }
            float lo = INFINITY, hi = -INFINITY, bad = 0.0f;
            if (mine) {
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    lo = fminf(lo, x[s]);
                    hi = fmaxf(hi, x[s]);
                    bad = fmaf(x[s], 0.0f, bad);  // NaN if one is not finite
                }
            }
            const int span = p.z.groups == 1 ? seg : p.z.group / 8;  // lanes of a group
#pragma unroll
            for (int d = 1; d < (VEC ? SEG : 32); d <<= 1) {
                if (d >= span) break;
                lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
                hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
                bad = bad + __shfl_xor_sync(0xFFFFFFFFu, bad, d);
            }
            if (!mine || !there) return;
            constexpr float TOP = (float)((1 << BITS) - 1), MOST = 65504.0f;
            lo = fminf(fmaxf(lo, -MOST), MOST);
            hi = fminf(fmaxf(hi, -MOST), MOST);
            __half offset = __float2half_rn(lo);
            const float o = __half2float(offset);
            __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, o), 1.0f / TOP));
            uint2 code = encode<BITS>(x, o, __half2float(scale));
            if (bad != 0.0f) {
                scale = offset = __float2half_rn(__int_as_float(0x7FC00000));
                code = make_uint2(0, 0);
            }
            uint8_t *row = static_cast<uint8_t *>(IS_V ? p.v_pages : p.k_pages) + at + h * p.head_stride + sl * BITS;
            if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(row) = code.x;
            else *reinterpret_cast<uint2 *>(row) = code;
            const int group = p.z.groups == 1 ? 0 : 8 * sl / p.z.group;
            if (8 * sl == group * p.z.group)
                const_cast<__half2 *>(IS_V ? p.z.v_scales : p.z.k_scales)[pairs + h * p.z.head_stride + group] = __halves2half2(scale, offset);
        }
    };

    for (int t = t0; t < t1; ++t) {
        Eight now, next;
        token(t);
        load(now, part);
        place(t);
        for (int i = part; i < items; i += p.parts) {
            if (i + p.parts < items) load(next, i + p.parts);
            if (i < q_items) finish(now, t, i, std::integral_constant<int, 0>());
            else if (i < q_items + kv_items) finish(now, t, i - q_items, std::integral_constant<int, 1>());
            else finish(now, t, i - q_items - kv_items, std::integral_constant<int, 2>());
            now = next;
        }
    }
}

template <typename S, typename T, int BITS> inline int launch_heads(HeadsParams &p, bool vec, cudaStream_t stream) {
    p.seg = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 16 : 32;
    const TokenRuns r = runs_of(p.tokens, ceil_div(p.q_heads, 32 / p.seg) + 2 * ceil_div(p.kv_heads, 32 / p.seg), HEADS_WARPS, HEADS_RESIDENT);
    p.run = r.run;
    p.parts = r.parts;
    p.inv_dim = 1.0 / p.head_dim;
    auto go = [&](auto seg) {
        kv_append_heads_kernel<S, T, BITS, decltype(seg)::value><<<r.blocks, 32 * HEADS_WARPS, 0, stream>>>(p);
    };
    if (!vec) go(std::integral_constant<int, 0>());
    else if (p.seg == 8) go(std::integral_constant<int, 8>());
    else if (p.seg == 16) go(std::integral_constant<int, 16>());
    else go(std::integral_constant<int, 32>());
    return check_launch("kv_append_heads_kernel");
}

inline int append_heads(const mgc_cuda_kv_append_heads_args &a, cudaStream_t stream) {
    const char *what = "mgc_cuda_kv_append_heads";
    const mgc_cuda_kv_append_args &b = a.append;
    const mgc_cuda_paged &c = b.paged;
    const bool codes = a.quantized.bits != 0;
    MGC_CHECK(check_paged(c, what));
    if (codes) MGC_CHECK(check_quantized(a.quantized, c, what));
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
    if (!b.k || !b.v || (b.q && !b.q_out) || b.q_heads < 0 || b.rot < 0 || b.rot > c.head_dim || b.rot % 2 ||
        (b.rot && (!b.cos || !b.sin || b.positions < 0 || b.table_row < 0)))
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: missing operand or bad rotation width %lld", what, (long long)b.rot);
    if (!(a.eps >= 0.0) || a.eps > 1e30) return fail(MGC_CUDA_BAD_ARGUMENT, "%s: eps %g", what, a.eps);
    if (b.src_dtype != c.dtype && (codes || b.src_dtype != MGC_F32))
        return fail(MGC_CUDA_UNSUPPORTED, "%s: sources of type %d for %s of type %d", what, (int)b.src_dtype, codes ? "queries" : "pages",
                    (int)c.dtype);
    if (b.q && b.q == b.q_out && (b.src_dtype != c.dtype || b.q_token_stride != b.qo_token_stride || b.q_head_stride != b.qo_head_stride))
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: q in place keeps its type and strides", what);
    const int64_t heads = (b.q ? b.q_heads : 0) + 2 * c.kv_heads;
    if (c.head_dim > 256 || heads > 1 << 20)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: %lld heads of %lld channels", what, (long long)heads, (long long)c.head_dim);
    HeadsParams p;
    memset(&p, 0, sizeof p);
    p.batch = batch_of(c);
    if (codes) p.z = quantized_of(a.quantized, c);
    p.k_pages = c.k; p.v_pages = c.v;
    p.page_stride = c.page_stride; p.token_stride = c.token_stride; p.head_stride = c.head_stride;
    p.q = b.q; p.k = b.k; p.v = b.v; p.q_out = b.q_out;
    p.q_ts = b.q_token_stride; p.q_hs = b.q_head_stride;
    p.k_ts = b.k_token_stride; p.k_hs = b.k_head_stride;
    p.v_ts = b.v_token_stride; p.v_hs = b.v_head_stride;
    p.qo_ts = b.qo_token_stride; p.qo_hs = b.qo_head_stride;
    p.cos = b.cos; p.sin = b.sin; p.table_row = b.table_row;
    p.q_norm = a.q_norm; p.k_norm = a.k_norm; p.eps = a.eps;
    p.positions = (int)(b.positions > 0x7FFFFFFF ? 0x7FFFFFFF : b.positions);
    p.rot = (int)b.rot; p.interleaved = b.interleaved != 0;
    p.q_heads = b.q ? (int)b.q_heads : 0; p.kv_heads = (int)c.kv_heads; p.head_dim = (int)c.head_dim;
    p.tokens = (int)c.tokens;
    const int64_t ss = elem_size(b.src_dtype) * 4, ts = elem_size(c.dtype) * 4;  // bytes of four elements
    auto rows = [](const void *x, int64_t y, int64_t z, int64_t bytes) {
        return aligned(x, (int)bytes) && y % 4 == 0 && z % 4 == 0;
    };
    const bool vec = p.head_dim % 8 == 0 && p.rot % 8 == 0 && rows(b.k, b.k_token_stride, b.k_head_stride, ss) &&
                     rows(b.v, b.v_token_stride, b.v_head_stride, ss) &&
                     (!b.q || (rows(b.q, b.q_token_stride, b.q_head_stride, ss) && rows(b.q_out, b.qo_token_stride, b.qo_head_stride, ts))) &&
                     (codes || (rows(c.k, c.page_stride, c.token_stride, ts) && rows(c.v, c.head_stride, 0, ts))) &&
                     (!p.rot || (aligned(b.cos, 16) && aligned(b.sin, 16) && b.table_row % 4 == 0)) &&
                     (!a.q_norm || aligned(a.q_norm, 16)) && (!a.k_norm || aligned(a.k_norm, 16));
    auto types = [&](auto src, auto page) {
        using S = decltype(src);
        using T = decltype(page);
        if constexpr (sizeof(S) == sizeof(T)) {
            if (a.quantized.bits == 4) return launch_heads<S, T, 4>(p, vec, stream);
            if (a.quantized.bits == 8) return launch_heads<S, T, 8>(p, vec, stream);
        }
        return launch_heads<S, T, 0>(p, vec, stream);
    };
    const bool wide = b.src_dtype == MGC_F32;
    if (c.dtype == MGC_F32) return types(float(), float());
    if (c.dtype == MGC_F16) return wide ? types(float(), __half()) : types(__half(), __half());
    return wide ? types(float(), __nv_bfloat16()) : types(__nv_bfloat16(), __nv_bfloat16());
}

}  // namespace paged
}  // namespace mgc
