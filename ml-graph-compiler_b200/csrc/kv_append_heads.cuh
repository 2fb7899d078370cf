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
//
// 19466 tokens of 48 heads x 128 in bf16, normalised and rotated: 121 us into plain pages (478 MB, 4.0 TB/s, 61 % of the
// copy bandwidth), 153 us into 4-bit ones (2.5 TB/s). Issue bounds it: some 160 instructions for two heads' 256
// values, 90 of them the norm's (sums in fp64), 300 where codes are made; the SMs issue in 62 % of their cycles.
// Tried: 64 and 96 registers (HEADS_RESIDENT), one loop over all kinds of heads (twice the instructions).
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

constexpr int HEADS_WARPS = 4;
// Blocks of an SM: 64 registers do for 16-bit sources into plain pages (19466 tokens, 48 heads of 128: 121 us, with 80
// 128 us), the others want 80 (4 bits 154 us, with 64 164 us; fp32 sources of 80 channels 22.8 and 24.8 us).
template <typename S, int BITS> constexpr int HEADS_RESIDENT = BITS == 0 && sizeof(S) == 2 ? 8 : 6;

// (mean + eps)^-1/2 as fp32. In fp32's range one Newton step from the hardware's root leaves 2^-43, so that
// the rounding to fp32 is the exact root's but for one case in 2^18.
__device__ __forceinline__ float inverse_root(double m) {
    if (!(m > 1e-30 && m < 1e30)) return (float)(1.0 / sqrt(m));
    float a;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"((float)m));
    const double r = (double)a;
    return (float)(r * fma(-0.5 * m * r, r, 1.5));
}

// Least and greatest, NaN if one is.
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Codes of eight values side by side.
template <int BITS> __device__ __forceinline__ uint2 encode(const float (&x)[8], float offset, float scale) {
    constexpr float TOP = (float)((1 << BITS) - 1), ROUND = 12582912.0f;  // 1.5 * 2^23: adding it rounds to whole numbers
    if (!(scale > 0.0f)) return make_uint2(0, 0);
    const float inv = __frcp_rn(scale);
    float q[8], far = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        // off by two roundings: 2^-22 of at most 255, below 1e-4
        const float y = fminf(fmaxf(__fmul_rn(__fsub_rn(x[s], offset), inv), 0.0f), TOP);
        q[s] = __fadd_rn(y, ROUND);
        far = fmaxf(far, fabsf(y - (q[s] - ROUND)));
    }
    if (far > 0.4999f) {
#pragma unroll
        for (int s = 0; s < 8; ++s) q[s] = __fadd_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(x[s], offset), scale), 0.0f), TOP), ROUND);
    }
    // ROUND's own bits, shifted alike, come off the sum at once
    constexpr uint32_t BASE = 0x4B400000u, ALL = BITS == 4 ? BASE * 0x11111111u : BASE * 0x01010101u;
    uint32_t code[2] = {0u - ALL, 0u - ALL};
#pragma unroll
    for (int s = 0; s < 8; ++s) code[BITS == 4 ? 0 : s >> 2] += __float_as_uint(q[s]) << (BITS == 4 ? 4 * s : 8 * (s & 3));
    return make_uint2(code[0], code[1]);
}

// Four values in a row.
template <typename T> __device__ __forceinline__ void store_four(T *dst, const float *x) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2 *>(dst) = make_uint2(two<T>(x[0], x[1]), two<T>(x[2], x[3]));
}

// SEG: lanes of a head where D and rot are multiples of 8 and rows allow accesses of four elements; 0: any other
// case, p.seg lanes.
template <typename S, typename T, int BITS, int SEG>
__global__ void __launch_bounds__(32 * HEADS_WARPS, HEADS_RESIDENT<S, BITS>) kv_append_heads_kernel(const __grid_constant__ HeadsParams p) {
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
    const int part = (int)(unit % (unsigned)p.parts);
    const bool mine = 8 * sl < p.head_dim, turned = 2 * 4 * sl < p.rot;  // (VEC) this lane's channels exist, are rotated
    const bool apart = turned && !p.interleaved;                        // (VEC) pairs rot / 2 apart

    // codes: the lane's group, the lanes of a group, whether it is the group's first
    const int group = BITS ? 8 * sl / p.z.group : 0, span = !BITS ? 1 : p.z.groups == 1 ? seg : p.z.group / 8;
    const bool leads = BITS && 8 * sl == group * p.z.group;

    // Channels of value s of the lane. VEC: two fours side by side; else pair 4 sl + s / 2, first or second.
    const int first_turned = apart ? 4 * sl : 8 * sl, second_turned = apart ? 4 * sl + p.rot / 2 : 8 * sl + 4;
    auto channel = [&](int s, bool is_v) {
        const int i = 4 * sl + (s >> 1);
        return !is_v && !p.interleaved && i < p.rot / 2 ? i + (s & 1) * (p.rot / 2) : 2 * i + (s & 1);
    };
    struct Eight {
        Pack<4, S> a, b;
    };
    auto load = [&](Eight &e, const S *src, bool have, bool is_v) {
        if constexpr (VEC) {
            if (!have) return;
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
    // pair: of the lane's group of the head
    auto finish = [&](const Eight &e, auto kind, auto *dst, __half2 *pair, bool there) {
        constexpr bool IS_Q = decltype(kind)::value == 0, IS_V = decltype(kind)::value == 2;
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
            if (there) store_row(dst, x, false);
        } else if constexpr (BITS == 0) {
            if (there && cached) store_row(dst, x, IS_V);
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
            float lo = INFINITY, hi = -INFINITY;
            if (mine) {
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    lo = min_nan(lo, x[s]);
                    hi = max_nan(hi, x[s]);
                }
            }
#pragma unroll
            for (int d = 1; d < (VEC ? SEG : 32); d <<= 1) {
                if (d >= span) break;
                lo = min_nan(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
                hi = max_nan(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
            }
            const bool bad = !(lo > -INFINITY && hi < INFINITY);  // a value is not finite
            if (!mine || !there) return;
            constexpr float TOP = (float)((1 << BITS) - 1), MOST = 65504.0f;
            lo = fminf(fmaxf(lo, -MOST), MOST);
            hi = fminf(fmaxf(hi, -MOST), MOST);
            __half offset = __float2half_rn(lo);
            const float o = __half2float(offset);
            __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, o), 1.0f / TOP));
            uint2 code = encode<BITS>(x, o, __half2float(scale));
            if (bad) {
                scale = offset = __float2half_rn(__int_as_float(0x7FC00000));
                code = make_uint2(0, 0);
            }
            if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(dst + sl * 4) = code.x;
            else *reinterpret_cast<uint2 *>(dst + sl * 8) = code;
            if (leads) *pair = __halves2half2(scale, offset);
        }
    };

    // One kind's heads of a token (0: queries, 1: keys, 2: values): items i, i + parts, ...
    auto heads_of = [&](auto kind, const S *src, long long src_hs, auto *dst, long long dst_hs, __half2 *pair, int count, int i) {
        constexpr bool IS_V = decltype(kind)::value == 2;
        const int step = p.parts * at_once;
        int h = i * at_once + sub;
        src += h * src_hs;
        dst += h * dst_hs;
        pair += h * p.z.head_stride + group;
        const long long src_step = step * src_hs, dst_step = step * dst_hs, pair_step = BITS ? step * p.z.head_stride : 0;
        Eight now, next;
#pragma unroll
        for (int k = 0; k < Pack<4, S>::N; ++k) now.a.raw[k] = now.b.raw[k] = next.a.raw[k] = next.b.raw[k] = typename Pack<4, S>::R{};
        load(now, src, h < count && (mine || !VEC), IS_V);
        for (; h - sub < count; h += step, now = next) {
            src += src_step;
            if (h - sub + step < count) load(next, src, h + step < count && (mine || !VEC), IS_V);
            finish(now, kind, dst, pair, h < count);
            dst += dst_step;
            pair += pair_step;
        }
    };
    // the first item of a kind with so many before it that is this part's
    auto first_item = [&](int before) {
        const int x = (part - before) % p.parts;
        return x < 0 ? x + p.parts : x;
    };
    const int k_first = first_item(q_items), v_first = first_item(q_items + kv_items);
    for (int t = t0; t < t1; ++t) {
        place(t);
        using Page = std::conditional_t<BITS != 0, uint8_t, T>;
        heads_of(std::integral_constant<int, 0>(), static_cast<const S *>(p.q) + (long long)t * p.q_ts, p.q_hs,
                 static_cast<T *>(p.q_out) + (long long)t * p.qo_ts, p.qo_hs, nullptr, p.q_heads, part);
        heads_of(std::integral_constant<int, 1>(), static_cast<const S *>(p.k) + (long long)t * p.k_ts, p.k_hs,
                 static_cast<Page *>(p.k_pages) + at, p.head_stride, const_cast<__half2 *>(p.z.k_scales) + pairs, p.kv_heads, k_first);
        heads_of(std::integral_constant<int, 2>(), static_cast<const S *>(p.v) + (long long)t * p.v_ts, p.v_hs,
                 static_cast<Page *>(p.v_pages) + at, p.head_stride, const_cast<__half2 *>(p.z.v_scales) + pairs, p.kv_heads, v_first);
    }
}

template <typename S, typename T, int BITS> inline int launch_heads(HeadsParams &p, bool vec, cudaStream_t stream) {
    p.seg = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 16 : 32;
    const TokenRuns r = runs_of(p.tokens, ceil_div(p.q_heads, 32 / p.seg) + 2 * ceil_div(p.kv_heads, 32 / p.seg), HEADS_WARPS, HEADS_RESIDENT<S, BITS>);
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
