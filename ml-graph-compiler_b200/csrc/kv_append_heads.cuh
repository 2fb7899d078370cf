// Append of new keys and values to a paged cache with what a decoder does to each head on the way: the
// root-mean-square norm of queries and keys, the position rotation, and the quantisation of pages in 4
// or 8 bits.
//
//   x' = (x r) w,  r = fp32((sum x^2 / D + eps)^-1/2);   x'' = R_p x' (kv_append.cuh);   page or q_out row = x''
// The sum of squares and the root are in fp64, everything else in fp32 with one rounding a step and no
// contraction: a code falls on one side of its border whatever the order of the sum, so that a call
// repeats its bits and any computation of these steps gives the same codes.
//
// Memory bounds it. A head takes SEG lanes (8, 16 or 32) of eight channels each, held as four pairs: pair i
// of the rotated channels is turned by one lane, and what a head needs of all its channels (the sum, a
// group's extremes) meets by shuffles. Pages of codes want a lane's eight channels side by side: where pairs
// lie rot / 2 apart the values change lanes through shared memory.
#pragma once

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
    int tokens, per_block;
};

constexpr int HEADS_WARPS = 4;

// (mean + eps)^-1/2 as fp32. In fp32's range one Newton step from the hardware's root leaves 2^-43, so that
// the rounding to fp32 is the exact root's but for one case in 2^18.
__device__ __forceinline__ float inverse_root(double m) {
    if (!(m > 1e-30 && m < 1e30)) return (float)(1.0 / sqrt(m));
    const double r = (double)rsqrtf((float)m);
    return (float)(r * (1.5 - 0.5 * m * r * r));
}

// Channel of slot s (0..7) of lane `sl` of a head: slots k and 4 + k are pair 4 sl + k.
__device__ __forceinline__ int channel_of(const HeadsParams &p, int sl, int s, bool halves) {
    const int i = 4 * sl + (s & 3);
    return halves && i < p.rot / 2 ? (s < 4 ? i : i + p.rot / 2) : 2 * i + (s >> 2);
}

// The eight values of a lane, as they come.
template <typename S> struct Eight {
    Pack<4, S> a, b;
};

// VEC: D and rot are multiples of 8 and rows allow accesses of four elements.
template <typename S, typename T, int BITS, bool VEC>
__global__ void __launch_bounds__(32 * HEADS_WARPS) kv_append_heads_kernel(const __grid_constant__ HeadsParams p) {
    __shared__ float exchange[BITS ? HEADS_WARPS : 1][BITS ? 256 : 1];
    const int lane = (int)(threadIdx.x & 31), warp = (int)(threadIdx.x >> 5);
    const int sl = lane & (p.seg - 1), at_once = 32 / p.seg;
    const int heads = p.q_heads + 2 * p.kv_heads, step = (int)gridDim.y * HEADS_WARPS * at_once;
    const int h_first = ((int)blockIdx.y * HEADS_WARPS + warp) * at_once + lane / p.seg;
    const int t0 = (int)blockIdx.x * p.per_block, t1 = min(t0 + p.per_block, p.tokens);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) check_rows(p.batch, p.tokens);

    auto source = [&](int t, int h) -> const S * {
        if (h < p.q_heads) return static_cast<const S *>(p.q) + t * p.q_ts + h * p.q_hs;
        h -= p.q_heads;
        if (h < p.kv_heads) return static_cast<const S *>(p.k) + t * p.k_ts + h * p.k_hs;
        return static_cast<const S *>(p.v) + t * p.v_ts + (h - p.kv_heads) * p.v_hs;
    };
    // values are apart (pairs rot / 2 apart) for queries and keys, side by side for values
    auto load = [&](Eight<S> &e, int t, int h) {
        if (h >= heads) return;
        const S *src = source(t, h);
        const bool halves = !p.interleaved && h < p.q_heads + p.kv_heads;
        if constexpr (VEC) {
            if (8 * sl >= p.head_dim) return;
            const bool apart = halves && 8 * sl < p.rot;
            e.a.load(src + (apart ? 4 * sl : 8 * sl));
            e.b.load(src + (apart ? 4 * sl + p.rot / 2 : 8 * sl + 4));
        } else {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const int c = channel_of(p, sl, s, halves);
                if (c >= p.head_dim) continue;
                if (s < 4) e.a.e[s] = src[c];
                else e.b.e[s - 4] = src[c];
            }
        }
    };
    // the channels of the two packs, in VEC form
    auto store_row = [&](T *dst, const float (&x)[8], bool halves) {
        if constexpr (VEC) {
            if (8 * sl >= p.head_dim) return;
            const bool apart = halves && 8 * sl < p.rot;
            Pack<4, T> a, b;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                a.e[k] = from_f<T>(apart ? x[k] : x[(k >> 1) + 4 * (k & 1)]);
                b.e[k] = from_f<T>(apart ? x[4 + k] : x[2 + (k >> 1) + 4 * (k & 1)]);
            }
            a.store(dst + (apart ? 4 * sl : 8 * sl));
            b.store(dst + (apart ? 4 * sl + p.rot / 2 : 8 * sl + 4));
        } else {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const int c = channel_of(p, sl, s, halves);
                if (c < p.head_dim) dst[c] = from_f<T>(x[s]);
            }
        }
    };

    TokenWalk walk;
    walk.start(t0);
    float cs[4], sn[4];
    bool turn = false;     // the token's heads are normalised and rotated
    bool cached = false;   // and its key and value written
    auto place = [&](int t) {
        walk.step(p.batch, t);
        turn = walk.pos >= 0;
        cached = walk.page >= 0;
        if (p.rot && walk.pos >= p.positions) {
            if (p.batch.status) *p.batch.status = MGC_CUDA_GATHER_OOB;
            turn = cached = false;
        }
        if (!turn || !p.rot) return;
        const float *c = p.cos + (long long)walk.pos * p.table_row, *s = p.sin + (long long)walk.pos * p.table_row;
        if (VEC && 8 * sl < p.rot) {
            Pack<4, float> x, y;
            x.load(c + 4 * sl);
            y.load(s + 4 * sl);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                cs[k] = x.e[k];
                sn[k] = y.e[k];
            }
        } else if (!VEC) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = 4 * sl + k;
                cs[k] = i < p.rot / 2 ? c[i] : 1.0f;
                sn[k] = i < p.rot / 2 ? s[i] : 0.0f;
            }
        }
    };
    auto finish = [&](const Eight<S> &e, int t, int h) {
        const bool is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads, is_v = !is_q && !is_k && h < heads;
        const bool halves = !p.interleaved && !is_v;
        float x[8];
        if constexpr (VEC) {
            const bool mine = h < heads && 8 * sl < p.head_dim, apart = halves && 8 * sl < p.rot;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float a = mine ? to_f(e.a.e[k]) : 0.0f, b = mine ? to_f(e.b.e[k]) : 0.0f;
                if (apart) {
                    x[k] = a;
                    x[4 + k] = b;
                } else {
                    x[(k >> 1) + 4 * (k & 1)] = a;
                    x[2 + (k >> 1) + 4 * (k & 1)] = b;
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const bool mine = h < heads && channel_of(p, sl, s, halves) < p.head_dim;
                x[s] = mine ? to_f(s < 4 ? e.a.e[s] : e.b.e[s - 4]) : 0.0f;
            }
        }
        const float *weight = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
        if (turn && (p.q_norm || p.k_norm)) {  // (the same branch for the whole warp)
            double sum = 0.0;
#pragma unroll
            for (int s = 0; s < 8; ++s) sum += (double)x[s] * (double)x[s];
            for (int d = 1; d < p.seg; d <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
            if (weight) {
                const float r = inverse_root(sum / p.head_dim + p.eps);
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const int c = channel_of(p, sl, s, halves);
                    if (c < p.head_dim) x[s] = __fmul_rn(__fmul_rn(x[s], r), __ldg(weight + c));
                }
            }
        }
        if (turn && !is_v && (VEC ? 8 * sl < p.rot : p.rot > 0)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (!VEC && 4 * sl + k >= p.rot / 2) continue;
                const float x1 = x[k], x2 = x[4 + k];
                x[k] = __fsub_rn(__fmul_rn(x1, cs[k]), __fmul_rn(x2, sn[k]));
                x[4 + k] = __fadd_rn(__fmul_rn(x2, cs[k]), __fmul_rn(x1, sn[k]));
            }
        }
        if (is_q) store_row(static_cast<T *>(p.q_out) + t * p.qo_ts + h * p.qo_hs, x, halves);
        if constexpr (BITS == 0) {
            if ((is_k || is_v) && cached) {
                const int kh = h - p.q_heads - (is_v ? p.kv_heads : 0);
                T *row = static_cast<T *>(is_k ? p.k_pages : p.v_pages) + walk.row(p.batch, p.page_stride, p.token_stride) +
                         kh * p.head_stride;
                store_row(row, x, halves);
            }
        } else {
            const bool some = h + at_once > p.q_heads && h < heads;
            if (!cached || !__any_sync(0xFFFFFFFFu, some && (is_k || is_v))) return;
            // channels 8 sl .. 8 sl + 7 side by side
            if (!VEC || (p.rot && !p.interleaved)) {
                float *row = exchange[warp] + (lane - sl) * 8;
                __syncwarp();
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const int c = channel_of(p, sl, s, halves);
                    if (c < p.head_dim) row[c] = x[s];
                }
                __syncwarp();
#pragma unroll
                for (int s = 0; s < 8; ++s) x[s] = row[8 * sl + s];
            } else {
                float y[8];
#pragma unroll
                for (int s = 0; s < 8; ++s) y[s] = x[(s >> 1) + 4 * (s & 1)];
#pragma unroll
                for (int s = 0; s < 8; ++s) x[s] = y[s];
            }
            const bool mine = 8 * sl < p.head_dim;
            float lo = INFINITY, hi = -INFINITY, bad = 0.0f;
            if (mine) {
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    lo = fminf(lo, x[s]);
                    hi = fmaxf(hi, x[s]);
                    bad = bad + x[s] * 0.0f;  // NaN if one is not finite
                }
            }
            const int span = p.z.group == p.head_dim ? p.seg : p.z.group / 8;  // lanes of a group
            for (int d = 1; d < span; d <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
                hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
                bad = bad + __shfl_xor_sync(0xFFFFFFFFu, bad, d);
            }
            if (!mine || !(is_k || is_v)) return;
            constexpr float TOP = (float)((1 << BITS) - 1), MOST = 65504.0f;
            lo = fminf(fmaxf(lo, -MOST), MOST);
            hi = fminf(fmaxf(hi, -MOST), MOST);
            __half offset = __float2half_rn(lo);
            const float o = __half2float(offset);
            __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, o), 1.0f / TOP));
            const float st = __half2float(scale);
            uint32_t code[2] = {0, 0};
            if (bad != 0.0f) {
                scale = offset = __float2half_rn(__int_as_float(0x7FC00000));
            } else if (st > 0.0f) {
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const float y = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[s], o), st)), 0.0f), TOP);
                    code[BITS == 4 ? 0 : s >> 2] |= (uint32_t)y << (BITS == 4 ? 4 * s : 8 * (s & 3));
                }
            }
            const int kh = h - p.q_heads - (is_v ? p.kv_heads : 0);
            uint8_t *row = static_cast<uint8_t *>(is_k ? p.k_pages : p.v_pages) + walk.row(p.batch, p.page_stride, p.token_stride) +
                           kh * p.head_stride + sl * BITS;
            if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(row) = code[0];
            else *reinterpret_cast<uint2 *>(row) = make_uint2(code[0], code[1]);
            if (sl % (p.z.group / 8) == 0) {
                __half2 *pair = const_cast<__half2 *>(is_k ? p.z.k_scales : p.z.v_scales) +
                                walk.row(p.batch, p.z.page_stride, p.z.token_stride) + kh * p.z.head_stride + 8 * sl / p.z.group;
                *pair = __halves2half2(scale, offset);
            }
        }
    };

    for (int t = t0; t < t1; ++t) {
        Eight<S> now, next;
        // the whole warp runs while one of its heads is there
        int h = h_first;
        load(now, t, h);
        place(t);
        while (h - lane / p.seg < heads) {
            if (h + step - lane / p.seg < heads) load(next, t, h + step);
            finish(now, t, h);
            now = next;
            h += step;
        }
    }
}

template <typename S, typename T, int BITS> inline int launch_heads(HeadsParams &p, bool vec, cudaStream_t stream) {
    p.seg = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 16 : 32;
    const int heads = p.q_heads + 2 * p.kv_heads;
    // few tokens: a token's heads over several blocks; many: runs of consecutive tokens
    const int64_t slots = (int64_t)sm_count() * 8, parts = ceil_div(heads, HEADS_WARPS * (32 / p.seg));
    int64_t split = slots / p.tokens;
    split = split < 1 ? 1 : split > parts ? parts : split;
    if (split > 65535) split = 65535;
    p.per_block = (int)ceil_div(p.tokens, slots / split);
    const dim3 grid((unsigned)ceil_div(p.tokens, p.per_block), (unsigned)split);
    if (vec) kv_append_heads_kernel<S, T, BITS, true><<<grid, 32 * HEADS_WARPS, 0, stream>>>(p);
    else kv_append_heads_kernel<S, T, BITS, false><<<grid, 32 * HEADS_WARPS, 0, stream>>>(p);
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
                     (!p.rot || (aligned(b.cos, 16) && aligned(b.sin, 16) && b.table_row % 4 == 0));
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
