// Reading quantised pages back: the packed rows of a batch get the values that their positions hold,
// scale * code + offset in fp32 (the product is exact), rounded once to the output's type: the inverse of
// the append with the same batch. Memory bounds it, the writes above all: 131071 positions of 8 heads x 128 in 4 bits to
// bf16, 679 MB, in 131 us (5.2 TB/s, 80 % of the copy bandwidth).
#pragma once

#include "quantized_common.cuh"

namespace mgc {
namespace paged {

struct ReadParams {
    Batch batch;
    Quantized z;
    const uint8_t *k_pages, *v_pages;
    long long page_stride, token_stride, head_stride;  // bytes
    void *k_out, *v_out;
    long long k_ts, k_hs, v_ts, v_hs;
    int kv_heads, head_dim;
    int seg;  // lanes of a head, eight channels each
    int tokens, run, parts;
};

// Eight consecutive codes as they are stored, and as the floats scale * code + offset. A code is put into the
// mantissa of 2^23, which comes off exactly (a conversion instruction takes a quarter of the rate); a nibble further up
// stays there, 16^k times as large, and the scale is as much smaller: the product is the same.
template <int BITS> struct EightCodes;
template <> struct EightCodes<4> {
    uint32_t w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = __ldg(reinterpret_cast<const unsigned int *>(p)); }
    __device__ __forceinline__ void values(float2 so, float (&x)[8]) const {
        const uint32_t up = w >> 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = i & 3;
            const float code = __uint_as_float(((i < 4 ? w : up) & 15u << 4 * k) | 0x4B000000u) - 8388608.0f;
            x[i] = fmaf(k == 0 ? so.x : k == 1 ? so.x * 0.0625f : k == 2 ? so.x * 0.00390625f : so.x * 0.000244140625f, code, so.y);
        }
    }
};
template <> struct EightCodes<8> {
    uint2 w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = __ldg(reinterpret_cast<const uint2 *>(p)); }
    __device__ __forceinline__ void values(float2 so, float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = fmaf(so.x, __uint_as_float(__byte_perm(i < 4 ? w.x : w.y, 0x4B000000u, 0x7650 | (i & 3))) - 8388608.0f, so.y);
    }
};

constexpr int READ_WARPS = 4, READ_RESIDENT = 8;

template <typename T, int BITS, bool VEC>
__global__ void __launch_bounds__(32 * READ_WARPS, READ_RESIDENT) kv_read_kernel(const __grid_constant__ ReadParams p) {
    const int lane = (int)(threadIdx.x & 31);
    const unsigned unit = blockIdx.x * READ_WARPS + threadIdx.x / 32;
    const int sl = lane & (p.seg - 1), at_once = 32 / p.seg, part = (int)(unit % (unsigned)p.parts);
    const long long t_first = (long long)(unit / (unsigned)p.parts) * p.run;
    if (unit == 0 && lane == 0) check_rows(p.batch, p.tokens);
    if (t_first >= p.tokens) return;
    const int t0 = (int)t_first, t1 = min(t0 + p.run, p.tokens);
    const int h0 = part * at_once + lane / p.seg, step = p.parts * at_once;
    const bool mine = 8 * sl < p.head_dim;
    const int group = 8 * sl / p.z.group;
    auto put = [&](T *dst, const EightCodes<BITS> &c, __half2 pair) {
        float x[8];
        c.values(__half22float2(pair), x);
        if constexpr (VEC) {
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<uint4 *>(dst) = make_uint4(two<T>(x[0], x[1]), two<T>(x[2], x[3]), two<T>(x[4], x[5]), two<T>(x[6], x[7]));
            } else {
                *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4 *>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = from_f<T>(x[e]);
        }
    };
    TokenWalk walk;
    walk.start(t0);
    for (int t = t0; t < t1; ++t) {
        walk.step(p.batch, t);
        const bool there = walk.page >= 0;
        const long long codes = (there ? walk.at(p.page_stride, p.token_stride) : 0) + h0 * p.head_stride + sl * BITS;
        const long long pairs = (there ? walk.at(p.z.page_stride, p.z.token_stride) : 0) + h0 * p.z.head_stride + group;
        const uint8_t *k = p.k_pages + codes, *v = p.v_pages + codes;
        const __half2 *ks = p.z.k_scales + pairs, *vs = p.z.v_scales + pairs;
        T *k_dst = static_cast<T *>(p.k_out) + (long long)t * p.k_ts + h0 * p.k_hs + 8 * sl;
        T *v_dst = static_cast<T *>(p.v_out) + (long long)t * p.v_ts + h0 * p.v_hs + 8 * sl;
        // two heads' keys and values in flight
        constexpr int BATCH = 2;
        for (int h = h0; h - lane / p.seg < p.kv_heads; h += BATCH * step) {
            EightCodes<BITS> c[BATCH][2];
            __half2 so[BATCH][2];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                so[i][0] = so[i][1] = __floats2half2_rn(0.0f, 0.0f);
                c[i][0] = c[i][1] = EightCodes<BITS>{};
                if (there && mine && h + i * step < p.kv_heads) {
                    c[i][0].load(k);
                    c[i][1].load(v);
                    so[i][0] = __ldg(ks);
                    so[i][1] = __ldg(vs);
                }
                k += step * p.head_stride;
                v += step * p.head_stride;
                ks += step * p.z.head_stride;
                vs += step * p.z.head_stride;
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                if (mine && h + i * step < p.kv_heads) {
                    put(k_dst, c[i][0], so[i][0]);
                    put(v_dst, c[i][1], so[i][1]);
                }
                k_dst += step * p.k_hs;
                v_dst += step * p.v_hs;
            }
        }
    }
}

template <typename T, int BITS> inline int launch_read(ReadParams &p, bool vec, cudaStream_t stream) {
    p.seg = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 16 : 32;
    const TokenRuns r = runs_of(p.tokens, ceil_div(p.kv_heads, 32 / p.seg), READ_WARPS, READ_RESIDENT);
    p.run = r.run;
    p.parts = r.parts;
    if (vec) kv_read_kernel<T, BITS, true><<<r.blocks, 32 * READ_WARPS, 0, stream>>>(p);
    else kv_read_kernel<T, BITS, false><<<r.blocks, 32 * READ_WARPS, 0, stream>>>(p);
    return check_launch("kv_read_kernel");
}

inline int read_back(const mgc_cuda_kv_read_args &a, cudaStream_t stream) {
    const char *what = "mgc_cuda_kv_read";
    const mgc_cuda_paged &c = a.paged;
    MGC_CHECK(check_paged(c, what));
    MGC_CHECK(check_quantized(a.quantized, c, what));
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
    if (!a.k_out || !a.v_out) return fail(MGC_CUDA_BAD_ARGUMENT, "%s: an output is NULL", what);
    ReadParams p;
    p.batch = batch_of(c);
    p.z = quantized_of(a.quantized, c);
    p.k_pages = static_cast<const uint8_t *>(c.k);
    p.v_pages = static_cast<const uint8_t *>(c.v);
    p.page_stride = c.page_stride; p.token_stride = c.token_stride; p.head_stride = c.head_stride;
    p.k_out = a.k_out; p.v_out = a.v_out;
    p.k_ts = a.k_token_stride; p.k_hs = a.k_head_stride; p.v_ts = a.v_token_stride; p.v_hs = a.v_head_stride;
    p.kv_heads = (int)c.kv_heads; p.head_dim = (int)c.head_dim;
    p.tokens = (int)c.tokens;
    const int chunk = 16 / elem_size(c.dtype);
    const bool vec = aligned(p.k_out, 16) && aligned(p.v_out, 16) && p.k_ts % chunk == 0 && p.k_hs % chunk == 0 && p.v_ts % chunk == 0 &&
                     p.v_hs % chunk == 0;
    auto types = [&](auto out) {
        using T = decltype(out);
        return a.quantized.bits == 4 ? launch_read<T, 4>(p, vec, stream) : launch_read<T, 8>(p, vec, stream);
    };
    if (c.dtype == MGC_F32) return types(float());
    return c.dtype == MGC_F16 ? types(__half()) : types(__nv_bfloat16());
}

}  // namespace paged
}  // namespace mgc
