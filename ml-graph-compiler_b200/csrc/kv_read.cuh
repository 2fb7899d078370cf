// Reading quantised pages back: the packed rows of a batch get the values that their positions hold,
// scale * code + offset in fp32 (the product is exact), rounded once to the output's type: the inverse of
// the append with the same batch. Memory bounds it, the writes above all.
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
    int tokens, per_block;
};

// Eight consecutive codes as floats.
template <int BITS> __device__ __forceinline__ void eight_codes(const uint8_t *p, float (&x)[8]) {
    if constexpr (BITS == 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)(w >> 4 * i & 15);
    } else {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)((i < 4 ? w.x : w.y) >> 8 * (i & 3) & 255);
    }
}

template <typename T, int BITS, bool VEC>
__global__ void __launch_bounds__(128) kv_read_kernel(const __grid_constant__ ReadParams p) {
    const int lane = (int)(threadIdx.x & 31), warp = (int)(threadIdx.x >> 5);
    const int sl = lane & (p.seg - 1), at_once = 32 / p.seg;
    const int step = (int)gridDim.y * 4 * at_once, h0 = ((int)blockIdx.y * 4 + warp) * at_once + lane / p.seg;
    const int t0 = (int)blockIdx.x * p.per_block, t1 = min(t0 + p.per_block, p.tokens);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) check_rows(p.batch, p.tokens);
    TokenWalk walk;
    walk.start(t0);
    for (int t = t0; t < t1; ++t) {
        walk.step(p.batch, t);
        const bool there = walk.page >= 0;
        const long long codes = there ? walk.row(p.batch, p.page_stride, p.token_stride) : 0;
        const long long pairs = there ? walk.row(p.batch, p.z.page_stride, p.z.token_stride) : 0;
        if (8 * sl >= p.head_dim) continue;  // (the next step's lanes meet again)
        for (int h = h0; h < 2 * p.kv_heads; h += step) {
            const bool is_v = h >= p.kv_heads;
            const int kh = is_v ? h - p.kv_heads : h;
            float x[8], scale = 0.0f, offset = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.0f;
            if (there) {
                eight_codes<BITS>((is_v ? p.v_pages : p.k_pages) + codes + kh * p.head_stride + sl * BITS, x);
                const float2 so = __half22float2((is_v ? p.z.v_scales : p.z.k_scales)[pairs + kh * p.z.head_stride + 8 * sl / p.z.group]);
                scale = so.x;
                offset = so.y;
            }
            T *dst = static_cast<T *>(is_v ? p.v_out : p.k_out) + t * (is_v ? p.v_ts : p.k_ts) + kh * (is_v ? p.v_hs : p.k_hs) + 8 * sl;
            Pack<8, T> y;
#pragma unroll
            for (int i = 0; i < 8; ++i) y.e[i] = from_f<T>(fmaf(scale, x[i], offset));
            if constexpr (VEC) {
                y.store(dst);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) dst[i] = y.e[i];
            }
        }
    }
}

template <typename T, int BITS> inline int launch_read(ReadParams &p, bool vec, cudaStream_t stream) {
    p.seg = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? 16 : 32;
    const int64_t slots = (int64_t)sm_count() * 16, parts = ceil_div(2 * p.kv_heads, 4 * (32 / p.seg));
    int64_t split = slots / p.tokens;
    split = split < 1 ? 1 : split > parts ? parts : split;
    p.per_block = (int)ceil_div(p.tokens, slots / split);
    const dim3 grid((unsigned)ceil_div(p.tokens, p.per_block), (unsigned)split);
    if (vec) kv_read_kernel<T, BITS, true><<<grid, 128, 0, stream>>>(p);
    else kv_read_kernel<T, BITS, false><<<grid, 128, 0, stream>>>(p);
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
