// Attention of new tokens over quantised pages (quantized_common.cuh): paged_attention_params.cuh's
// definition with k_j and v_j the values that the codes stand for.
#pragma once

#include "paged_work.cuh"
#include "quantized_common.cuh"

namespace mgc {
namespace paged {

// One warp per (token, query head), lane l holding channels l, l + 32, ...
template <typename T, int BITS>
__global__ void __launch_bounds__(128) quantized_attention_row_kernel(const __grid_constant__ AttendParams p, const Quantized z) {
    constexpr int C = MAX_HEAD_DIM / 32;
    const int lane = (int)(threadIdx.x & 31);
    const int t = (int)blockIdx.x;
    const int h = (int)blockIdx.y * 4 + (int)(threadIdx.x >> 5);
    if (t == 0 && h == 0)
        for (int i = lane; i < p.batch.batch; i += 32) check_sequence(p, i);
    const int b = sequence_of(p.batch, t);
    if (h >= p.q_heads) return;
    T *out = static_cast<T *>(p.out) + t * p.o_ts + h * p.o_hs;
    const int end = b < 0 ? t : __ldg(p.batch.q_starts + b + 1);
    if (t >= end) {  // in no sequence
        for (int d = lane; d < p.head_dim; d += 32) out[d] = from_f<T>(0.0f);
        return;
    }
    const int length = __ldg(p.batch.kv_lens + b), kh = h / p.group;
    int lo, hi;
    visible(p, min(length, p.max_positions), length - (end - t), lo, hi);
    const T *q = static_cast<const T *>(p.q) + t * p.q_ts + h * p.q_hs;
    float qv[C], o[C], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int d = lane + 32 * c;
        qv[c] = lo < hi && d < p.head_dim ? to_f(q[d]) * p.scale_log2 : 0.0f;
        o[c] = 0.0f;
    }
    for (int j = lo; j < hi; ++j) {
        const int page = page_of(p.batch, b, j / p.batch.page_size);
        if (page < 0) continue;
        const int r = j % p.batch.page_size;
        const long long at = page * p.page_stride + r * p.token_stride + kh * p.head_stride;
        const long long pair = page * z.page_stride + r * z.token_stride + kh * z.head_stride;
        auto value = [&](const void *pages, const __half2 *scales, int d) {
            const uint8_t *row = static_cast<const uint8_t *>(pages) + at;
            const int code = BITS == 8 ? row[d] : row[d >> 1] >> 4 * (d & 1) & 15;
            const float2 so = __half22float2(scales[pair + d / z.group]);
            return fmaf(so.x, (float)code, so.y);
        };
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = lane + 32 * c;
            if (d < p.head_dim) s += qv[c] * value(p.k_pages, z.k_scales, d);
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
        if (s == -INFINITY) continue;
        const float m2 = fmaxf(m, s), scale = exp2f(m - m2), w = exp2f(s - m2);
        l = l * scale + w;
        m = m2;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = lane + 32 * c;
            if (d < p.head_dim) o[c] = o[c] * scale + w * value(p.v_pages, z.v_scales, d);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : l != l ? l : 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int d = lane + 32 * c;
        if (d < p.head_dim) out[d] = from_f<T>(o[c] * inv);
    }
}

inline int check_attend_quantized(const mgc_cuda_paged_attention_quantized_args &a, const char *what) {
    MGC_CHECK(check_attend(a.attention, what));
    return check_quantized(a.quantized, a.attention.paged, what);
}

inline int64_t attend_quantized_workspace(const mgc_cuda_paged_attention_quantized_args &a) {
    if (check_attend_quantized(a, "mgc_cuda_paged_attention_quantized_workspace") != MGC_CUDA_OK) return -1;
    return 0;
}

inline int attend_quantized(const mgc_cuda_paged_attention_quantized_args &a, cudaStream_t stream) {
    const char *what = "mgc_cuda_paged_attention_quantized";
    const mgc_cuda_paged &c = a.attention.paged;
    MGC_CHECK(check_attend_quantized(a, what));
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
    const AttendParams p = attend_params(a.attention);
    const Quantized z = quantized_of(a.quantized, c);
    const dim3 grid((unsigned)p.tokens, (unsigned)ceil_div(p.q_heads, 4));
    auto go = [&](auto type) {
        using T = decltype(type);
        if (z.bits == 4) quantized_attention_row_kernel<T, 4><<<grid, 128, 0, stream>>>(p, z);
        else quantized_attention_row_kernel<T, 8><<<grid, 128, 0, stream>>>(p, z);
        return check_launch("quantized_attention_row_kernel");
    };
    if (c.dtype == MGC_F32) return go(float());
    return c.dtype == MGC_F16 ? go(__half()) : go(__nv_bfloat16());
}

}  // namespace paged
}  // namespace mgc
