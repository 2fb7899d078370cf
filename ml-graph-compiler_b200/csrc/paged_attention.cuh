// Attention of new tokens over a paged cache.
//
//   o_t[h] = sum_j w_j v_j,   w = softmax over the visible positions j of scale * q_t[h] . k_j
// computed in one pass over the keys with the running maximum m and sum l of the softmax:
//   m' = max(m, s_j),  l' = l e^(m - m') + e^(s_j - m'),  o' = o e^(m - m') + e^(s_j - m') v_j,
// exponentials in base 2 (scale carries log2 e), everything in fp32.
#pragma once

#include "paged_common.cuh"

namespace mgc {
namespace paged {

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
};

constexpr int MAX_HEAD_DIM = 256;

// Visible positions [lo, hi) of a token at position pos of a sequence of n positions.
__device__ __forceinline__ void visible(const AttendParams &p, int n, int pos, int &lo, int &hi) {
    hi = p.causal ? min(n, pos + 1) : n;
    lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
}

// One warp per (token, query head), lane l holding channels l, l + 32, ...: any type, head width,
// stride and page size.
template <typename T>
__global__ void __launch_bounds__(128) paged_attention_row_kernel(const __grid_constant__ AttendParams p) {
    constexpr int C = MAX_HEAD_DIM / 32;
    const int lane = (int)(threadIdx.x & 31);
    const int t = (int)blockIdx.x;
    const int h = (int)blockIdx.y * 4 + (int)(threadIdx.x >> 5);
    const int b = sequence_of(p.batch, t);
    if (b < 0 || h >= p.q_heads) return;
    const int end = __ldg(p.batch.q_starts + b + 1);
    if (t >= end) return;
    const int n = __ldg(p.batch.kv_lens + b);
    int lo, hi;
    visible(p, n, n - (end - t), lo, hi);
    const T *q = static_cast<const T *>(p.q) + t * p.q_ts + h * p.q_hs;
    const long long head = (h / p.group) * p.head_stride;
    float qv[C], o[C], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int d = lane + 32 * c;
        qv[c] = d < p.head_dim ? to_f(q[d]) * p.scale_log2 : 0.0f;
        o[c] = 0.0f;
    }
    for (int j = lo; j < hi; ++j) {
        const int page = page_of(p.batch, b, j / p.batch.page_size);
        if (page < 0) continue;
        const long long at = page * p.page_stride + (j % p.batch.page_size) * p.token_stride + head;
        const T *k = static_cast<const T *>(p.k_pages) + at, *v = static_cast<const T *>(p.v_pages) + at;
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = lane + 32 * c;
            if (d < p.head_dim) s += qv[c] * to_f(k[d]);
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
        if (s == -INFINITY) continue;  // weighs nothing (and would leave -inf - -inf at the start)
        const float m2 = fmaxf(m, s), scale = exp2f(m - m2), w = exp2f(s - m2);
        l = l * scale + w;
        m = m2;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = lane + 32 * c;
            if (d < p.head_dim) o[c] = o[c] * scale + w * to_f(v[d]);
        }
    }
    T *out = static_cast<T *>(p.out) + t * p.o_ts + h * p.o_hs;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int d = lane + 32 * c;
        if (d < p.head_dim) out[d] = from_f<T>(o[c] * inv);
    }
}

inline int64_t attend_workspace(const mgc_cuda_paged_attention_args &a) {
    (void)a;
    return 0;
}

inline int attend(const mgc_cuda_paged_attention_args &a, cudaStream_t stream) {
    const char *what = "mgc_cuda_paged_attention";
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
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
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
    const dim3 grid((unsigned)p.tokens, (unsigned)ceil_div(p.q_heads, 4));
    if (c.dtype == MGC_F32) paged_attention_row_kernel<float><<<grid, 128, 0, stream>>>(p);
    else if (c.dtype == MGC_F16) paged_attention_row_kernel<__half><<<grid, 128, 0, stream>>>(p);
    else paged_attention_row_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(p);
    return check_launch("paged_attention_row_kernel");
}

}  // namespace paged
}  // namespace mgc
