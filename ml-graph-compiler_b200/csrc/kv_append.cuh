// Append of new keys and values to a paged cache, the position rotation on the way.
//
//   k_pages[page(p)][p % page_size] = R_p k_t,   v_pages[...] = v_t,   q_out[t] = R_p q_t
// with R_p turning pair (x1, x2) of the first `rot` channels by the angle whose cosine and sine
// are row p of the tables: x1' = x1 c - x2 s, x2' = x2 c + x1 s, in fp32, rounded once.
//
// Every value is read once and written once and the arithmetic is three operations per rotated
// value, so memory bounds it (latency for a few tokens). A block takes a run of consecutive tokens:
// its warps find a sequence with one ballot per 32 sequences and count on from there, looking up a
// page where one begins. Each thread moves units of V channels of a head (16 bytes), a rotated unit
// being the two chunks whose channels pair up, so that each pair is read and written by one thread
// and q may be rotated in place. A thread's units are the same channels of several heads, so it
// reads a token's angles once. 19466 tokens of 48 heads x 128, bf16: 86 to 88 us, 5.5 TB/s (85 % of the
// copy bandwidth).
#pragma once

#include "paged_common.cuh"

namespace mgc {
namespace paged {

struct AppendParams {
    Batch batch;
    void *k_pages, *v_pages;
    long long page_stride, token_stride, head_stride;
    const void *q, *k, *v;
    void *q_out;
    long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs;
    const float *cos, *sin;
    long long table_row;
    int positions, rot, interleaved;
    int q_heads, kv_heads, head_dim;
    int threads;  // that work: a multiple of units
    int tokens, per_block;
    int units;    // per head: rot / 2V rotated pairs of chunks, then (head_dim - rot) / V plain chunks
};

// V values of the tables, which the vector forms read 16 bytes at a time.
template <int V> __device__ __forceinline__ void load_angles(const float *p, float (&x)[V]) {
    Pack<V, float> a;
    a.load(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = a.e[i];
}

// One unit of a head on its way.
template <typename S, typename T, int V> struct Unit {
    Pack<V, S> x, y;
};

// Blocks an SM holds, by registers: 4 (64 registers) ran 19466 tokens of 48 heads x 128 bf16 in 84 us,
// 5 to 8 (spills) in 124 to 247 us, unbounded (85 registers) in 138 us. The wide fp32 units need more.
template <typename S, int V> constexpr int RESIDENT = V * (int)sizeof(S) > 16 ? 2 : 4;

template <typename S, typename T, int V>
__global__ void __launch_bounds__(256, RESIDENT<S, V>) kv_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int BATCH = 2;
    const int t0 = (int)blockIdx.x * p.per_block, t1 = min(t0 + p.per_block, p.tokens);
    // thread (w, h0) takes unit w of heads h0, h0 + step, ...
    const int h0 = (int)threadIdx.x / p.units, w = (int)threadIdx.x - h0 * p.units, step = p.threads / p.units;
    const int heads = p.q_heads + 2 * p.kv_heads, pairs = p.rot / (2 * V);
    const bool pair = w < pairs, active = (int)threadIdx.x < p.threads;
    const int c0 = !pair ? p.rot + (w - pairs) * V : p.interleaved ? w * 2 * V : w * V;
    const int c1 = p.interleaved ? c0 + V : c0 + p.rot / 2;
    auto load = [&](Unit<S, T, V> &z, int t, int h) {
        if (h >= heads || !active) return;
        const S *src;
        if (h < p.q_heads) {
            src = static_cast<const S *>(p.q) + t * p.q_ts + h * p.q_hs;
        } else if (h < p.q_heads + p.kv_heads) {
            src = static_cast<const S *>(p.k) + t * p.k_ts + (h - p.q_heads) * p.k_hs;
        } else {
            src = static_cast<const S *>(p.v) + t * p.v_ts + (h - p.q_heads - p.kv_heads) * p.v_hs;
        }
        z.x.load(src + c0);
        if (pair) z.y.load(src + c1);
    };
    // the place of token t: looked up where a sequence or a page begins, counted on in between
    int b = -1, end = t0, n = 0, page = -1, held = -1;
    float c[V], s[V];
    auto finish = [&](Unit<S, T, V> &z, int t, int h, bool turn, long long slot) {
        if (h >= heads || !active) return;
        T *dst;
        bool rotate = turn;
        if (h < p.q_heads) {
            dst = static_cast<T *>(p.q_out) + t * p.qo_ts + h * p.qo_hs;
        } else {
            if (slot < 0) return;
            h -= p.q_heads;
            rotate = rotate && h < p.kv_heads;
            dst = static_cast<T *>(h < p.kv_heads ? p.k_pages : p.v_pages) + slot + (h < p.kv_heads ? h : h - p.kv_heads) * p.head_stride;
        }
        Pack<V, T> ox, oy;
        if (!pair) {
#pragma unroll
            for (int i = 0; i < V; ++i) ox.e[i] = from_f<T>(to_f(z.x.e[i]));
            ox.store(dst + c0);
            return;
        }
        float v[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = to_f(z.x.e[i]);
            v[V + i] = to_f(z.y.e[i]);
        }
        if (rotate) {
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float x1 = v[2 * i], x2 = v[2 * i + 1];
                    v[2 * i] = x1 * c[i] - x2 * s[i];
                    v[2 * i + 1] = x2 * c[i] + x1 * s[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float x1 = v[i], x2 = v[V + i];
                    v[i] = x1 * c[i] - x2 * s[i];
                    v[V + i] = x2 * c[i] + x1 * s[i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            ox.e[i] = from_f<T>(v[i]);
            oy.e[i] = from_f<T>(v[V + i]);
        }
        ox.store(dst + c0);
        oy.store(dst + c1);
    };
    auto place = [&](Unit<S, T, V> (&u)[BATCH], int t) {
        if (t >= end) {
            b = sequence_of(p.batch, t);
            end = b < 0 ? t : __ldg(p.batch.q_starts + b + 1);
            n = b < 0 ? 0 : __ldg(p.batch.kv_lens + b);
            if (t >= end) {  // in no sequence: position -1, nowhere to cache, nothing to rotate by
                end = t + 1;
                n = 0;
            }
            held = -1;
        }
        const int pos = n - (end - t);
        if (pos >= 0 && (held < 0 || pos / p.batch.page_size != held)) {
            held = pos / p.batch.page_size;
            page = page_of(p.batch, b, held);
        }
        bool turn = pos >= 0 && p.rot > 0;
        long long slot = pos < 0 || page < 0
                             ? -1
                             : (long long)page * p.page_stride + (long long)(pos - held * p.batch.page_size) * p.token_stride;
        if (turn && pos >= p.positions) {
            if (p.batch.status) *p.batch.status = MGC_CUDA_GATHER_OOB;
            turn = false;
            slot = -1;
        }
        if (turn && pair) {
            load_angles<V>(p.cos + (long long)pos * p.table_row + w * V, c);
            load_angles<V>(p.sin + (long long)pos * p.table_row + w * V, s);
        }
        for (int h = h0;;) {
#pragma unroll
            for (int i = 0; i < BATCH; ++i) finish(u[i], t, h + i * step, turn, slot);
            h += BATCH * step;
            if (h >= heads) break;
#pragma unroll
            for (int i = 0; i < BATCH; ++i) load(u[i], t, h + i * step);
        }
    };
    // a token's sources load while its place is found (the next token's in a second set of registers
    // left fewer blocks on an SM: 144 us)
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.batch.status && __ldg(p.batch.q_starts + p.batch.batch) > p.tokens)
        *p.batch.status = MGC_CUDA_GATHER_OOB;
    Unit<S, T, V> u[BATCH];
    for (int t = t0; t < t1; ++t) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) load(u[i], t, h0 + i * step);
        place(u, t);
    }
}

template <typename S, typename T, int V> inline int run_append(AppendParams &p, int tokens, cudaStream_t stream) {
    p.units = p.rot / (2 * V) + (p.head_dim - p.rot) / V;
    const int heads = p.q_heads + 2 * p.kv_heads;
    if (p.units > 256) return fail(MGC_CUDA_UNSUPPORTED, "mgc_cuda_kv_append: %d channels in units of %d", p.head_dim, V);
    // whole heads of units, at most 256 threads
    p.threads = (heads < 256 / p.units ? heads : 256 / p.units) * p.units;
    // runs of consecutive tokens, as many as the GPU holds blocks
    p.tokens = tokens;
    p.per_block = (int)ceil_div(tokens, (int64_t)sm_count() * RESIDENT<S, V>);
    kv_append_kernel<S, T, V><<<(unsigned)ceil_div(tokens, p.per_block), (unsigned)ceil_div(p.threads, 32) * 32, 0, stream>>>(p);
    return check_launch("kv_append_kernel");
}

// The widest unit that the sizes, strides and addresses allow: 16-byte stores, half of that (head
// widths and rotated widths that come in fours), else single channels.
template <typename S, typename T> inline int launch_append(AppendParams &p, int tokens, cudaStream_t stream) {
    auto fits = [&](int v) {
        const int sb = v * (int)sizeof(S) > 16 ? 16 : v * (int)sizeof(S), tb = v * (int)sizeof(T);
        auto src = [&](const void *q, long long ts, long long hs) {
            return aligned(q, sb) && ts * (long long)sizeof(S) % sb == 0 && hs * (long long)sizeof(S) % sb == 0;
        };
        auto dst = [&](const void *q, long long ts, long long hs) {
            return aligned(q, tb) && ts * (long long)sizeof(T) % tb == 0 && hs * (long long)sizeof(T) % tb == 0;
        };
        return p.head_dim % v == 0 && p.rot % (2 * v) == 0 && src(p.k, p.k_ts, p.k_hs) && src(p.v, p.v_ts, p.v_hs) &&
               (!p.q || (src(p.q, p.q_ts, p.q_hs) && dst(p.q_out, p.qo_ts, p.qo_hs))) &&
               dst(p.k_pages, p.token_stride, p.head_stride) && dst(p.v_pages, p.page_stride, p.head_stride) &&
               (!p.rot || (aligned(p.cos, 16) && aligned(p.sin, 16) && p.table_row % 4 == 0));
    };
    constexpr int WIDE = 16 / (int)sizeof(T);
    if (fits(WIDE)) return run_append<S, T, WIDE>(p, tokens, stream);
    if (WIDE > 4 && fits(4)) return run_append<S, T, 4>(p, tokens, stream);
    return run_append<S, T, 1>(p, tokens, stream);
}

inline int append(const mgc_cuda_kv_append_args &a, cudaStream_t stream) {
    const char *what = "mgc_cuda_kv_append";
    const mgc_cuda_paged &c = a.paged;
    MGC_CHECK(check_paged(c, what));
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
    if (!a.k || !a.v || (a.q && !a.q_out) || a.q_heads < 0 || a.rot < 0 || a.rot > c.head_dim || a.rot % 2 ||
        (a.rot && (!a.cos || !a.sin || a.positions < 0 || a.table_row < 0)))
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: missing operand or bad rotation width %lld", what, (long long)a.rot);
    if (a.src_dtype != c.dtype && a.src_dtype != MGC_F32)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: sources of type %d for pages of type %d", what, (int)a.src_dtype, (int)c.dtype);
    if (a.q && a.q == a.q_out &&
        (a.src_dtype != c.dtype || a.q_token_stride != a.qo_token_stride || a.q_head_stride != a.qo_head_stride))
        return fail(MGC_CUDA_BAD_ARGUMENT, "%s: q rotated in place keeps its type and strides", what);
    const int64_t heads = (a.q ? a.q_heads : 0) + 2 * c.kv_heads;
    if (c.head_dim > 256 || heads > 1 << 20 || heads * c.head_dim > 0x7FFFFFFF)
        return fail(MGC_CUDA_UNSUPPORTED, "%s: %lld heads of %lld channels", what, (long long)heads, (long long)c.head_dim);
    AppendParams p;
    p.batch = batch_of(c);
    p.k_pages = c.k; p.v_pages = c.v;
    p.page_stride = c.page_stride; p.token_stride = c.token_stride; p.head_stride = c.head_stride;
    p.q = a.q; p.k = a.k; p.v = a.v; p.q_out = a.q_out;
    p.q_ts = a.q_token_stride; p.q_hs = a.q_head_stride;
    p.k_ts = a.k_token_stride; p.k_hs = a.k_head_stride;
    p.v_ts = a.v_token_stride; p.v_hs = a.v_head_stride;
    p.qo_ts = a.qo_token_stride; p.qo_hs = a.qo_head_stride;
    p.cos = a.cos; p.sin = a.sin; p.table_row = a.table_row;
    p.positions = (int)(a.positions > 0x7FFFFFFF ? 0x7FFFFFFF : a.positions);
    p.rot = (int)a.rot; p.interleaved = a.interleaved != 0;
    p.q_heads = a.q ? (int)a.q_heads : 0; p.kv_heads = (int)c.kv_heads; p.head_dim = (int)c.head_dim;
    const int n = (int)c.tokens;
    const bool wide = a.src_dtype == MGC_F32;
    if (c.dtype == MGC_F32) return launch_append<float, float>(p, n, stream);
    if (c.dtype == MGC_F16)
        return wide ? launch_append<float, __half>(p, n, stream) : launch_append<__half, __half>(p, n, stream);
    return wide ? launch_append<float, __nv_bfloat16>(p, n, stream)
                : launch_append<__nv_bfloat16, __nv_bfloat16>(p, n, stream);
}

}  // namespace paged
}  // namespace mgc
