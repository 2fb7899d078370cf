// How the work of an attention call is cut evenly over its CTAs, and the kernel that adds the pieces.
#pragma once

#include "paged_attention_params.cuh"

namespace mgc {
namespace paged {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A sequence: its first new token's row and position, its new tokens (rows of q outside it do not
// exist and are left out), and the positions that can be read (its length, cut off where the block
// table ends). Neither cut moves the tokens that are left.
struct Sequence { int start, base, nq, n; };
__device__ __forceinline__ Sequence load_sequence(const AttendParams &p, int b) {
    const int start = __ldg(p.batch.q_starts + b), end = __ldg(p.batch.q_starts + b + 1), length = __ldg(p.batch.kv_lens + b);
    Sequence s;
    s.start = max(start, 0);
    s.nq = max(min(end, p.tokens) - s.start, 0);
    s.base = length - (end - s.start);
    s.n = min(length, p.max_positions);
    return s;
}
// Sets the status word if something of sequence b was cut off.
__device__ __forceinline__ void check_sequence(const AttendParams &p, int b) {
    const int start = __ldg(p.batch.q_starts + b), end = __ldg(p.batch.q_starts + b + 1);
    if (p.batch.status && (start < 0 || end < start || end > p.tokens || (end > start && __ldg(p.batch.kv_lens + b) > p.max_positions)))
        *p.batch.status = MGC_CUDA_GATHER_OOB;
}

// Zeros in the rows of out that no sequence has (a batch padded to a fixed number of rows): this warp
// takes heads h0, h0 + step, ... of tokens t0, t0 + t_step, ... For kernels whose rows are 16-byte
// chunks.
template <typename T> __device__ __forceinline__ void zero_outside(const AttendParams &p, int t0, int t_step, int h0, int h_step, int lane) {
    const int first = min(max(__ldg(p.batch.q_starts), 0), p.tokens);
    const int last = min(max(__ldg(p.batch.q_starts + p.batch.batch), first), p.tokens);
    if (first == 0 && last == p.tokens) return;
    for (long long i = t0; i < first + p.tokens - last; i += t_step) {
        T *row = static_cast<T *>(p.out) + (i < first ? i : i - first + last) * p.o_ts;
        for (int h = h0; h < p.q_heads; h += h_step)
            for (int d = lane * (16 / (int)sizeof(T)); d < p.head_dim; d += 32 * (16 / (int)sizeof(T)))
                *reinterpret_cast<uint4 *>(row + h * p.o_hs + d) = make_uint4(0, 0, 0, 0);
    }
}

// Visible keys of a row (a token and a head); rows past the last see nothing.
struct RowRange { int lo, hi; };
__device__ __forceinline__ RowRange row_range(const AttendParams &p, const Sequence &s, int row) {
    RowRange r{0, 0};
    const int i = row / p.group;
    if (i < s.nq) visible(p, s.n, s.base + i, r.lo, r.hi);
    return r;
}

// One query row by the definition, a key at a time, lane l holding channels l, l + 32, ...: maximum
// (scaled, base 2), sum, output. What the kernels for unaligned operands and the pieces with missing
// pages or values that are not finite take.
template <int C> struct RowSum {
    float o[C], m, l;
    __device__ __forceinline__ RowSum() {}
    template <typename T>
    __device__ __forceinline__ void over_keys(const AttendParams &p, int b, int kh, const T *q, int lo, int hi, int lane) {
        const long long head = kh * p.head_stride;
        float qv[C];
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = lane + 32 * c;
            qv[c] = lo < hi && d < p.head_dim ? to_f(q[d]) * p.scale_log2 : 0.0f;
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
            const float m2 = fmaxf(m, s), scale = exp2f(m - m2), w = exp2f(s - m2 + Weight<T>::LIFT);
            l = l * scale + w;
            m = m2;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int d = lane + 32 * c;
                if (d < p.head_dim) o[c] = o[c] * scale + w * to_f(v[d]);
            }
        }
    }
};

// A unit is (key head, sequence, ROWS query rows) and is as long as it has tiles of KEYS keys (at
// least 1). All units lie end to end, key head by key head; CTA c takes the c-th of `ctas` equal
// stretches. A stretch that ends inside a unit cuts it (unless a piece would be below MIN_PIECE
// tiles): each piece leaves its rows' partial results, and paged_combine_units_kernel adds them in
// order. Whole units on whole SMs would leave the last round part empty: 256 equal units on 148 SMs
// take two rounds, the second 73% full, and sequences of mixed lengths do worse.
constexpr int MIN_PIECE = 2;

struct Item {
    int rows, row0;     // query rows of the sequence; first of the unit's
    Sequence seq;
    int b, h;
    int lo, hi, tiles;  // keys [lo, hi) of this piece in `tiles` tiles
    int first;          // first key that any row of the unit sees
    int slot;           // where partial results go: -1 (the whole unit), 0 (a later piece), 1 (the first)
};

struct Walk {
    int h, b, t;  // unit
    int skip;     // its tiles before this CTA's stretch
    int left;     // tiles left of the stretch
    int share;    // tiles of a whole stretch
    int heads;    // end of the key heads of these stretches
    Sequence seq;  // sequence b
};

// Keys [lo, hi) that rows [ROWS t, ROWS t + ROWS) see, lo rounded down to a tile; the unit's length.
template <int ROWS, int KEYS>
__device__ __forceinline__ int unit_length(const AttendParams &p, const Sequence &s, int t, int &first, int &lo, int &hi) {
    const int rows = s.nq * p.group, row0 = t * ROWS;
    const RowRange a = row_range(p, s, row0), z = row_range(p, s, min(row0 + ROWS, rows) - 1);
    first = a.lo;
    lo = a.lo & ~(KEYS - 1);
    hi = max(z.hi, 0);
    return hi > lo ? (hi - lo + KEYS - 1) / KEYS : 1;
}

// The next piece of the stretch; false at its end. Advances the walk.
template <int ROWS, int KEYS>
__device__ __forceinline__ bool next_item(const AttendParams &p, Walk &k, Item &w) {
    while (k.left > 0 && k.h < k.heads) {
        w.seq = k.seq;
        w.rows = w.seq.nq * p.group;
        w.row0 = k.t * ROWS;
        if (w.row0 >= w.rows) {  // past the sequence: the next one
            k.t = 0;
            if (++k.b == p.batch.batch) {
                k.b = 0;
                ++k.h;
            }
            k.seq = load_sequence(p, k.b);
            continue;
        }
        int lo, hi;
        const int length = unit_length<ROWS, KEYS>(p, w.seq, k.t, w.first, lo, hi);
        int take = length - k.skip;
        if (take > k.left) {
            const int at = k.skip + k.left;  // where the stretch ends in the unit
            if (at < MIN_PIECE) break;
            if (length - at >= MIN_PIECE) take = k.left;
        }
        w.b = k.b;
        w.h = k.h;
        w.lo = lo + k.skip * KEYS;
        w.hi = min(hi, w.lo + take * KEYS);
        w.tiles = w.hi > w.lo ? (w.hi - w.lo + KEYS - 1) / KEYS : 0;
        w.slot = take == length ? -1 : k.skip > 0 ? 0 : 1;
        k.left -= take;
        if (k.skip + take == length) {
            k.skip = 0;
            ++k.t;
        } else {
            k.skip += take;
        }
        return true;
    }
    return false;
}

// Start of stretch c of `ctas` over the units of key heads [h0, h1) (one warp). Units are looked at
// 32 at a time; their lengths are the same for every key head.
template <int ROWS, int KEYS>
__device__ __forceinline__ Walk find_stretch(const AttendParams &p, int c, int ctas, int h0, int h1, int lane) {
    int most = 0;  // row tiles of the longest sequence
    for (int b = lane; b < p.batch.batch; b += 32) {
        const Sequence s = load_sequence(p, b);
        check_sequence(p, b);
        most = max(most, (s.nq * p.group + ROWS - 1) / ROWS);
    }
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    const unsigned count = (unsigned)p.batch.batch * (unsigned)most;
    auto length_of = [&](unsigned i) {
        if (i >= count) return 0;
        int first, lo, hi;
        const unsigned b = i / (unsigned)most;
        const Sequence s = load_sequence(p, (int)b);
        const int t = (int)(i - b * (unsigned)most);
        return t * ROWS < s.nq * p.group ? unit_length<ROWS, KEYS>(p, s, t, first, lo, hi) : 0;
    };
    // the lanes' lengths summed up to and including each; the first 32 units' are kept
    auto scan = [&](int v) {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (lane >= d) v += u;
        }
        return v;
    };
    const int mine0 = length_of(lane), upto0 = scan(mine0);
    long long head = __shfl_sync(0xFFFFFFFFu, upto0, 31);  // tiles of one key head
    for (unsigned i = 32; i < count; i += 32) head += __reduce_add_sync(0xFFFFFFFFu, length_of(i + lane));
    Walk k{h1, 0, 0, 0, 0, 0, h1, {0, 0, 0, 0}};
    const long long all = head * (h1 - h0);
    long long share, x0;
    if (all < 0x7FFFFFFF) {
        share = ((unsigned)all + ctas - 1) / (unsigned)ctas;
        share = max(share, (long long)MIN_PIECE);
        x0 = c * share;
        if (x0 >= all) return k;
        k.h = (int)((unsigned)x0 / (unsigned)head);
    } else {
        share = (all + ctas - 1) / ctas;
        x0 = c * share;
        if (x0 >= all) return k;
        k.h = (int)(x0 / head);
    }
    long long at = x0 - k.h * head;
    k.h += h0;
    for (unsigned i = 0; i < count; i += 32) {
        const int mine = i ? length_of(i + lane) : mine0, upto = i ? scan(mine) : upto0;
        const unsigned past = __ballot_sync(0xFFFFFFFFu, upto > at);
        if (past) {
            const int who = __ffs(past) - 1;
            const int length = __shfl_sync(0xFFFFFFFFu, mine, who);
            const int off = (int)at - (__shfl_sync(0xFFFFFFFFu, upto, who) - length);
            k.b = (int)((i + who) / (unsigned)most);
            k.t = (int)((i + who) % (unsigned)most);
            k.seq = load_sequence(p, k.b);
            k.left = k.share = (int)share;
            if (off < MIN_PIECE) {
                k.left += off;
            } else if (length - off < MIN_PIECE) {
                k.left -= length - off;
                ++k.t;
            } else {
                k.skip = off;
            }
            break;
        }
        at -= __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return k;
}

// What adding up the unit cut at the stretch's end (piece w, slot 1) needs: the later stretches that
// end in it are one share apart.
template <int ROWS, int KEYS>
__device__ __forceinline__ CutUnit cut_of(const AttendParams &p, const Walk &k, const Item &w) {
    int first, lo, hi;
    CutUnit cut{w.h, w.b, w.row0 / ROWS, 1};
    const int length = unit_length<ROWS, KEYS>(p, w.seq, cut.t, first, lo, hi);
    for (int at = w.tiles; length - at >= MIN_PIECE; at += k.share) ++cut.pieces;
    return cut;
}

// Adds up out of the rows of units that were cut, the pieces in order; `next` CTAs lie between a stretch and
// the one after it. Units of many rows are cut into few pieces: a warp per row. Units of few rows can
// be cut into many (a long context on all SMs): a block per row, its warps taking every fourth piece.
// The factors come first, their loads together: a loop that loaded each piece's maximum before its
// row took 26 us for 37 pieces.
template <typename T, int ROWS>
__global__ void __launch_bounds__(128) paged_combine_units_kernel(const __grid_constant__ AttendParams p, const int next) {
    constexpr int WARPS = ROWS > 64 ? 1 : 4;  // that share a row
    __shared__ float4 sum[WARPS][32];
    __shared__ float warp_l[WARPS];
    const int c = (int)blockIdx.x, lane = (int)(threadIdx.x & 31), warp = (int)(threadIdx.x >> 5);
    const int share = WARPS > 1 ? warp : 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const CutUnit cut = p.cut[c];
    if (cut.pieces < 2) return;
    const Sequence s = load_sequence(p, cut.b);
    const int rows = s.nq * p.group;
    const int r0 = WARPS > 1 ? (int)blockIdx.y : (int)blockIdx.y * 4 + warp, step = (int)gridDim.y * (4 / WARPS);
    for (int r = r0; r < ROWS; r += step) {
        const int row = cut.t * ROWS + r;
        if (row >= rows) break;
        auto at = [&](int i) { return ((long long)(c + i * next) * 2 + (i == 0 ? 1 : 0)) * ROWS + r; };
        float m = -INFINITY, l = 0.0f;
        for (int i = lane; i < cut.pieces; i += 32) m = fmaxf(m, p.part_ml[at(i)].x);
#pragma unroll
        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x));
        T *out = static_cast<T *>(p.out) + (long long)(s.start + row / p.group) * p.o_ts +
                 (long long)(cut.h * p.group + row % p.group) * p.o_hs;
        for (int d0 = 0; d0 < p.head_dim; d0 += 128) {
            const int d = d0 + lane * 4;
            const bool mine = d < p.head_dim;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            l = 0.0f;
            for (int i0 = 0; i0 < cut.pieces; i0 += 32 * WARPS) {
                // lane k holds the factor of this warp's k-th piece of the batch
                const int i = i0 + lane * WARPS + share;
                const float2 ml = i < cut.pieces ? p.part_ml[at(i)] : make_float2(0.0f, 0.0f);
                const float f = ml.y > 0.0f ? ex2(ml.x - m) : 0.0f;
                l += f * ml.y;
                const int count = min(32, (cut.pieces - i0 - share + WARPS - 1) / WARPS);
#pragma unroll 8
                for (int k = 0; k < count; ++k) {
                    const float g = __shfl_sync(0xFFFFFFFFu, f, k);
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (mine) v = *reinterpret_cast<const float4 *>(p.part + at(i0 + k * WARPS + share) * p.head_dim + d);
                    a.x += g * v.x;
                    a.y += g * v.y;
                    a.z += g * v.z;
                    a.w += g * v.w;
                }
            }
#pragma unroll
            for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
            if constexpr (WARPS > 1) {
                sum[warp][lane] = a;
                if (lane == 0) warp_l[warp] = l;
                __syncthreads();
                if (warp == 0) {
                    l = (warp_l[0] + warp_l[1]) + (warp_l[2] + warp_l[3]);
                    const float4 x = sum[1][lane], y = sum[2][lane], z = sum[3][lane];
                    a = make_float4((a.x + x.x) + (y.x + z.x), (a.y + x.y) + (y.y + z.y), (a.z + x.z) + (y.z + z.z),
                                    (a.w + x.w) + (y.w + z.w));
                }
                __syncthreads();
            }
            if (!mine || (WARPS > 1 && warp)) continue;
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            Pack<4, T> v;
            v.e[0] = from_f<T>(a.x * inv);
            v.e[1] = from_f<T>(a.y * inv);
            v.e[2] = from_f<T>(a.z * inv);
            v.e[3] = from_f<T>(a.w * inv);
            v.store(out + d);
        }
    }
}

}  // namespace paged
}  // namespace mgc
