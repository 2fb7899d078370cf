// Attention over quantised pages on warp-level matrix instructions: decoding and other calls with few query
// rows per key head, which the bytes of the cache bound.
//
// Codes go into the products as halves, which hold them exactly, and what a group's channels share comes after:
//   score:  q . k_j = sum_g scale_jg (q_g . (code_jg - c)) + (offset_jg + c scale_jg) sum(q_g)
//   output: o_d     = sum_j (w_j scale_jg) (code_jd - c) + sum_j w_j (offset_jg + c scale_jg),  c = 2^(bits - 1)
// so a value costs its conversion and nothing else: no rounding of keys or values, fp32 queries and weights
// in two halves each (22 bits).
//
// A CTA takes a unit of R = 8 NB query rows (row = token * group + head of the group) of one key head. Keys are
// the M = 16 side of m16n8k16 products and rows the N = 8 side: a key head's 4 to 8 query heads leave less of
// them empty than M = 16 rows would. Each of four warps takes 32 keys of every 128 with its own ring of
// stages (cp.async), maximum, sum and output, so warps meet only at the end of a piece.
//  * K: both operands may take the contraction's channels in any order, so lane (g, t) of a fragment takes
//    eight consecutive codes of key g's 32 (a 4- or 8-byte load) and Q's fragments follow that order.
//  * V: as V^T, 16 channels by 16 keys: lane (g, t) takes eight consecutive channels of keys t and t + 4 and pairs
//    the two keys' codes by byte permutations. Key i of a fragment is therefore position (i / 2) + 4 (i % 2)
//    of its eight; scores are made in the same order, and movmatrix turns weights [key][row] into the second
//    product's operand.
//  * 16-byte chunks of a row are permuted by the row's number so that both reads are free of bank conflicts.
//  * weights times scales are halves 2^14 times as large (paged_attention_params.cuh's reasons), relative to
//    S_g, a power of two at or above the group's scales so far: tokens' scales may differ by far.
//  * query rows are scaled by a power of two into half's range (bf16 and fp32 have more exponent).
#pragma once

#include <type_traits>

#include "paged_mma.cuh"
#include "quantized_common.cuh"

namespace mgc {
namespace paged {

template <typename T, int BITS, int DP, int NB> struct QuantConfig {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int WARPS = 4, THREADS = 32 * WARPS;
    static constexpr int R = 8 * NB;             // query rows of a unit
    static constexpr int KW = 32, BN = KW * WARPS;  // keys of a warp's step, of a tile
    static constexpr int ROW = DP * BITS / 8, CPR = ROW / 16;  // bytes and chunks of a row of codes
    static constexpr int SLABS = DP / 64;        // most groups, too
    static constexpr int CODES = KW * ROW, PAIRS = KW * SLABS * 4;
    static constexpr int STAGE = 2 * (CODES + PAIRS);
    static constexpr int STAGES = STAGE > 8192 ? 2 : 3;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int ORED = DP + 4;
    static constexpr int RED = WARPS * R * (ORED + 2) * 4;
    static constexpr int SMEM = RING > RED ? RING : RED;
    // blocks of an SM, by shared memory and by registers (128 threads of 128, 168 or 255)
    static constexpr int BY_SMEM = 232448 / (SMEM + 1024 + 64);
    static constexpr int BY_REGS = (NB > 1 && DP > 64) || (F32 && DP > 128) ? 2 : DP > 128 || (F32 && DP * NB > 64) ? 3 : 4;
    static constexpr int RESIDENT = BY_SMEM < BY_REGS ? BY_SMEM : BY_REGS;
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int BYTES> __device__ __forceinline__ void cp_async_small(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t sub_half2(uint32_t a, uint32_t b) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&d);
}
// (x & mask) | bits: a code put into the mantissa of 1024 (its low bits) or 64 (bits 4 to 7 of the half).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
    return y;
}
constexpr uint32_t HALF2_1024 = 0x64006400u, HALF2_64 = 0x54005400u;
constexpr uint32_t HALF2_1032 = 0x64086408u, HALF2_72 = 0x54805480u, HALF2_1152 = 0x64806480u;

// Eight codes of a key, less c, as four pairs; channel(i, s) is the s-th of pair i.
template <int BITS> struct Key;
template <> struct Key<4> {
    uint32_t w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = *reinterpret_cast<const uint32_t *>(p); }
    __device__ __forceinline__ void pairs(uint32_t (&h)[4]) const {
        h[0] = sub_half2(and_or(w, 0x000F000Fu, HALF2_1024), HALF2_1032);
        h[1] = sub_half2(and_or(w, 0x00F000F0u, HALF2_64), HALF2_72);
        h[2] = sub_half2(and_or(w >> 8, 0x000F000Fu, HALF2_1024), HALF2_1032);
        h[3] = sub_half2(and_or(w >> 8, 0x00F000F0u, HALF2_64), HALF2_72);
    }
    static __device__ __forceinline__ constexpr int channel(int i, int second) { return i + 4 * second; }
};
template <> struct Key<8> {
    uint2 w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void pairs(uint32_t (&h)[4]) const {
        h[0] = sub_half2(__byte_perm(w.x, 0x64646464u, 0x4140), HALF2_1152);
        h[1] = sub_half2(__byte_perm(w.x, 0x64646464u, 0x4342), HALF2_1152);
        h[2] = sub_half2(__byte_perm(w.y, 0x64646464u, 0x4140), HALF2_1152);
        h[3] = sub_half2(__byte_perm(w.y, 0x64646464u, 0x4342), HALF2_1152);
    }
    static __device__ __forceinline__ constexpr int channel(int i, int second) { return 2 * i + second; }
};
// Codes 2 j and 2 j + 1 of two keys a and b, less c: (a's, b's) pairs.
template <int J> __device__ __forceinline__ void two_keys(const Key<4> &a, const Key<4> &b, uint32_t &even, uint32_t &odd) {
    const uint32_t x = __byte_perm(a.w, b.w, J | J << 4 | (4 + J) << 8 | (4 + J) << 12);
    even = sub_half2(and_or(x, 0x000F000Fu, HALF2_1024), HALF2_1032);
    odd = sub_half2(and_or(x, 0x00F000F0u, HALF2_64), HALF2_72);
}
template <int J> __device__ __forceinline__ void two_keys(const Key<8> &a, const Key<8> &b, uint32_t &even, uint32_t &odd) {
    constexpr int I = 2 * (J & 1);
    const uint32_t x = __byte_perm(J < 2 ? a.w.x : a.w.y, J < 2 ? b.w.x : b.w.y, I | (4 + I) << 4 | (I + 1) << 8 | (5 + I) << 12);
    even = sub_half2(__byte_perm(x, 0x64646464u, 0x4140), HALF2_1152);
    odd = sub_half2(__byte_perm(x, 0x64646464u, 0x4342), HALF2_1152);
}

// What row r (0..7 of eight) exclusive-ors its chunks' numbers with. A warp reads one chunk of eight rows
// (keys, 4 bits), two adjacent chunks of rows {0, 4, 1, 5} or {2, 6, 3, 7} (8 bits) and of rows 0..3 or 4..7
// (values): in each the chunks land in different banks.
template <int ROW> __device__ __forceinline__ int swizzle(int r) {
    if constexpr (ROW == 32) return r >> 2 & 1;
    else if constexpr (ROW == 64) return ((r >> 1 ^ r >> 2) & 1) << 1 | (r >> 2 & 1);
    else return ((r & 3) ^ (r >> 2 & 1) << 1) << 1 | (r >> 2 & 1);
}

// Zeros in the rows of out that no sequence has, whatever their alignment (zero_outside's work).
template <typename T> __device__ __forceinline__ void zero_outside_rows(const AttendParams &p, int t0, int t_step, int h0, int h_step, int lane) {
    const int first = min(max(__ldg(p.batch.q_starts), 0), p.tokens);
    const int last = min(max(__ldg(p.batch.q_starts + p.batch.batch), first), p.tokens);
    for (long long i = t0; i < first + p.tokens - last; i += t_step) {
        T *row = static_cast<T *>(p.out) + (i < first ? i : i - first + last) * p.o_ts;
        for (int h = h0; h < p.q_heads; h += h_step)
            for (int d = lane; d < p.head_dim; d += 32) row[h * p.o_hs + d] = from_f<T>(0.0f);
    }
}

// A call in two parts: these kernels leave sequences with more than `rows_left` query rows a key head to the
// other (quantized_attention.cuh), if they have at most `kv_left` positions. kv_left 0: all are taken here.
struct QuantAttend : AttendParams {
    int rows_left, kv_left;
};
__device__ __forceinline__ bool left_out(const QuantAttend &p, const Sequence &s) {
    return s.n <= p.kv_left && s.nq * p.group > p.rows_left;
}
__device__ __forceinline__ Sequence load_sequence(const QuantAttend &p, int b) {
    Sequence s = load_sequence(static_cast<const AttendParams &>(p), b);
    if (p.kv_left && left_out(p, s)) s.nq = 0;
    return s;
}

struct QuantParams {
    QuantAttend a;
    Quantized z;
    int pair_bytes;  // pairs of a row copied at once: 4, or all of them (8, 16)
    int q_wide;      // rows of q allow 16-byte loads
};

// EVEN: the CTA takes an even share of all units' keys (paged_work.cuh); else one unit's keys.
template <typename T, int BITS, int DP, int NB, bool EVEN>
__global__ void __launch_bounds__(QuantConfig<T, BITS, DP, NB>::THREADS, QuantConfig<T, BITS, DP, NB>::RESIDENT)
quantized_attention_kernel(const __grid_constant__ QuantParams params) {
    using C = QuantConfig<T, BITS, DP, NB>;
    constexpr int R = C::R, BN = C::BN, KW = C::KW, ROW = C::ROW, CPR = C::CPR, SLABS = C::SLABS, STAGES = C::STAGES;
    constexpr float LIFT = Weight<__half>::LIFT;
    const QuantAttend &p = params.a;
    const Quantized &z = params.z;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t there[C::WARPS][STAGES];  // keys of a stage that were loaded
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g4 = lane >> 2, t4 = lane & 3;
    const int key0 = (g4 >> 1) + 4 * (g4 & 1);  // position of fragment key g4 within its eight
    uint8_t *ring = smem + warp * STAGES * C::STAGE;
    // the group of 64 channels from 64 x on, and whether it begins there
    int group_of[SLABS];
    bool begins[SLABS + 1];
#pragma unroll
    for (int x = 0; x < SLABS; ++x) {
        group_of[x] = x == 0 ? 0 : 64 * x / z.group;
        begins[x] = x == 0 || group_of[x] != group_of[x - 1];
    }
    begins[SLABS] = true;
    const int slabs32 = (p.head_dim + 31) / 32, slabs64 = (p.head_dim + 63) / 64, row_bytes = p.head_dim * BITS / 8;

    // one piece: rows row0 .. of (sequence b, key head kh) over keys [k_lo, k_hi)
    auto piece = [&](int b, int kh, const Sequence &seq, int row0, int k_lo, int k_hi, int slot) {
        const int rows = seq.nq * p.group, tiles = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
        const uint8_t *kp = static_cast<const uint8_t *>(p.k_pages) + kh * p.head_stride;
        const uint8_t *vp = static_cast<const uint8_t *>(p.v_pages) + kh * p.head_stride;
        const __half2 *ksp = z.k_scales + kh * z.head_stride, *vsp = z.v_scales + kh * z.head_stride;
        // keys below first.lo no row sees; all rows see [last.lo, first.hi)
        const RowRange first = row_range(p, seq, row0), last = row_range(p, seq, min(row0 + R, rows) - 1);
        const int ps = p.batch.page_size;

        auto fetch_page = [&](int it) {
            const int j = k_lo + it * BN + warp * KW + lane, at = j / ps;
            return j < k_hi && j >= first.lo && at < p.batch.table_pages
                       ? __ldg(p.batch.table + (long long)b * p.batch.table_stride + at) : -1;
        };
        auto load_stage = [&](int it, int page) {
            uint8_t *st = ring + (it % STAGES) * C::STAGE;
            const int j = k_lo + it * BN + warp * KW + lane;
            const bool in = j < k_hi && j >= first.lo, ok = in && page >= 0 && page < p.batch.pages;
            if (in && !ok && p.batch.status) *p.batch.status = MGC_CUDA_GATHER_OOB;
            const unsigned mask = __ballot_sync(0xFFFFFFFFu, ok);
            if (lane == 0) there[warp][it % STAGES] = mask;
            const int in_page = j % ps;
            const long long codes = ok ? page * p.page_stride + in_page * p.token_stride : -1;
            const long long pairs = ok ? page * z.page_stride + in_page * z.token_stride : 0;
#pragma unroll
            for (int i = 0; i < CPR; ++i) {
                const int r = i * (KW / CPR) + lane / CPR, c = lane % CPR;
                const long long o = __shfl_sync(0xFFFFFFFFu, codes, r);
                const long long at = o < 0 ? 0 : o + c * 16;
                const int bytes = o < 0 ? 0 : min(16, row_bytes - c * 16);
                if (c * 16 < row_bytes) {
                    const uint32_t dst = smem_u32(st + r * ROW + (c ^ swizzle<ROW>(r & 7)) * 16);
                    cp_async16(dst, kp + at, bytes);
                    cp_async16(dst + C::CODES, vp + at, bytes);
                }
            }
            const uint32_t dst = smem_u32(st + 2 * C::CODES + lane * SLABS * 4);
            if (SLABS >= 2 && params.pair_bytes == 8) {
                cp_async_small<8>(dst, ksp + pairs, ok ? 8 : 0);
                cp_async_small<8>(dst + C::PAIRS, vsp + pairs, ok ? 8 : 0);
            } else if (SLABS >= 4 && params.pair_bytes == 16) {
                cp_async_small<16>(dst, ksp + pairs, ok ? 16 : 0);
                cp_async_small<16>(dst + C::PAIRS, vsp + pairs, ok ? 16 : 0);
            } else {
#pragma unroll
                for (int g = 0; g < SLABS; ++g) {
                    if (g >= z.groups) break;
                    cp_async_small<4>(dst + 4 * g, ksp + pairs + g, ok ? 4 : 0);
                    cp_async_small<4>(dst + C::PAIRS + 4 * g, vsp + pairs + g, ok ? 4 : 0);
                }
            }
        };

        // the first stages' loads, Q meanwhile
        int page_next = -1;
        {
            int page[STAGES];
#pragma unroll
            for (int it = 0; it < STAGES; ++it) page[it] = fetch_page(it);
#pragma unroll
            for (int it = 0; it < STAGES - 1; ++it) {
                if (it < tiles) load_stage(it, page[it]);
                cp_async_commit();
            }
            page_next = page[STAGES - 1];
        }
        // fragments of Q (row 8 nb + g4, channels 32 i + 8 t4 .. + 7 in Key's order), times a power of two; what
        // rows 2 t4 and 2 t4 + 1 need: that power's inverse times the scale, the groups' sums
        uint32_t qh[DP / 32][NB][4], ql[C::F32 ? DP / 32 : 1][NB][4];
        float rs[NB][2], qs[NB][2][SLABS];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int row = row0 + 8 * nb + g4;
            const T *q = static_cast<const T *>(p.q) + (long long)(seq.start + row / p.group) * p.q_ts +
                         (long long)(kh * p.group + row % p.group) * p.q_hs;
            float top = 0.0f;
            Pack<8, T> raw[DP / 32];
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const int c = 32 * i + 8 * t4;
#pragma unroll
                for (int x = 0; x < 8; ++x) raw[i].e[x] = from_f<T>(0.0f);
                if (row < rows && c < p.head_dim) {
                    if (params.q_wide) {
                        raw[i].load(q + c);
                    } else {
#pragma unroll
                        for (int x = 0; x < 8; ++x) raw[i].e[x] = q[c + x];
                    }
                }
#pragma unroll
                for (int x = 0; x < 8; ++x) top = fmaxf(top, fabsf(to_f(raw[i].e[x])));
            }
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            // 2^up, the row's largest then in [1, 2), in fp32 in [2^13, 2^14): its lower halves keep their bits
            const int e = (int)(__float_as_uint(top) >> 23);
            int up = e == 0 || e == 255 ? 0 : (C::F32 ? 13 : 0) + 127 - e;
            up = max(min(up, 126), -126);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
            const float scale = p.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
            float sum[SLABS];
#pragma unroll
            for (int s = 0; s < SLABS; ++s) sum[s] = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                float part = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float a = to_f(raw[i].e[Key<BITS>::channel(k, 0)]) * f, c = to_f(raw[i].e[Key<BITS>::channel(k, 1)]) * f;
                    qh[i][nb][k] = pack2<__half>(a, c);
                    if constexpr (C::F32) {
                        const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&qh[i][nb][k]));
                        ql[i][nb][k] = pack2<__half>(a - h.x, c - h.y);
                    }
                    part += a + c;
                }
#pragma unroll
                for (int s = 0; s < SLABS; ++s) sum[s] += s == group_of[i / 2] ? part : 0.0f;
            }
            rs[nb][0] = __shfl_sync(0xFFFFFFFFu, scale, 8 * t4);
            rs[nb][1] = __shfl_sync(0xFFFFFFFFu, scale, 8 * t4 + 4);
#pragma unroll
            for (int s = 0; s < SLABS; ++s) {
                sum[s] += __shfl_xor_sync(0xFFFFFFFFu, sum[s], 1);
                sum[s] += __shfl_xor_sync(0xFFFFFFFFu, sum[s], 2);
                qs[nb][0][s] = __shfl_sync(0xFFFFFFFFu, sum[s], 8 * t4);
                qs[nb][1][s] = __shfl_sync(0xFFFFFFFFu, sum[s], 8 * t4 + 4);
            }
        }
        RowRange see[NB][2];
        float o[SLABS][4][NB][4], off[NB][2][SLABS], m[NB][2], l[NB][2], top_scale[SLABS];
#pragma unroll
        for (int s = 0; s < SLABS; ++s) {
            top_scale[s] = __uint_as_float((127u - 24) << 23);  // the least scale that half has
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[s][j][nb][0] = o[s][j][nb][1] = o[s][j][nb][2] = o[s][j][nb][3] = 0.0f;
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                see[nb][e] = row_range(p, seq, row0 + 8 * nb + 2 * t4 + e);
                m[nb][e] = -INFINITY;
                l[nb][e] = 0.0f;
#pragma unroll
                for (int s = 0; s < SLABS; ++s) off[nb][e][s] = 0.0f;
            }
        }

        for (int it = 0; it < tiles; ++it) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            // (the slot's last readers were this warp's lanes, a step ago)
            if (it + STAGES - 1 < tiles) load_stage(it + STAGES - 1, page_next);
            cp_async_commit();
            page_next = fetch_page(it + STAGES);
            const int j0 = k_lo + it * BN + warp * KW;
            if (j0 >= k_hi) continue;
            const uint8_t *st = ring + (it % STAGES) * C::STAGE;
            const uint32_t loaded = there[warp][it % STAGES];
            const __half2 *kpair = reinterpret_cast<const __half2 *>(st + 2 * C::CODES), *vpair = kpair + KW * SLABS;

            // ---- scores ----
            float s[2][NB][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int ra = 16 * mt + key0, rb = ra + 8;
                const uint8_t *rowa = st + ra * ROW, *rowb = st + rb * ROW;
                float acc[NB][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[nb][e] = s[mt][nb][e] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) {
                    if (i >= slabs32) break;
                    Key<BITS> a, c;
                    // chunk of channels 32 i + 8 t4: BITS bytes a lane, 4 BITS a quad
                    const int chunk = (i * 4 * BITS + t4 * BITS) / 16, in = (i * 4 * BITS + t4 * BITS) % 16;
                    a.load(rowa + (chunk ^ swizzle<ROW>(ra & 7)) * 16 + in);
                    c.load(rowb + (chunk ^ swizzle<ROW>(rb & 7)) * 16 + in);
                    uint32_t ha[4], hc[4];
                    a.pairs(ha);
                    c.pairs(hc);
                    const uint32_t a0[4] = {ha[0], hc[0], ha[1], hc[1]}, a1[4] = {ha[2], hc[2], ha[3], hc[3]};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        mma16<__half>(acc[nb], a0, qh[i][nb][0], qh[i][nb][1]);
                        mma16<__half>(acc[nb], a1, qh[i][nb][2], qh[i][nb][3]);
                        if constexpr (C::F32) {
                            mma16<__half>(acc[nb], a0, ql[i][nb][0], ql[i][nb][1]);
                            mma16<__half>(acc[nb], a1, ql[i][nb][2], ql[i][nb][3]);
                        }
                    }
                    // a group's end (fp32: every 64 channels, the instruction truncates its sums)
                    const bool ends = ((i & 1) && begins[i / 2 + 1]) || i + 1 == slabs32;
                    if (ends || (C::F32 && (i & 1))) {
                        const int gi = group_of[i / 2];
                        const float2 pa = __half22float2(kpair[ra * SLABS + gi]), pb = __half22float2(kpair[rb * SLABS + gi]);
                        const float oa = fmaf((float)(1 << (BITS - 1)), pa.x, pa.y), ob = fmaf((float)(1 << (BITS - 1)), pb.x, pb.y);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            float q0 = qs[nb][0][0], q1 = qs[nb][1][0];
#pragma unroll
                            for (int x = 1; x < SLABS; ++x) {
                                q0 = x == gi ? qs[nb][0][x] : q0;
                                q1 = x == gi ? qs[nb][1][x] : q1;
                            }
                            s[mt][nb][0] = fmaf(pa.x, acc[nb][0], s[mt][nb][0]);
                            s[mt][nb][1] = fmaf(pa.x, acc[nb][1], s[mt][nb][1]);
                            s[mt][nb][2] = fmaf(pb.x, acc[nb][2], s[mt][nb][2]);
                            s[mt][nb][3] = fmaf(pb.x, acc[nb][3], s[mt][nb][3]);
                            if (ends) {
                                s[mt][nb][0] = fmaf(oa, q0, s[mt][nb][0]);
                                s[mt][nb][1] = fmaf(oa, q1, s[mt][nb][1]);
                                s[mt][nb][2] = fmaf(ob, q0, s[mt][nb][2]);
                                s[mt][nb][3] = fmaf(ob, q1, s[mt][nb][3]);
                            }
                            acc[nb][0] = acc[nb][1] = acc[nb][2] = acc[nb][3] = 0.0f;
                        }
                    }
                }
            }
            // ---- weights ----
            // `whole`: every row sees every key of the step
            const bool whole = loaded == 0xFFFFFFFFu && j0 >= last.lo && j0 + KW <= first.hi;
            uint32_t hidden = 0;  // bits 8 nb + 4 mt + e
            if (!whole) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = 16 * mt + key0 + (e < 2 ? 0 : 8), j = j0 + r;
                            if (j < see[nb][e & 1].lo || j >= see[nb][e & 1].hi || !(loaded >> r & 1)) hidden |= 1u << (8 * nb + 4 * mt + e);
                        }
                    }
                }
            }
            bool moved = false;
            float fall[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = m[nb][e];
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                        for (int k = 0; k < 4; k += 2) {
                            s[mt][nb][e + k] *= rs[nb][e];
                            if (hidden >> (8 * nb + 4 * mt + e + k) & 1) s[mt][nb][e + k] = -INFINITY;
                            x = fmaxf(x, s[mt][nb][e + k]);
                        }
                    }
                    x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 16));
                    const float y = x == -INFINITY ? 0.0f : x;  // nothing seen yet: subtract 0
                    fall[nb][e] = ex2(m[nb][e] - y);
                    moved = moved || fall[nb][e] != 1.0f;
                    m[nb][e] = x;
                    float sum = 0.0f;
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                        for (int k = 0; k < 4; k += 2) {
                            s[mt][nb][e + k] = ex2(s[mt][nb][e + k] - y + LIFT);
                            sum += s[mt][nb][e + k];
                        }
                    }
                    l[nb][e] = fmaf(l[nb][e], fall[nb][e], sum);
                }
            }
            if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int x = 0; x < SLABS; ++x) {
                        off[nb][0][x] *= fall[nb][0];
                        off[nb][1][x] *= fall[nb][1];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            o[x][j][nb][0] *= fall[nb][0];
                            o[x][j][nb][1] *= fall[nb][1];
                            o[x][j][nb][2] *= fall[nb][0];
                            o[x][j][nb][3] *= fall[nb][1];
                        }
                    }
                }
            }
            // ---- values ----
            uint32_t bh[2][NB][2], bl[C::F32 ? 2 : 1][NB][2];
#pragma unroll
            for (int x = 0; x < SLABS; ++x) {
                if (x >= slabs64) break;
                const int gi = group_of[x];
                if (begins[x]) {  // a group begins: its weights
                    // the largest scale so far, as a power of two (scales that are not finite make their own NaN)
                    uint32_t mine = __float_as_uint(__low2float(vpair[lane * SLABS + gi])) & 0x7FFFFFFFu;
                    if (mine >= 0x7F800000u || !(loaded >> lane & 1)) mine = 0;
                    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, mine);
                    float up = 0.0f;  // the group's S
#pragma unroll
                    for (int y = 0; y < SLABS; ++y) up = y == gi ? top_scale[y] : up;
                    if (most > __float_as_uint(up)) {
                        const float now = __uint_as_float((most + 0x7FFFFFu) & 0xFF800000u), ratio = up / now;
                        up = now;
#pragma unroll
                        for (int y = 0; y < SLABS; ++y) {
                            if (y == gi) top_scale[y] = now;
                            if (group_of[y] != gi) continue;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e) o[y][j][nb][e] *= ratio;
                                }
                            }
                        }
                    }
                    // (S is a power of two from 2^-24 to 2^16)
                    const float inv = __uint_as_float((254u << 23) - __float_as_uint(up));
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        const float2 pa = __half22float2(vpair[(16 * mt + key0) * SLABS + gi]);
                        const float2 pb = __half22float2(vpair[(16 * mt + key0 + 8) * SLABS + gi]);
                        const float oa = fmaf((float)(1 << (BITS - 1)), pa.x, pa.y), ob = fmaf((float)(1 << (BITS - 1)), pb.x, pb.y);
                        const float fa = pa.x * inv, fb = pb.x * inv;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            float w[4], t[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                w[e] = s[mt][nb][e] * (e < 2 ? fa : fb);
                                t[e] = s[mt][nb][e] * (e < 2 ? oa : ob);
                                if (hidden >> (8 * nb + 4 * mt + e) & 1) w[e] = t[e] = 0.0f;  // 0 times what is not finite
                            }
#pragma unroll
                            for (int y = 0; y < SLABS; ++y) {
                                if (y == gi) {
                                    off[nb][0][y] += t[0] + t[2];
                                    off[nb][1][y] += t[1] + t[3];
                                }
                            }
                            const uint32_t h0 = pack2<__half>(w[0], w[1]), h1 = pack2<__half>(w[2], w[3]);
                            bh[mt][nb][0] = movmatrix(h0);
                            bh[mt][nb][1] = movmatrix(h1);
                            if constexpr (C::F32) {
                                const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0));
                                const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
                                bl[mt][nb][0] = movmatrix(pack2<__half>(w[0] - f0.x, w[1] - f0.y));
                                bl[mt][nb][1] = movmatrix(pack2<__half>(w[2] - f1.x, w[3] - f1.y));
                            }
                        }
                    }
                }
                float sum[C::F32 ? 4 : 1][NB][4];
                if constexpr (C::F32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) sum[j][nb][0] = sum[j][nb][1] = sum[j][nb][2] = sum[j][nb][3] = 0.0f;
                    }
                }
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    // eight channels from 64 x + 8 g4 on of keys t4, t4 + 4 and eight further: BITS bytes a lane
                    const int chunk = (x * 8 * BITS + g4 * BITS) / 16, in = (x * 8 * BITS + g4 * BITS) % 16;
                    Key<BITS> key[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = 16 * mt + t4 + 4 * k;
                        key[k].load(st + C::CODES + r * ROW + (chunk ^ swizzle<ROW>(r & 7)) * 16 + in);
                    }
                    auto tile = [&](auto index) {
                        constexpr int J = decltype(index)::value;
                        uint32_t a[4];
                        two_keys<J>(key[0], key[1], a[0], a[1]);
                        two_keys<J>(key[2], key[3], a[2], a[3]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            if constexpr (C::F32) {
                                mma16<__half>(sum[J][nb], a, bh[mt][nb][0], bh[mt][nb][1]);
                                mma16<__half>(sum[J][nb], a, bl[mt][nb][0], bl[mt][nb][1]);
                            } else {
                                mma16<__half>(o[x][J][nb], a, bh[mt][nb][0], bh[mt][nb][1]);
                            }
                        }
                    };
                    tile(std::integral_constant<int, 0>());
                    tile(std::integral_constant<int, 1>());
                    tile(std::integral_constant<int, 2>());
                    tile(std::integral_constant<int, 3>());
                }
                if constexpr (C::F32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[x][j][nb][e] += sum[j][nb][e];
                        }
                    }
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();

        // ---- the warps' partial results ----
        float *red = reinterpret_cast<float *>(smem), *sm = red + C::WARPS * R * C::ORED, *sl = sm + C::WARPS * R;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = warp * R + 8 * nb + 2 * t4 + e;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nb][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nb][e], d);
#pragma unroll
                for (int x = 0; x < SLABS; ++x) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) off[nb][e][x] += __shfl_xor_sync(0xFFFFFFFFu, off[nb][e][x], d);
                }
#pragma unroll
                for (int x = 0; x < SLABS; ++x) {
                    if (x >= slabs64) break;
                    const int gi = group_of[x];
                    float add = off[nb][e][0], up = top_scale[0];
#pragma unroll
                    for (int y = 1; y < SLABS; ++y) {
                        add = y == gi ? off[nb][e][y] : add;
                        up = y == gi ? top_scale[y] : up;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<float2 *>(red + r * C::ORED + 64 * x + 8 * g4 + 2 * j) =
                            make_float2(fmaf(up, o[x][j][nb][e], add), fmaf(up, o[x][j][nb][2 + e], add));
                }
                if (g4 == 0) {
                    sm[r] = m[nb][e];
                    sl[r] = l[nb][e];
                }
            }
        }
        __syncthreads();
        const int quads = p.head_dim / 4, live = min(R, rows - row0);
        for (int x = tid; x < live * quads; x += C::THREADS) {
            const int r = x / quads, c = x - r * quads;
            float top = sm[r], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < C::WARPS; ++w) top = fmaxf(top, sm[w * R + r]);
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < C::WARPS; ++w) {
                const float f = top == -INFINITY ? 0.0f : ex2(sm[w * R + r] - top);
                const float4 y = *reinterpret_cast<const float4 *>(red + (w * R + r) * C::ORED + c * 4);
                sum += f * sl[w * R + r];
                a.x += f * y.x;
                a.y += f * y.y;
                a.z += f * y.z;
                a.w += f * y.w;
            }
            if (!EVEN || slot < 0) {
                const float inv = sum > 0.0f ? 1.0f / sum : sum != sum ? sum : 0.0f;
                const int row = row0 + r;
                T *out = static_cast<T *>(p.out) + (long long)(seq.start + row / p.group) * p.o_ts +
                         (long long)(kh * p.group + row % p.group) * p.o_hs + c * 4;
                out[0] = from_f<T>(a.x * inv);
                out[1] = from_f<T>(a.y * inv);
                out[2] = from_f<T>(a.z * inv);
                out[3] = from_f<T>(a.w * inv);
            } else {
                const long long at = ((long long)blockIdx.x * 2 + slot) * R + r;
                *reinterpret_cast<float4 *>(p.part + at * p.head_dim + c * 4) = a;
                if (c == 0) p.part_ml[at] = make_float2(top, sum);
            }
        }
        __syncthreads();
    };

    if constexpr (EVEN) {
        __shared__ Walk stretch;
        const int heads = p.interleaved ? p.kv_heads : 1, h0 = (int)blockIdx.x % heads;
        if (warp == 0) {
            const Walk k = find_stretch<R, BN>(p, (int)blockIdx.x / heads, (int)gridDim.x / heads, h0,
                                               p.interleaved ? h0 + 1 : p.kv_heads, lane);
            if (lane == 0) stretch = k;
        } else {
            zero_outside_rows<T>(p, (int)blockIdx.x, (int)gridDim.x, warp - 1, C::WARPS - 1, lane);
        }
        __syncthreads();
        asm volatile("griddepcontrol.launch_dependents;");
        Walk walk = stretch;
        Item w;
        CutUnit cut{0, 0, 0, 0};
        while (next_item<R, BN>(p, walk, w)) {
            if (w.slot == 1) cut = cut_of<R, BN>(p, walk, w);
            piece(w.b, w.h, w.seq, w.row0, w.lo, w.hi, w.slot);
        }
        if (tid == 0) p.cut[blockIdx.x] = cut;
    } else {
        unsigned u = blockIdx.x;
        const int kh = (int)(u % (unsigned)p.kv_heads);
        u /= (unsigned)p.kv_heads;
        const int tile0 = p.row_tiles - 1 - (int)(u % (unsigned)p.row_tiles);
        const int b = (int)(u / (unsigned)p.row_tiles);
        const Sequence seq = load_sequence(p, b);
        if (tid == 0) check_sequence(p, b);
        zero_outside_rows<T>(p, (int)blockIdx.x, (int)gridDim.x, warp, C::WARPS, lane);
        for (int tile = tile0; tile * R < seq.nq * p.group; tile += p.row_tiles) {
            int first, lo, hi;
            unit_length<R, BN>(p, seq, tile, first, lo, hi);
            piece(b, kh, seq, tile * R, lo, hi, -1);
        }
    }
}

}  // namespace paged
}  // namespace mgc
