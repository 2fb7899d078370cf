// Attention over quantised pages on warp-level matrix instructions: decoding and other calls with few query
// rows per key head, which the bytes of the cache bound.
//
// Codes go into the products as halves, which hold them exactly, and what a group's channels share comes after:
//   score:  q . k_j = sum_g scale_jg (q_g . code_jg) + offset_jg sum(q_g)
//   output: o_d     = sum_j (w_j scale_jg) code_jd + sum_j w_j offset_jg
// so a value costs its conversion and nothing else: no rounding of keys or values, fp32 queries and weights
// in two halves each (22 bits). With c = 2^(bits - 1), codes become halves
//  * exactly and centred, as 1024 + code (or 64 + code), less 1024 + c: values, whose weights are rounded, so that
//    the error goes with |code - c| and not with the code (0.04 % of the output over 131071 keys, 0.02 % centred),
//    and the keys of fp32 calls;
//  * by masks alone: 16-bit calls' keys. Bits 4 to 7 of a half that is otherwise zero are the subnormal
//    code * 2^-20, a byte is code * 2^-24, and the power of two comes off with the scales. A subnormal's products are
//    cut off at 2^-24 of what a normal operand would have given, 2^-18 of a 4-bit step times the largest query value.
//
// A CTA takes a unit of R = 8 NB query rows (row = token * group + head of the group) of one key head. Keys are
// the M = 16 side of m16n8k16 products and rows the N = 8 side: a key head's 4 to 8 query heads leave less of
// them empty than M = 16 rows would. Each of four warps takes 32 keys of every 128 with its own ring of
// stages (cp.async), maximum, sum and output, so warps meet only at the end of a piece.
//  * K: both operands may take the contraction's channels in any order, so lane (g, t) of a fragment takes
//    eight consecutive codes of key g's 32 (a 4- or 8-byte load) and Q's fragments follow that order.
//  * V: as V^T, 16 channels by 16 keys: lane (g, t) takes eight consecutive channels of two keys at a time and pairs
//    the two keys' codes by byte permutations (first(t) and second(t) below). Scores are made in
//    the same order of keys, and movmatrix turns weights [key][row] into the second product's operand.
//  * rows are padded so that both reads are free of bank conflicts (QuantConfig).
//  * scales and offsets: lane l reads key l's a step ahead and leaves them as floats in shared memory.
//  * weights are 2^(score - reference + 11): the reference moves when a score passes it by 4, and not otherwise, so
//    a step needs no maximum over the lanes; halves then hold them from 2^15 down (paged_attention_params.cuh).
//  * weights times scales are relative to S_g, a power of two at or above the group's scales so far: tokens'
//    scales may differ by far.
//  * query rows are scaled by a power of two into half's range (bf16 and fp32 have more exponent).
//
// 64 sequences up to 8192 positions, 32 heads over 8 of 128 in 4 bits (372 MB): 104 us and 8 for the second kernel, 3.6 TB/s,
// 55 % of the copy bandwidth; one of 131071 positions, one group a head (143 MB): 41 and 10 us. Issue and latency bound it: 800
// instructions for a warp's 32 keys (K 190, V 190, loads 85, the rest weights, scales and control), of which the ALU
// pipe's take half of all cycles; four warps a scheduler issue in 63 % of theirs. Measured on the way (the first
// case): three blocks an SM instead of four with 168 registers and 10 % fewer instructions 147 against 127 us; five with 96
// registers 167 against 119; each lane copying its own key's row instead of sharing addresses by shuffles 117
// against 113; a maximum over the lanes at every step 127 against 119 with Q in registers.
#pragma once

#include <type_traits>

#include "paged_mma.cuh"
#include "quantized_common.cuh"

namespace mgc {
namespace paged {

// ONE: a head is one group. Else every 64 channels are treated as a group of their own.
template <typename T_, int BITS_, int DP_, int NB_, bool ONE_> struct QuantConfig {
    using T = T_;
    static constexpr int BITS = BITS_, DP = DP_, NB = NB_;
    static constexpr bool ONE = ONE_, F32 = sizeof(T) == 4;
    static constexpr int WARPS = 4, THREADS = 32 * WARPS;
    static constexpr int R = 8 * NB;             // query rows of a unit
    static constexpr int KW = 32, BN = KW * WARPS;  // keys of a warp's step, of a tile
    // Bytes and chunks of a row of codes, bytes between rows. A warp reads 16 bytes of each of a fragment's eight
    // rows (keys, 4 bits), 32 of its rows 0 to 3 and 4 to 7 (8 bits), and 32 of the four rows first(t) or second(t)
    // (values): 16 times an odd number lets eight rows' 16 bytes and four even or four odd rows' 32 bytes fall into
    // different banks, 32 times an odd number four rows' 32 bytes if the rows differ modulo 4.
    static constexpr int ROW = DP * BITS / 8, CPR = ROW / 16, PITCH = ROW + (BITS == 4 ? 16 : 32);
    static __device__ __forceinline__ int first(int t) { return BITS == 4 ? 2 * t : t; }
    static __device__ __forceinline__ int second(int t) { return BITS == 4 ? 2 * t + 1 : 4 + (t ^ 2); }
    static constexpr int SLABS = DP / 64, GS = ONE ? 1 : SLABS;  // groups that are told apart
    static constexpr int CODES = KW * PITCH, STAGE = 2 * CODES;
    static constexpr int STAGES = DP > 64 || BITS > 4 ? 2 : 3;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int PAIRS = KW * GS * 8;    // bytes of a step's scales and offsets of K or V
    static constexpr int ORED = DP + 4;
    static constexpr int RED = WARPS * R * (ORED + 2) * 4;
    static constexpr int Q_AT = RING + WARPS * 2 * PAIRS > RED ? RING + WARPS * 2 * PAIRS : RED;
    static constexpr int Q = NB * (DP / 32) * 32 * 16;  // bytes of Q's fragments (their upper halves)
    static constexpr int SMEM = Q_AT + Q * (F32 ? 2 : 1);
    // blocks of an SM, by shared memory and by registers (128 threads of 128, 168 or 255)
    static constexpr int BY_SMEM = 232448 / (SMEM + 1024 + 64);
    static constexpr int BY_REGS = (NB > 1 && DP > 64) || (F32 && DP > 128) ? 2 : DP > 128 || (F32 && DP * NB > 64) ? 3 : 4;
    static constexpr int RESIDENT = BY_SMEM < BY_REGS ? BY_SMEM : BY_REGS;
};

// a b with a zero accumulator.
__device__ __forceinline__ void mma16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t sub_half2(uint32_t a, uint32_t b) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&d);
}
// (x & mask) | bits
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
    return y;
}

// Eight codes of a row as four pairs of halves; channel(i, s) is the s-th of pair i. UNIT: the half of code
// MID + 1. EXACT: normal halves.
template <int BITS, bool EXACT> struct Key;
template <bool EXACT> struct Key<4, EXACT> {
    static constexpr float UNIT = EXACT ? 1.0f : 1.0f / 1048576.0f, MID = EXACT ? 8.0f : 0.0f;
    uint32_t w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = *reinterpret_cast<const uint32_t *>(p); }
    // a nibble in bits 0 to 3, 4 to 7 of both halves of x
    static __device__ __forceinline__ uint32_t low(uint32_t x) {
        return EXACT ? sub_half2(and_or(x, 0x000F000Fu, 0x64006400u), 0x64086408u) : x << 4 & 0x00F000F0u;
    }
    static __device__ __forceinline__ uint32_t high(uint32_t x) {
        return EXACT ? sub_half2(and_or(x, 0x00F000F0u, 0x54005400u), 0x54805480u) : x & 0x00F000F0u;
    }
    __device__ __forceinline__ void pairs(uint32_t (&h)[4]) const {
        h[0] = low(w);
        h[1] = high(w);
        h[2] = EXACT ? low(w >> 8) : high(w >> 4);
        h[3] = high(w >> 8);
    }
    static __device__ __forceinline__ constexpr int channel(int i, int second) { return i + 4 * second; }
    // codes 2 J and 2 J + 1 of rows a and b: (a's, b's) pairs
    template <int J> static __device__ __forceinline__ void two_rows(const Key &a, const Key &b, uint32_t &even, uint32_t &odd) {
        const uint32_t x = __byte_perm(a.w, b.w, J | J << 4 | (4 + J) << 8 | (4 + J) << 12);
        even = low(x);
        odd = high(x);
    }
};
template <bool EXACT> struct Key<8, EXACT> {
    static constexpr float UNIT = EXACT ? 1.0f : 1.0f / 16777216.0f, MID = EXACT ? 128.0f : 0.0f;
    uint2 w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = *reinterpret_cast<const uint2 *>(p); }
    // bytes 0 and 1, 2 and 3 of x
    static __device__ __forceinline__ uint32_t low(uint32_t x) {
        return EXACT ? sub_half2(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u) : __byte_perm(x, 0, 0x4140);
    }
    static __device__ __forceinline__ uint32_t high(uint32_t x) {
        return EXACT ? sub_half2(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u) : __byte_perm(x, 0, 0x4342);
    }
    __device__ __forceinline__ void pairs(uint32_t (&h)[4]) const {
        h[0] = low(w.x);
        h[1] = high(w.x);
        h[2] = low(w.y);
        h[3] = high(w.y);
    }
    static __device__ __forceinline__ constexpr int channel(int i, int second) { return 2 * i + second; }
    template <int J> static __device__ __forceinline__ void two_rows(const Key &a, const Key &b, uint32_t &even, uint32_t &odd) {
        constexpr int I = 2 * (J & 1);
        const uint32_t x = __byte_perm(J < 2 ? a.w.x : a.w.y, J < 2 ? b.w.x : b.w.y, I | (4 + I) << 4 | (I + 1) << 8 | (5 + I) << 12);
        even = low(x);
        odd = high(x);
    }
};

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
    int q_wide;             // rows of q allow 16-byte loads
    int pairs_wide;         // two groups, whose pairs allow 8-byte loads
    int slabs, group_of[4]; // of 64 channels; their groups
    uint32_t page_magic;    // j / page_size = j * page_magic >> page_shift for 0 <= j < 2^31
    int page_shift;
    // strides that fit 32 bits: of codes in bytes, of scales in pairs
    uint32_t code_page, code_token, pair_page, pair_token;
};

// What a CTA takes: one unit's keys; the part of them that its rank in a cluster names; an even share of all units'
// keys (paged_work.cuh).
enum QuantWork { WORK_UNIT, WORK_CLUSTER, WORK_EVEN };
template <typename C, int WORK>
__global__ void __launch_bounds__(C::THREADS, C::RESIDENT) quantized_attention_kernel(const __grid_constant__ QuantParams params) {
    using T = typename C::T;
    constexpr bool EVEN = WORK == WORK_EVEN;
    constexpr int BITS = C::BITS, DP = C::DP, NB = C::NB, R = C::R, BN = C::BN, KW = C::KW, PITCH = C::PITCH, CPR = C::CPR;
    constexpr int SLABS = C::SLABS, GS = C::GS, STAGES = C::STAGES;
    constexpr float LIFT = Weight<__half>::LAZY_LIFT, MOST = LIFT + Weight<__half>::LAZY, FRESH = 1e30f;
    using KCodes = Key<BITS, C::F32>;
    using VCodes = Key<BITS, true>;
    const QuantAttend &p = params.a;
    const Quantized &z = params.z;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t there[C::WARPS][STAGES];  // keys of a stage that were loaded
    __shared__ float row_scale[R], row_sum[R][GS];  // of Q's rows: what takes a score to base 2, the groups' sums
    __shared__ RowRange row_sees[R];
    uint4 *q_upper = reinterpret_cast<uint4 *>(smem + C::Q_AT) + (threadIdx.x & 31), *q_lower = q_upper + C::Q / 16;
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g4 = lane >> 2, t4 = lane & 3;
    const int key0 = g4 & 1 ? C::second(g4 >> 1) : C::first(g4 >> 1);  // row of fragment key g4 among its eight
    uint8_t *ring = smem + warp * STAGES * C::STAGE;
    float2 *kpair = reinterpret_cast<float2 *>(smem + C::RING) + warp * 2 * KW * GS, *vpair = kpair + KW * GS;
    const int row_bytes = p.head_dim * BITS / 8;

    // one piece: rows row0 .. of (sequence b, key head kh) over keys [k_lo, k_hi)
    auto piece = [&](int b, int kh, const Sequence &seq, int row0, int k_lo, int k_hi, int slot) {
        const int rows = seq.nq * p.group, tiles = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
        // this lane's part of a copied row: chunk lane % CPR of row lane / CPR of those copied at once
        constexpr int AT_ONCE = KW / CPR;
        const int part = lane % CPR, copied = max(0, min(16, row_bytes - part * 16));
        const uint8_t *kp = static_cast<const uint8_t *>(p.k_pages) + kh * p.head_stride + part * 16;
        const uint8_t *vp = static_cast<const uint8_t *>(p.v_pages) + kh * p.head_stride + part * 16;
        const __half2 *ksp = z.k_scales + kh * z.head_stride, *vsp = z.v_scales + kh * z.head_stride;
        // keys below first.lo no row sees; all rows see [last.lo, first.hi)
        const RowRange first = row_range(p, seq, row0), last = row_range(p, seq, min(row0 + R, rows) - 1);
        const int ps = p.batch.page_size;
        const int32_t *table = p.batch.table + (long long)b * p.batch.table_stride;

        // Lane l looks after key l of the warp's step: its page (-1: nothing to load) and row within the page,
        // looked up a step ahead of the loads.
        struct Place { int page, row; };
        bool missing = false;
        auto fetch = [&](int it) {
            const int j = k_lo + it * BN + warp * KW + lane;
            Place x{-1, 0};
            if (j >= k_hi || j < first.lo) return x;
            const int at = (int)((unsigned long long)(unsigned)j * params.page_magic >> params.page_shift);
            x.row = j - at * ps;
            if (at < p.batch.table_pages) x.page = __ldg(table + at);
            return x;
        };
        // pages out of range: nothing to load
        auto checked = [&](int it, Place x) {
            const int j = k_lo + it * BN + warp * KW + lane;
            if ((unsigned)x.page >= (unsigned)p.batch.pages) {
                missing = missing || (j < k_hi && j >= first.lo);
                x.page = -1;
            }
            return x;
        };
        const long long v_past_k = vp - kp;
        auto load_stage = [&](int it, Place x) {
            uint8_t *st = ring + (it % STAGES) * C::STAGE;
            const unsigned mask = __ballot_sync(0xFFFFFFFFu, x.page >= 0);
            if (lane == 0) there[warp][it % STAGES] = mask;
            const uint32_t dst = smem_u32(st + (lane / CPR) * PITCH + part * 16), in_page = (uint32_t)x.row * params.code_token;
#pragma unroll
            for (int i = 0; i < CPR; ++i) {
                const unsigned page = (unsigned)__shfl_sync(0xFFFFFFFFu, x.page, i * AT_ONCE + lane / CPR);
                const uint32_t row = __shfl_sync(0xFFFFFFFFu, in_page, i * AT_ONCE + lane / CPR);
                const int bytes = (int)page >= 0 ? copied : 0;
                // (a page that is not there: nothing is read)
                const uint8_t *src = kp + (unsigned long long)page * params.code_page + row;
                cp_async16(dst + i * AT_ONCE * PITCH, src, bytes);
                cp_async16(dst + i * AT_ONCE * PITCH + C::CODES, src + v_past_k, bytes);
            }
        };
        // key l's pairs of a step into registers
        uint32_t kraw[GS], vraw[GS];
        auto load_pairs = [&](Place x) {
            const unsigned long long o = (unsigned long long)(unsigned)x.page * params.pair_page + (uint32_t)x.row * params.pair_token;
            const unsigned int *k = reinterpret_cast<const unsigned int *>(ksp + o), *v = reinterpret_cast<const unsigned int *>(vsp + o);
#pragma unroll
            for (int s = 0; s < GS; ++s) kraw[s] = vraw[s] = 0u;
            if (x.page >= 0) {
                if (GS == 2 && params.pairs_wide) {
                    const uint2 a = __ldg(reinterpret_cast<const uint2 *>(k)), b = __ldg(reinterpret_cast<const uint2 *>(v));
                    kraw[0] = a.x;
                    kraw[GS - 1] = a.y;
                    vraw[0] = b.x;
                    vraw[GS - 1] = b.y;
                } else {
#pragma unroll
                    for (int s = 0; s < GS; ++s) {
                        if (s >= params.slabs) break;
                        kraw[s] = __ldg(k + params.group_of[s]);
                        vraw[s] = __ldg(v + params.group_of[s]);
                    }
                }
            }
        };

        // the first stages' loads, Q meanwhile
        Place at[STAGES];  // of steps it + 1, it + 2, ...
#pragma unroll
        for (int it = 0; it < STAGES; ++it) at[it] = fetch(it);
#pragma unroll
        for (int it = 0; it < STAGES - 1; ++it) {
            at[it] = checked(it, at[it]);
            if (it < tiles) load_stage(it, at[it]);
            cp_async_commit();
        }
        load_pairs(at[0]);
        // Fragments of Q (row 8 nb + g4, channels 32 i + 8 t4 .. + 7 in KCodes's order), times a power of two, left in
        // shared memory by warp nb: in registers they cost a fifth more instructions
        if (warp < NB) {
            const int nb = warp, row = row0 + 8 * nb + g4;
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
            // 2^up: the row's largest then in [2^8, 2^9), in fp32 in [2^13, 2^14) (its second halves keep their bits)
            const int e = (int)(__float_as_uint(top) >> 23);
            int up = e == 0 || e == 255 ? 0 : (C::F32 ? 13 : 8) + 127 - e;
            up = max(min(up, 126), -126);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
            float sum[GS];
#pragma unroll
            for (int x = 0; x < GS; ++x) sum[x] = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                uint32_t h[4], l[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float a = to_f(raw[i].e[KCodes::channel(k, 0)]) * f, c = to_f(raw[i].e[KCodes::channel(k, 1)]) * f;
                    h[k] = pack2<__half>(a, c);
                    const float2 hf = __half22float2(*reinterpret_cast<const __half2 *>(&h[k]));
                    l[k] = pack2<__half>(a - hf.x, c - hf.y);
                    sum[C::ONE ? 0 : i / 2] += a + c;
                }
                q_upper[(nb * (DP / 32) + i) * 32] = make_uint4(h[0], h[1], h[2], h[3]);
                if constexpr (C::F32) q_lower[(nb * (DP / 32) + i) * 32] = make_uint4(l[0], l[1], l[2], l[3]);
            }
#pragma unroll
            for (int x = 0; x < GS; ++x) {
                sum[x] += __shfl_xor_sync(0xFFFFFFFFu, sum[x], 1);
                sum[x] += __shfl_xor_sync(0xFFFFFFFFu, sum[x], 2);
                if (t4 == 0) row_sum[8 * nb + g4][x] = sum[x];
            }
            if (t4 == 0) {
                // (not 0, which times the -inf of hidden keys would be NaN)
                row_scale[8 * nb + g4] = fmaxf(p.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23), 1.2e-38f);
                row_sees[8 * nb + g4] = row_range(p, seq, row);
            }
        }
        __syncthreads();
        // what rows 2 t4 and 2 t4 + 1 need
        float rs[NB][2], qs[NB][2][GS];
        float o[SLABS][4][NB][4], off[NB][2][GS], ref[NB][2], l[NB][2], top_scale[GS];
#pragma unroll
        for (int x = 0; x < GS; ++x) top_scale[x] = 1.0f / 16777216.0f;  // the least scale that half has
#pragma unroll
        for (int x = 0; x < SLABS; ++x) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[x][j][nb][0] = o[x][j][nb][1] = o[x][j][nb][2] = o[x][j][nb][3] = 0.0f;
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                rs[nb][e] = row_scale[8 * nb + 2 * t4 + e];
                ref[nb][e] = FRESH;  // LIFT less the reference
                l[nb][e] = 0.0f;
#pragma unroll
                for (int x = 0; x < GS; ++x) {
                    qs[nb][e][x] = row_sum[8 * nb + 2 * t4 + e][x];
                    off[nb][e][x] = 0.0f;
                }
            }
        }

        for (int it = 0; it < tiles; ++it) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            // (the slot's last readers were this warp's lanes, a step ago)
            // the page looked up in the last step is first looked at here
            at[STAGES - 1] = checked(it + STAGES - 1, at[STAGES - 1]);
            if (it + STAGES - 1 < tiles) load_stage(it + STAGES - 1, at[STAGES - 1]);
            cp_async_commit();
            const int j0 = k_lo + it * BN + warp * KW;
            const uint32_t loaded = there[warp][it % STAGES];
            const Place next = fetch(it + STAGES);
            // key l's scales: K's, and V's relative to S, a power of two at or above all so far (scales that are
            // not finite make their own NaN)
            bool odd = false;
#pragma unroll
            for (int x = 0; x < GS; ++x) {
                float2 k = __half22float2(*reinterpret_cast<const __half2 *>(&kraw[x]));
                float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&vraw[x]));
                odd = odd || fmaf(v.x, 0.0f, v.y * 0.0f) != 0.0f;
                const float mine = fabsf(v.x) < INFINITY ? fabsf(v.x) : 0.0f;
                if (__any_sync(0xFFFFFFFFu, mine > top_scale[x])) {
                    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(mine));
                    const float now = __uint_as_float((most + 0x7FFFFFu) & 0xFF800000u), ratio = top_scale[x] / now;
                    top_scale[x] = now;
#pragma unroll
                    for (int y = C::ONE ? 0 : x; y < (C::ONE ? SLABS : x + 1); ++y) {
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
                k.y = fmaf(KCodes::MID, k.x, k.y);
                k.x *= 1.0f / KCodes::UNIT;
                v.y = fmaf(VCodes::MID, v.x, v.y);
                v.x *= __uint_as_float((254u << 23) - __float_as_uint(top_scale[x]));  // 1 / S, S from 2^-24 to 2^16
                kpair[lane * GS + x] = k;
                vpair[lane * GS + x] = v;
            }
            // the next step's, and the place of the one after the stages
            load_pairs(at[1]);
#pragma unroll
            for (int x = 0; x + 1 < STAGES; ++x) at[x] = at[x + 1];
            at[STAGES - 1] = next;
            __syncwarp();
            if (j0 >= k_hi) continue;
            const uint8_t *st = ring + (it % STAGES) * C::STAGE;
            const int k_at = key0 * PITCH + t4 * BITS;

            // ---- scores ----
            float s[2][NB][4], acc[2][NB][4];
            // (channels past the head width: whatever is there is finite and the query has zeros)
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                uint4 qh[NB], ql[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    qh[nb] = q_upper[(nb * (DP / 32) + i) * 32];
                    if constexpr (C::F32) ql[nb] = q_lower[(nb * (DP / 32) + i) * 32];
                }
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    KCodes a, c;  // channels 32 i + 8 t4: BITS bytes a lane
                    a.load(st + k_at + 16 * mt * PITCH + i * 4 * BITS);
                    c.load(st + k_at + (16 * mt + 8) * PITCH + i * 4 * BITS);
                    uint32_t ha[4], hc[4];
                    a.pairs(ha);
                    c.pairs(hc);
                    const uint32_t a0[4] = {ha[0], hc[0], ha[1], hc[1]}, a1[4] = {ha[2], hc[2], ha[3], hc[3]};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        // (the first of a group; fp32 calls add up every 64 channels, as the instruction truncates its sums)
                        if (i == 0 || (!(i & 1) && (!C::ONE || C::F32))) mma16_first(acc[mt][nb], a0, qh[nb].x, qh[nb].y);
                        else mma16<__half>(acc[mt][nb], a0, qh[nb].x, qh[nb].y);
                        mma16<__half>(acc[mt][nb], a1, qh[nb].z, qh[nb].w);
                        if constexpr (C::F32) {
                            mma16<__half>(acc[mt][nb], a0, ql[nb].x, ql[nb].y);
                            mma16<__half>(acc[mt][nb], a1, ql[nb].z, ql[nb].w);
                        }
                    }
                }
                const bool ends = i + 1 == DP / 32 || (!C::ONE && (i & 1));
                if (ends || (C::F32 && (i & 1))) {
                    const int x = C::ONE ? 0 : i / 2;
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        const float2 pa = kpair[(16 * mt + key0) * GS + x], pb = kpair[(16 * mt + key0 + 8) * GS + x];
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 &pair = e < 2 ? pa : pb;
                                if (i == (C::ONE && !C::F32 ? DP / 32 - 1 : 1)) s[mt][nb][e] = pair.x * acc[mt][nb][e];
                                else s[mt][nb][e] = fmaf(pair.x, acc[mt][nb][e], s[mt][nb][e]);
                                if (ends) s[mt][nb][e] = fmaf(pair.y, qs[nb][e & 1][x], s[mt][nb][e]);
                            }
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
                            const RowRange see = row_sees[8 * nb + 2 * t4 + (e & 1)];
                            if (j < see.lo || j >= see.hi || !(loaded >> r & 1)) {
                                hidden |= 1u << (8 * nb + 4 * mt + e);
                                s[mt][nb][e] = -INFINITY;
                            }
                        }
                    }
                }
            }
            // exponents; a row whose reference they pass by more than LAZY, or that has none yet
            float e_[2][NB][4];
            bool passed = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        e_[mt][nb][e] = fmaf(s[mt][nb][e], rs[nb][e], ref[nb][e]);
                        e_[mt][nb][e + 2] = fmaf(s[mt][nb][e + 2], rs[nb][e], ref[nb][e]);
                    }
                    passed = passed || fmaxf(fmaxf(e_[0][nb][e], e_[0][nb][e + 2]), fmaxf(e_[1][nb][e], e_[1][nb][e + 2])) > MOST;
                }
            }
            if (__any_sync(0xFFFFFFFFu, passed)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float fall[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(fmaxf(s[0][nb][e], s[0][nb][e + 2]), fmaxf(s[1][nb][e], s[1][nb][e + 2]));
                        x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 16));
                        fall[e] = 1.0f;
                        // (products rounded on their own: scores past 2^24 would leave the fused one's rest as an exponent)
                        const float top = __fmul_rn(x, rs[nb][e]);
                        if (x > -INFINITY && top + ref[nb][e] > MOST) {
                            const float now = LIFT - top;
                            if (ref[nb][e] != FRESH) fall[e] = ex2(now - ref[nb][e]);
                            ref[nb][e] = now;
                        }
                        l[nb][e] *= fall[e];
#pragma unroll
                        for (int y = 0; y < GS; ++y) off[nb][e][y] *= fall[e];
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt) {
                            e_[mt][nb][e] = __fmul_rn(s[mt][nb][e], rs[nb][e]) + ref[nb][e];
                            e_[mt][nb][e + 2] = __fmul_rn(s[mt][nb][e + 2], rs[nb][e]) + ref[nb][e];
                        }
                    }
#pragma unroll
                    for (int x = 0; x < SLABS; ++x) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            o[x][j][nb][0] *= fall[0];
                            o[x][j][nb][1] *= fall[1];
                            o[x][j][nb][2] *= fall[0];
                            o[x][j][nb][3] *= fall[1];
                        }
                    }
                }
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[mt][nb][e] = ex2(e_[mt][nb][e]);
                        l[nb][e & 1] += s[mt][nb][e];
                    }
                }
            }
            // a scale that is not finite, of a key that some row does not see: 0 times it is left out
            const bool careful = __any_sync(0xFFFFFFFFu, odd) && !whole;
            // ---- values ----
            // CAREFUL: hidden weights leave out what they would be multiplied by
            auto values = [&](auto careful_) {
                constexpr bool CAREFUL = decltype(careful_)::value;
                uint32_t bh[2][NB][2], bl[C::F32 ? 2 : 1][NB][2];
#pragma unroll
                for (int x = 0; x < SLABS; ++x) {
                    if (x == 0 || !C::ONE) {  // a group's weights
                        const int y = C::ONE ? 0 : x;
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt) {
                            const float2 pa = vpair[(16 * mt + key0) * GS + y], pb = vpair[(16 * mt + key0 + 8) * GS + y];
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                const float (&u)[4] = s[mt][nb];
                                float w[4] = {u[0] * pa.x, u[1] * pa.x, u[2] * pb.x, u[3] * pb.x};
                                if constexpr (CAREFUL) {
                                    const uint32_t hide = hidden >> (8 * nb + 4 * mt);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        w[e] = hide >> e & 1 ? 0.0f : w[e];
                                        off[nb][e & 1][y] += hide >> e & 1 ? 0.0f : u[e] * (e < 2 ? pa.y : pb.y);
                                    }
                                } else {
                                    off[nb][0][y] = fmaf(u[0], pa.y, fmaf(u[2], pb.y, off[nb][0][y]));
                                    off[nb][1][y] = fmaf(u[1], pa.y, fmaf(u[3], pb.y, off[nb][1][y]));
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
                        // eight channels from 64 x + 8 g4 on of four keys: BITS bytes a lane
                        VCodes key[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            key[k].load(st + C::CODES + (k & 1 ? C::second(t4) : C::first(t4)) * PITCH + g4 * BITS + (16 * mt + 8 * (k >> 1)) * PITCH + x * 8 * BITS);
                        auto tile = [&](auto index) {
                            constexpr int J = decltype(index)::value;
                            uint32_t a[4];
                            VCodes::template two_rows<J>(key[0], key[1], a[0], a[1]);
                            VCodes::template two_rows<J>(key[2], key[3], a[2], a[3]);
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
            };
            if (careful) values(std::true_type());
            else values(std::false_type());
        }
        if (missing && p.batch.status) *p.batch.status = MGC_CUDA_GATHER_OOB;
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
                for (int x = 0; x < GS; ++x) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) off[nb][e][x] += __shfl_xor_sync(0xFFFFFFFFu, off[nb][e][x], d);
                }
#pragma unroll
                for (int x = 0; x < SLABS; ++x) {
                    const float add = off[nb][e][C::ONE ? 0 : x], up = top_scale[C::ONE ? 0 : x] / VCodes::UNIT;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<float2 *>(red + r * C::ORED + 64 * x + 8 * g4 + 2 * j) =
                            make_float2(fmaf(up, o[x][j][nb][e], add), fmaf(up, o[x][j][nb][2 + e], add));
                }
                if (g4 == 0) {
                    sm[r] = ref[nb][e] == FRESH ? -INFINITY : LIFT - ref[nb][e];
                    sl[r] = l[nb][e];
                }
            }
        }
        __syncthreads();
        const int quads = p.head_dim / 4, live = min(R, rows - row0);
        auto warps_sum = [&](int r, int c, float &top, float &sum) {
            top = sm[r];
            sum = 0.0f;
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
            return a;
        };
        auto put = [&](int r, int c, float4 a, float sum) {
            const float inv = sum > 0.0f ? 1.0f / sum : sum != sum ? sum : 0.0f;
            const int row = row0 + r;
            T *out = static_cast<T *>(p.out) + (long long)(seq.start + row / p.group) * p.o_ts +
                     (long long)(kh * p.group + row % p.group) * p.o_hs + c * 4;
            out[0] = from_f<T>(a.x * inv);
            out[1] = from_f<T>(a.y * inv);
            out[2] = from_f<T>(a.z * inv);
            out[3] = from_f<T>(a.w * inv);
        };
        if constexpr (WORK != WORK_CLUSTER) {
            for (int x = tid; x < live * quads; x += C::THREADS) {
                const int r = x / quads, c = x - r * quads;
                float top, sum;
                const float4 a = warps_sum(r, c, top, sum);
                if (!EVEN || slot < 0) {
                    put(r, c, a, sum);
                } else {
                    const long long at = ((long long)blockIdx.x * 2 + slot) * R + r;
                    *reinterpret_cast<float4 *>(p.part + at * p.head_dim + c * 4) = a;
                    if (c == 0) p.part_ml[at] = make_float2(top, sum);
                }
            }
            __syncthreads();
        } else {
            // this CTA's sum over its first warp's rows (each four read and written by one thread), then the cluster's
            float own_top = -INFINITY, own_sum = 0.0f;  // of row tid
            if (tid < live) warps_sum(tid, 0, own_top, own_sum);
            for (int x = tid; x < live * quads; x += C::THREADS) {
                const int r = x / quads, c = x - r * quads;
                float top, sum;
                const float4 a = warps_sum(r, c, top, sum);
                *reinterpret_cast<float4 *>(red + r * C::ORED + c * 4) = a;
            }
            __syncthreads();
            if (tid < live) {
                sm[tid] = own_top;
                sl[tid] = own_sum;
            }
            cluster_barrier();
            const uint32_t a_red = smem_u32(red), a_m = smem_u32(sm), a_l = smem_u32(sl);
            for (int x = (int)blockIdx.y * C::THREADS + tid; x < live * quads; x += p.splits * C::THREADS) {
                const int r = x / quads, c = x - r * quads;
                float mk[MAX_CLUSTER], top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) mk[k] = k < p.splits ? ld_cluster(a_m + r * 4, k) : -INFINITY;
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) top = fmaxf(top, mk[k]);
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) {
                    if (k >= p.splits) break;
                    const float f = top == -INFINITY ? 0.0f : ex2(mk[k] - top);
                    const float4 v = ld_cluster4(a_red + (r * C::ORED + c * 4) * 4, k);
                    sum += f * ld_cluster(a_l + r * 4, k);
                    a.x += f * v.x;
                    a.y += f * v.y;
                    a.z += f * v.z;
                    a.w += f * v.w;
                }
                put(r, c, a, sum);
            }
            cluster_barrier();  // every partial read before the next tile or the exit reuses it
        }
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
        zero_outside_rows<T>(p, (int)(blockIdx.y * gridDim.x + blockIdx.x), (int)(gridDim.x * gridDim.y), warp, C::WARPS, lane);
        for (int tile = tile0; tile * R < seq.nq * p.group; tile += p.row_tiles) {
            int first, lo, hi;
            const int length = unit_length<R, BN>(p, seq, tile, first, lo, hi);
            // this CTA's part of the tiles that some row of the unit sees
            const int per = WORK == WORK_CLUSTER ? (length + p.splits - 1) / p.splits * BN : length * BN;
            const int k_lo = lo + (WORK == WORK_CLUSTER ? (int)blockIdx.y * per : 0);
            piece(b, kh, seq, tile * R, k_lo, min(hi, k_lo + per), -1);
        }
    }
}

}  // namespace paged
}  // namespace mgc
