// Paged attention on tcgen05 for 16-bit types: chunks of many query rows.
//
// A CTA takes one (sequence, key head), 256 query rows (row = token * group + head of the group) as
// two tiles of 128, and one part of the rows' visible keys in tiles of 128. Per key tile and row
// tile: S = Q K^T (M = N = 128, K = D) into TMEM; a warpgroup, one row per thread, turns the row
// into weights 2^(scale s - m), writes them as 16-bit values over S; O += P V (M = 128, N = D,
// K = 128) with P read from TMEM. The two row tiles alternate: while one warpgroup exponentiates,
// the tensor core works for the other.
//
// * Q rows: a warp copies its 32 rows together into 128B-swizzled shared memory (any strides).
// * K and V tiles arrive by TMA from the pages, one box of min(page_size, 128) rows x 64 channels
//   per page and channel half, lane l of the loading warp issuing box l; a ring of stages holds
//   K and V tiles in the order K0 V0 K1 V1 ... K is a K-major operand, V (channels contiguous) an
//   MN-major one. Channels past the head width are the tensor map's zero fill.
// * The maximum is lazy: O (in TMEM) is rescaled only when a row's maximum has grown by more than
//   2^8 (f16: 2^4) since the last time; the weights then stay below 2^8 (f16: 2^15, Weight), far from
//   overflow, and the row sum carries the same reference, so the result is unchanged. With 128 channels a
//   rescale needs no wait: S of tile j is committed after P V of tile j - 1.
// * 64 channels leave TMEM for weights apart from the scores: the next tile's scores are made
//   while this one's weights are.
// * A page number out of range: its keys are not loaded, the products use whatever the stage held, and
//   at the unit's end its rows are computed again one per thread, without those keys (row_again).
// * A value that is not finite, at a key that some rows of a tile see and others do not: 0 * inf is NaN.
//   Rows that come out with NaN or infinities and do not see such a key of their tiles are computed
//   again too.
// * Rows of V that no row sees (past the last visible key, before the first) are zeroed in shared
//   memory before they are used: a page's unused rows hold anything, and 0 * NaN is NaN.
//
// Bound: the tensor core and the exponential unit about equally (2048 cycles each per key tile and
// pair of row tiles at 128 channels); measured 2930 cycles a pair, the rest being the chain scores ->
// weights -> products of each row tile. 2048 tokens x 32 heads of 128 over 16384 positions, bf16: 520 us
// in calls one after the other for seconds, 0.99 PFLOP/s, with the clock at the power cap. The softmax role
// of the 128-channel kernel spills (260 bytes written, 408 read a thread), the 64-channel one does not.
//
// Every mbarrier wait is bounded; on timeout the CTA sets the status word, drains its copies,
// frees its TMEM and returns.
#pragma once

#include <string.h>

#include <type_traits>

#include "paged_mma.cuh"
#include "umma_ptx.cuh"

namespace mgc {
namespace paged {

using umma::mbar_arrive;
using umma::mbar_expect_tx;
using umma::mbar_init;
using umma::mbar_wait;
using umma::smem_addr;
using umma::sw128_desc;
using umma::tc_fence_after;
using umma::tc_fence_before;

struct UmmaMaps {
    CUtensorMap k, v;  // {head_dim, page_size, kv_heads, pages}, boxes {64, box_rows, 1, 1}
    int box_rows;      // min(page_size, 128)
};

template <int DP> struct UmmaConfig {
    static constexpr int HALVES = DP / 64;            // 64-channel (128-byte) column blocks
    static constexpr uint32_t HALF = 128 * 128;       // bytes of a 128-row block
    static constexpr uint32_t TILE = HALVES * HALF;   // a Q, K or V tile
    static constexpr int STAGES = DP == 64 ? 8 : 5;
    static constexpr uint32_t SMEM = 1024 + 2 * TILE + STAGES * TILE;
    // two softmax warpgroups, then a warpgroup of the MMA warp (8), the load warp (9), one that zeroes
    // rows of V (10) and an idle one.
    // 384 threads launch with 168 registers each (64,512); the split keeps that sum:
    // 256 x 224 + 128 x 56
    static constexpr int THREADS = 384;
    static constexpr int SOFTMAX_REGS = 224, OTHER_REGS = 56;
    // TMEM columns: S0 S1 O0 O1, the weights of a tile over its scores; with 64 channels there is room
    // for weights of their own (S0 S1 P0 P1 O0 O1), so the next tile's scores are made while this
    // one's weights are
    static constexpr bool APART = DP == 64;
    static constexpr uint32_t S_COL = 0, P_COL = APART ? 256 : 0, P_STEP = APART ? 64 : 128, O_COL = APART ? 384 : 256;
};

// D = A B with A in TMEM (16-bit values packed in pairs along K) or shared memory.
// Executed by the lane whose `e` is set (elect_one); the whole warp calls.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void mma_f16_ss(uint32_t e, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(e) : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t e, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(e) : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t e, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
        ::"r"(smem_addr(bar)), "r"(e) : "memory");
}
// MN-major operand of 16-bit elements in 128B-swizzled rows of 64 (M / N) elements, consecutive K
// rows 128 bytes apart: 8-row groups 1024 bytes apart along K, 64-element blocks `lbo` bytes apart.
__device__ __forceinline__ uint64_t mn128_desc(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <typename T> __device__ __forceinline__ constexpr uint32_t idesc_f16(int n, int b_mn) {
    return (1u << 4) | ((sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) * ((1u << 7) | (1u << 10))) |
           ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
          "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
          "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait of a converged warp, polled by the elected lane only.
__device__ __forceinline__ bool poll(uint32_t e, uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %3, 0;\n\tsetp.ne.b32 p, 0, 0;\n\t"
        "@q mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done) : "r"(smem_addr(bar)), "r"(parity), "r"(e) : "memory");
    return __any_sync(0xFFFFFFFFu, done != 0);
}
constexpr long long WAIT_LIMIT = 4 * umma::WAIT_LIMIT_CYCLES;  // what row_again may take
__device__ __forceinline__ bool warp_wait(uint32_t e, uint64_t *bar, uint32_t parity) {
    if (poll(e, bar, parity)) return true;
    const long long t0 = clock64();
    while (!poll(e, bar, parity))
        if (__any_sync(0xFFFFFFFFu, clock64() - t0 > WAIT_LIMIT)) return false;
    return true;
}

// Tensor maps of the pages: {head_dim, page_size, kv_heads, pages}.
inline bool umma_maps(UmmaMaps *m, const mgc_cuda_paged &c) {
    auto fn = umma::encode_tiled_fn();
    if (!fn) return false;
    m->box_rows = (int)(c.page_size < 128 ? c.page_size : 128);
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.token_stride * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64u, (cuuint32_t)m->box_rows, 1u, 1u}, unit[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = c.dtype == MGC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    void *const base[2] = {c.k, c.v};
    CUtensorMap *const map[2] = {&m->k, &m->v};
    for (int i = 0; i < 2; ++i)
        if (fn(map[i], type, 4, base[i], dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

// Page sizes whose boxes tile 128 keys and keep the swizzle's 8-row groups whole, strides TMA takes.
inline bool umma_fits(const mgc_cuda_paged &c) {
    const int64_t most = (1ll << 39) - 16;  // elements of a stride below 2^40 bytes
    return c.dtype != MGC_F32 && c.head_dim <= 128 &&
           (c.page_size % 128 == 0 || c.page_size == 8 || c.page_size == 16 || c.page_size == 32 || c.page_size == 64) &&
           c.token_stride > 0 && c.head_stride > 0 && c.page_stride > 0 && c.token_stride < most && c.head_stride < most &&
           c.page_stride < most;
}

// Key tiles that row tile x of a unit's piece needs (the rows of tile 0 stop earlier if causal).
__device__ __forceinline__ int tiles_needed(const AttendParams &p, const Item &w, int x) {
    if (x) return w.rows - w.row0 > 128 ? w.tiles : 0;
    const RowRange mid = row_range(p, w.seq, min(w.row0 + 128, w.rows) - 1);
    return min(w.tiles, (max(mid.hi - w.lo, 0) + 127) >> 7);
}

// The slow way round for rows whose tiles held something that they do not see: this thread's row over
// the keys of piece w that it sees, on the FMA units, into TMEM where the products would have left it.
// `q` names the row's 16-byte chunks in shared memory. The whole warp calls; threads without `all` compute
// their row only if a key that it does not see has a value that is not finite. A piece of 16384 keys of 128
// channels takes about 40 ms while the other roles wait: WAIT_LIMIT, 4.5 s, covers pieces of 1.7 million.
template <typename T, int DP, typename Q>
__device__ __forceinline__ void row_again(const AttendParams &p, const Item &w, int row, Q q, bool all, bool maybe, uint32_t to, float &m, float &l) {
    const RowRange see = row_range(p, w.seq, row);
    const int lo = max(see.lo, w.lo), hi = min(see.hi, w.hi), ps = p.batch.page_size;
    const long long head = (long long)w.h * p.head_stride;
    // calls f with the offset of each key of [from, to) that has a page, until it returns false
    auto keys = [&](int from, int to, auto f) {
        for (int j = from; j < to;) {
            const int at = j / ps, end = to - at * ps < ps ? to : (at + 1) * ps, page = page_of(p.batch, w.b, at);
            long long off = (long long)page * p.page_stride + (long long)(j - at * ps) * p.token_stride + head;
            if (page >= 0) {
#pragma unroll 1
                for (; j < end; ++j, off += p.token_stride)
                    if (!f(off)) return;
            }
            j = end;
        }
    };
    if (!all && maybe) {
        auto finite = [&](long long off) {
            float z = 0.0f;
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
                if (c * 8 >= p.head_dim) continue;
                Pack<8, T> v;
                v.load(static_cast<const T *>(p.v_pages) + off + c * 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) z = fmaf(to_f(v.e[i]), 0.0f, z);
            }
            all = z != z;
            return !all;
        };
        keys(max(w.lo, w.first), min(lo, w.hi), finite);
        if (!all) keys(max(max(hi, w.lo), w.first), w.hi, finite);
    }
    if (!__any_sync(0xFFFFFFFFu, all)) return;
    float o[DP];
#pragma unroll
    for (int i = 0; i < DP; ++i) o[i] = 0.0f;
    if (all) {
        m = -INFINITY;
        l = 0.0f;
        keys(lo, hi, [&](long long off) {
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
                if (c * 8 >= p.head_dim) continue;
                Pack<8, T> x, y;
                x.load(q(c));
                y.load(static_cast<const T *>(p.k_pages) + off + c * 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) part[i & 3] = fmaf(to_f(x.e[i]), to_f(y.e[i]), part[i & 3]);
            }
            const float s = __fmul_rn((part[0] + part[1]) + (part[2] + part[3]), p.scale_log2);
            if (s == -INFINITY) return true;
            if (s > m) {
                const float f = ex2(m - s);
                m = s;
                l *= f;
#pragma unroll
                for (int i = 0; i < DP; ++i) o[i] *= f;
            }
            const float wgt = ex2(s - m + Weight<T>::LAZY_LIFT);
            l += wgt;
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
                if (c * 8 >= p.head_dim) continue;
                Pack<8, T> v;
                v.load(static_cast<const T *>(p.v_pages) + off + c * 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[c * 8 + i] = fmaf(wgt, to_f(v.e[i]), o[c * 8 + i]);
            }
            return true;
        });
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
        uint32_t t[32];
        umma::tmem_ld32(to + c * 32, t);
        umma::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) t[i] = all ? __float_as_uint(o[c * 32 + i]) : t[i];
        tmem_st32(to + c * 32, t);
    }
    tmem_wait_st();
}

template <typename T, int DP>
__global__ void __launch_bounds__(UmmaConfig<DP>::THREADS, 1)
paged_attention_umma_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ UmmaMaps maps) {
    using C = UmmaConfig<DP>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[C::STAGES], empty[C::STAGES], q_full[2], s_full[2], s_free[2], p_half[2], p_full[2], p_free[2], o_full[2];
    __shared__ __align__(8) uint64_t z_ask, z_done;
    __shared__ uint32_t tslot;
    __shared__ Walk stretch;
    __shared__ int bad_page;  // a page number was out of range
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sQ = base, *ring = base + 2 * C::TILE;
    const int tid = (int)threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        bad_page = 0;
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&q_full[x], 4);
            mbar_init(&s_full[x], 1);
            mbar_init(&s_free[x], 4);
            mbar_init(&p_free[x], 1);
            mbar_init(&p_half[x], 4);
            mbar_init(&p_full[x], 4);
            mbar_init(&o_full[x], 1);
        }
        mbar_init(&z_ask, 1);
        mbar_init(&z_done, 1);
        umma::fence_barrier_init();
        umma::prefetch_tmap(&maps.k);
        umma::prefetch_tmap(&maps.v);
    }
    if (warp == 8) umma::tmem_alloc(&tslot, 512);
    if (warp == 11) {
        const Walk k = find_stretch<256, 128>(p, (int)blockIdx.x, (int)gridDim.x, 0, p.kv_heads, lane);
        if (lane == 0) stretch = k;
    }
    if (warp == 10) zero_outside<T>(p, (int)blockIdx.x, (int)gridDim.x, 0, 1, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tslot;
    Walk walk = stretch;
    Item w;
    // A wait that runs out ends its role, and every role that waits for it.
    const uint32_t e = elect_one();
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (warp_wait(e, bar, parity)) return true;
        umma::set_error(p.batch.status, MGC_CUDA_TIMEOUT);
        return false;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
        if (warp == 9) {
            // ---------------- loads ----------------
            int slot = 0, laps = 0, issued = 0;
            const int boxes = (128 / maps.box_rows) * C::HALVES;  // of a tile: at most 32
            const int part = lane / C::HALVES, half = lane % C::HALVES;
            bool ok = true;
            while (ok && next_item<256, 128>(p, walk, w)) {
                // this lane's box of key tile j: page and first row in it; -1 if no row sees its keys
                auto box = [&](int j, int &row) {
                    const int at = w.lo + j * 128 + part * maps.box_rows;
                    row = at % p.batch.page_size;
                    if (lane >= boxes || j >= w.tiles || at >= w.hi || at + maps.box_rows <= w.first) return -1;
                    const int page = page_of(p.batch, w.b, at / p.batch.page_size);
                    if (page < 0) *static_cast<volatile int *>(&bad_page) = 1;
                    return page;
                };
                int row, page = box(0, row);
                for (int j = 0; ok && j < w.tiles; ++j) {
                    int next_row, next = box(j + 1, next_row);  // looked up one tile ahead
                    const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xFFFFFFFFu, page >= 0)) * (uint32_t)maps.box_rows * 128u;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        if (laps > 0) ok = ok && wait(&empty[slot], (uint32_t)(laps - 1) & 1u);
                        if (!ok) break;
                        if (lane == 0) mbar_expect_tx(&full[slot], bytes);
                        __syncwarp();
                        if (page >= 0)
                            umma::tma_load_4d(ring + slot * C::TILE + half * C::HALF + part * maps.box_rows * 128,
                                              kv ? &maps.v : &maps.k, &full[slot], half * 64, row, w.h, page);
                        ++issued;
                        if (++slot == C::STAGES) {
                            slot = 0;
                            ++laps;
                        }
                    }
                    page = next;
                    row = next_row;
                }
            }
            // after a timeout, the copies still in flight
            if (!ok) {
                for (int k = issued - 1; k >= 0 && k >= issued - C::STAGES; --k)
                    mbar_wait(&full[k % C::STAGES], (uint32_t)((k / C::STAGES) & 1));
            }
        } else if (warp == 8) {
            // ---------------- MMA ----------------
            // The tensor pipe takes an MMA only when the one before is nearly done, so whatever
            // stands between two of them is time lost. The warp runs this code converged, with one
            // elected lane's predicate on the MMAs: descriptors then live in uniform registers and
            // a chain of products issues without a gap (a loop of one lane's branch took 1.25-1.55
            // times as long for the same products).
            int slot = 0;
            uint32_t lap = 0, q_phase = 0, z_phase = 0, phase0 = 0, phase1 = 0;
            bool ok = true;
            constexpr uint32_t id_s = idesc_f16<T>(128, 0), id_o = idesc_f16<T>(DP, 1);
            const uint32_t tb = __shfl_sync(0xFFFFFFFFu, tbase, 0);
            auto step = [&]() {
                if (++slot == C::STAGES) {
                    slot = 0;
                    lap ^= 1u;
                }
            };
            auto scores = [&](int x, int stage) {
                const uint64_t a = sw128_desc(smem_addr(sQ) + x * C::TILE), k = sw128_desc(smem_addr(ring) + stage * C::TILE);
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) {
                    const uint32_t at = ((uint32_t)(ks >> 2) * C::HALF + (uint32_t)(ks & 3) * 32u) >> 4;
                    mma_f16_ss(e, tb + C::S_COL + x * 128, a + at, k + at, id_s, ks > 0);
                }
                commit_if(e, &s_full[x]);
            };
            while (ok && next_item<256, 128>(p, walk, w)) {
                const int need0 = tiles_needed(p, w, 0), need1 = tiles_needed(p, w, 1);
                // the first scores of each row tile as soon as its queries are there
                if (w.tiles > 0) ok = wait(&full[slot], lap);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    ok = ok && wait(&q_full[x], q_phase);
                    tc_fence_after();
                    if (ok && (x ? need1 : need0) > 0) scores(x, slot);
                    // a warpgroup whose rows see nothing here waits all the same: it must not be two
                    // items ahead, where q_full's parity would say the opposite
                    else if (ok && lane == 0) mbar_arrive(&o_full[x]);
                    __syncwarp();
                }
                q_phase ^= 1u;
                if (ok && w.tiles > 0) {
                    commit_if(e, &empty[slot]);
                    step();
                }
                for (int j = 0; ok && j < w.tiles; ++j) {
                    const int vs = slot;
                    ok = wait(&full[vs], lap);
                    step();
                    const int ks = slot;
                    const bool more = j + 1 < w.tiles;
                    const int key0 = w.lo + j * 128;
                    if (ok && (key0 < w.first || key0 + 128 > w.hi)) {
                        // rows of V that no row sees: warp 10 zeroes them
                        if (lane == 0) mbar_arrive(&z_ask);
                        __syncwarp();
                        ok = wait(&z_done, z_phase);
                        z_phase ^= 1u;
                    }
                    if (more) {
                        ok = ok && wait(&full[ks], lap);
                        step();
                    }
                    const uint64_t v = mn128_desc(smem_addr(ring) + vs * C::TILE, C::HALF);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (!ok || j >= (x ? need1 : need0)) continue;
                        const uint32_t o = tb + C::O_COL + x * DP, w16 = tb + C::P_COL + x * C::P_STEP;
                        uint32_t &phase = x ? phase1 : phase0;
                        if (C::APART && j + 1 < (x ? need1 : need0)) {
                            ok = wait(&s_free[x], phase);
                            if (!ok) continue;
                            tc_fence_after();
                            scores(x, ks);
                        }
                        ok = wait(&p_half[x], phase);
                        if (!ok) continue;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) mma_f16_ts(e, o, w16 + kk * 8, v + kk * (2048 >> 4), id_o, j > 0 || kk > 0);
                        ok = wait(&p_full[x], phase);
                        phase ^= 1u;
                        if (!ok) continue;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 4; kk < 8; ++kk) mma_f16_ts(e, o, w16 + kk * 8, v + kk * (2048 >> 4), id_o, 1);
                        if (j + 1 >= (x ? need1 : need0)) commit_if(e, &o_full[x]);
                        else if (C::APART) commit_if(e, &p_free[x]);
                        else scores(x, ks);
                    }
                    if (ok) {
                        commit_if(e, &empty[vs]);
                        if (more) commit_if(e, &empty[ks]);
                    }
                }
            }
        } else if (warp == 10) {
            // ---------------- zero rows of V, when the MMA warp asks ----------------
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            while (ok && next_item<256, 128>(p, walk, w)) {
                for (int j = 0; ok && j < w.tiles; ++j) {
                    const int vs = (slot + 2 * j + 1) % C::STAGES, key0 = w.lo + j * 128;
                    if (key0 >= w.first && key0 + 128 <= w.hi) continue;
                    ok = wait(&z_ask, phase);
                    phase ^= 1u;
                    if (!ok) break;
                    const int r0 = max(w.first - key0, 0), r1 = min(w.hi - key0, 128);
                    const int out = r0 + 128 - r1;  // rows outside
#pragma unroll 1
                    for (int i = lane; i < out * C::HALVES * 8; i += 32) {
                        int r = i / (C::HALVES * 8);
                        const int c = i % (C::HALVES * 8);
                        if (r >= r0) r += r1 - r0;
                        *reinterpret_cast<uint4 *>(ring + vs * C::TILE + (c >> 3) * C::HALF + r * 128 + (c & 7) * 16) =
                            make_uint4(0, 0, 0, 0);
                    }
                    umma::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&z_done);
                }
                slot = (slot + 2 * w.tiles) % C::STAGES;
            }
        } else {
            // ---------------- warp 11: how many pieces has the unit cut at the stretch's end? ----------------
            CutUnit cut{0, 0, 0, 0};
            while (next_item<256, 128>(p, walk, w))
                if (w.slot == 1) cut = cut_of<256, 128>(p, walk, w);
            if (lane == 0) p.cut[blockIdx.x] = cut;
        }
    } else {
        // ---------------- softmax: one row per thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
        const int x = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tbase + lanes + C::S_COL + x * 128, to = tbase + lanes + C::O_COL + x * DP;
        const uint32_t tp = tbase + lanes + C::P_COL + x * C::P_STEP;
        uint32_t s_phase = 0, o_phase = 0, free_phase = 0;
        bool ok = true;
        while (ok && next_item<256, 128>(p, walk, w)) {
            const int row = w.row0 + x * 128 + r;
            const bool live = row < w.rows;
            // element offsets of this thread's row of q and of out; a warp moves its 32 rows together,
            // 16 bytes a lane along the rows (a row per thread touches 32 lines an instruction)
            const int head = w.h * p.group + row % p.group;
            const long long token = w.seq.start + row / p.group;
            const long long q_off = token * p.q_ts + (long long)head * p.q_hs, o_off = token * p.o_ts + (long long)head * p.o_hs;
            constexpr int CHUNKS = DP / 8;               // 16-byte chunks of a 16-bit row
            uint8_t *rows32 = sQ + x * C::TILE + (r & 96) * 128;  // the warp's 32 rows of the Q tile
            auto chunk = [&](int rr, int c) { return rows32 + (c >> 3) * C::HALF + rr * 128 + (((c & 7) ^ (rr & 7)) << 4); };
            const int lives = min(32, w.rows - (w.row0 + x * 128 + (r & 96)));  // rows of the warp that exist
            {
                uint4 v[CHUNKS];  // every load in flight before the first store
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i) {
                    const int rr = (i * 32 + lane) / CHUNKS, c = (i * 32 + lane) % CHUNKS;
                    const long long off = __shfl_sync(0xFFFFFFFFu, q_off, rr);
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (rr < lives && c * 8 < p.head_dim)
                        v[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + off + c * 8));
                }
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i)
                    *reinterpret_cast<uint4 *>(chunk((i * 32 + lane) / CHUNKS, (i * 32 + lane) % CHUNKS)) = v[i];
                umma::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[x]);
            }
            const RowRange see = row_range(p, w.seq, row);
            float m = -INFINITY, l = 0.0f;  // m: the (lazy) reference of the weights, scaled
            const int need = tiles_needed(p, w, x);
            for (int j = 0; j < need; ++j) {
                ok = ok && wait(&s_full[x], s_phase);
                s_phase ^= 1u;
                if (!ok) break;
                tc_fence_after();
                float s[128];
                uint32_t t[32];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    umma::tmem_ld32(ts + c * 32, t);
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[c * 32 + i] = __uint_as_float(t[i]);
                }
                umma::tmem_wait_ld();
                if (C::APART) {  // the next tile's scores may take this one's place
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[x]);
                }
                const int key0 = w.lo + j * 128;
                if (__any_sync(0xFFFFFFFFu, live && (key0 < see.lo || key0 + 128 > see.hi))) {
                    // only the 32-key slices that some row of the warp does not see whole
                    const int from = live ? see.lo - key0 : 0, to_ = live ? see.hi - key0 : 128;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (__any_sync(0xFFFFFFFFu, to_ < c * 32 + 32)) {
#pragma unroll
                            for (int i = c * 32; i < c * 32 + 32; ++i)
                                if (i >= to_) s[i] = -INFINITY;
                        }
                        if (__any_sync(0xFFFFFFFFu, from > c * 32)) {
#pragma unroll
                            for (int i = c * 32; i < c * 32 + 32; ++i)
                                if (i < from) s[i] = -INFINITY;
                        }
                    }
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < 124; i += 8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = max3(top[e], s[i + 2 * e], s[i + 2 * e + 1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], s[124 + e]);
                const float mt = __fmul_rn(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), p.scale_log2);
                // grown by more than 2^LAZY (or the first finite maximum): move the reference
                const bool grow = mt > m + Weight<T>::LAZY;
                if (C::APART && j > 0) {  // the products with the last tile's weights are done
                    ok = wait(&p_free[x], free_phase);
                    free_phase ^= 1u;
                    if (!ok) break;
                    tc_fence_after();
                }
                if (j > 0 && __any_sync(0xFFFFFFFFu, grow)) {
                    const float f = grow ? ex2(m - mt) : 1.0f;
                    l *= f;
#pragma unroll
                    for (int c = 0; c < DP / 32; ++c) {
                        uint32_t t[32];
                        umma::tmem_ld32(to + c * 32, t);
                        umma::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) t[i] = __float_as_uint(__uint_as_float(t[i]) * f);
                        tmem_st32(to + c * 32, t);
                    }
                }
                if (grow) m = mt;
                const float y = m == -INFINITY ? 0.0f : m;
                const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), y2 = make_float2(Weight<T>::LAZY_LIFT - y, Weight<T>::LAZY_LIFT - y);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < 2; ++c) {  // the first 64 keys' products start while the others' weights are made
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float2 z = fma2(make_float2(s[c * 64 + 2 * i], s[c * 64 + 2 * i + 1]), scale2, y2);
                        z.x = ex2(z.x);
                        z.y = ex2(z.y);
                        sum[i & 1] = add2(sum[i & 1], z);
                        t[i] = pack2<T>(z.x, z.y);
                    }
                    tmem_st32(tp + c * 32, t);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(c ? &p_full[x] : &p_half[x]);
                }
                sum[0] = add2(sum[0], sum[1]);
                l += sum[0].x + sum[0].y;
            }
            ok = ok && wait(&o_full[x], o_phase);
            o_phase ^= 1u;
            tc_fence_after();
            if (!ok) break;
            if (need > 0) {
                bool bad = false;  // a page of this piece
                if (*static_cast<volatile int *>(&bad_page)) {
                    for (int at = max(w.lo, w.first) / p.batch.page_size + lane; at <= (w.hi - 1) / p.batch.page_size; at += 32)
                        bad = bad || page_of(p.batch, w.b, at) < 0;
                    bad = __any_sync(0xFFFFFFFFu, bad);
                }
                // a row that is not finite, although its scores are, and that does not see all of the piece
                bool maybe = live && l == l && (see.lo > max(w.lo, w.first) || see.hi < w.hi);
                if (__any_sync(0xFFFFFFFFu, maybe)) {
                    float odd[2] = {0.0f, 0.0f};  // NaN once a channel is not finite
#pragma unroll
                    for (int c = 0; c < DP / 32; ++c) {
                        uint32_t t[32];
                        umma::tmem_ld32(to + c * 32, t);
                        umma::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) odd[i & 1] = fmaf(__uint_as_float(t[i]), 0.0f, odd[i & 1]);
                    }
                    maybe = maybe && odd[0] + odd[1] != 0.0f;
                }
                if (bad || __any_sync(0xFFFFFFFFu, maybe)) {
                    auto q = [&](int c) { return reinterpret_cast<const T *>(chunk(lane, c)); };
                    row_again<T, DP>(p, w, w.row0 + x * 128 + r, q, bad, maybe, to, m, l);
                }
            }
            // ---- O: through the warp's rows of the Q tile (no longer read) to whole rows of memory ----
            const bool whole = w.slot < 0;
            const long long at = ((long long)blockIdx.x * 2 + w.slot) * 256 + x * 128 + (r & 96);  // a piece's first row
            const float inv = whole ? (l > 0.0f ? 1.0f / l : 0.0f) : 1.0f;
            if (!whole && live) p.part_ml[at + lane] = make_float2(m, l);
#pragma unroll
            for (int pass = 0; pass < 2; ++pass) {  // half of the channels at a time
                uint32_t t[32];
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) {
                    if (need > 0) {
                        umma::tmem_ld32(to + pass * (DP / 2) + c * 32, t);
                        umma::tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) t[i] = 0u;
                    }
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t q[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                q[u] = pack2<T>(__uint_as_float(t[8 * i + 2 * u]) * inv, __uint_as_float(t[8 * i + 2 * u + 1]) * inv);
                            *reinterpret_cast<uint4 *>(chunk(lane, pass * (DP / 16) + c * 4 + i)) = make_uint4(q[0], q[1], q[2], q[3]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4 *>(chunk(lane, c * 8 + i)) =
                                make_uint4(t[4 * i], t[4 * i + 1], t[4 * i + 2], t[4 * i + 3]);
                    }
                }
                if (whole && pass == 0) continue;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i) {
                    const int rr = (i * 32 + lane) / CHUNKS, c = (i * 32 + lane) % CHUNKS;
                    const long long off = __shfl_sync(0xFFFFFFFFu, o_off, rr);
                    if (rr >= lives) continue;
                    const uint4 v = *reinterpret_cast<const uint4 *>(chunk(rr, c));
                    if (whole) {
                        if (c * 8 < p.head_dim) *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + off + c * 8) = v;
                    } else if (pass * (DP / 2) + c * 4 < p.head_dim) {
                        *reinterpret_cast<uint4 *>(p.part + (at + rr) * p.head_dim + pass * (DP / 2) + c * 4) = v;
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        umma::tmem_dealloc(tbase, 512);
    }
}

}  // namespace paged
}  // namespace mgc
