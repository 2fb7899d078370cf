// Paged attention on tcgen05 for 16-bit types: chunks of many query rows.
//
// A CTA takes one (sequence, key head), 256 query rows (row = token * group + head of the group) as
// two tiles of 128, and one part of the rows' visible keys in tiles of 128. Per key tile and row
// tile: S = Q K^T (M = N = 128, K = D) into TMEM; a warpgroup, one row per thread, turns the row
// into weights 2^(scale s - m), writes them as 16-bit values over S; O += P V (M = 128, N = D,
// K = 128) with P read from TMEM. The two row tiles alternate: while one warpgroup exponentiates,
// the tensor core works for the other.
//
// * Q rows: each thread copies its own row into 128B-swizzled shared memory (any strides).
// * K and V tiles arrive by TMA from the pages, one box of min(page_size, 128) rows x 64 channels
//   per page and channel half, lane l of the loading warp issuing box l; a ring of stages holds
//   K and V tiles in the order K0 V0 K1 V1 ... K is a K-major operand, V (channels contiguous) an
//   MN-major one. Channels past the head width are the tensor map's zero fill.
// * The maximum is lazy: O (in TMEM) is rescaled only when a row's maximum has grown by more than
//   2^8 since the last time; the weights then stay below 2^8, far from overflow in either type,
//   and the row sum carries the same reference, so the result is unchanged. A rescale needs no
//   wait: S of tile j is committed after P V of tile j - 1.
// * Rows of V that no row sees (past the last visible key, before the first) are zeroed in shared
//   memory before they are used: a page's unused rows hold anything, and 0 * NaN is NaN.
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
using umma::mma_commit;
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
    // two softmax warpgroups, then a warpgroup of the MMA warp, the load warp and two idle ones.
    // 384 threads launch with 168 registers each (64,512); the split keeps that sum:
    // 256 x 224 + 128 x 56
    static constexpr int THREADS = 384;
    static constexpr int SOFTMAX_REGS = 224, OTHER_REGS = 56;
    static constexpr uint32_t S_COL = 0, O_COL = 256; // TMEM columns: S0 S1 O0 O1
};

// D = A B with A in TMEM (16-bit values packed in pairs along K) or shared memory.
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
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
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

// The keys of one CTA's work item: [lo, hi) in tiles of 128 from lo, `tiles` of them, and how many
// of those row tile x needs (rows of the first tile stop earlier under a causal mask).
struct Item {
    int rows, row0;        // query rows of the sequence; first of the CTA's
    int lo, hi, tiles;
    int first;             // first key that any of the rows sees
    int need0, need1;
    __device__ __forceinline__ int need(int x) const { return x ? need1 : need0; }
};

__device__ __forceinline__ Item umma_item(const AttendParams &p, int n, int nq, int tile, int split) {
    Item w;
    w.rows = nq * p.group;
    w.row0 = tile * 256;
    const RowRange a = row_range(p, n, nq, w.row0), z = row_range(p, n, nq, min(w.row0 + 256, w.rows) - 1);
    const RowRange mid = row_range(p, n, nq, min(w.row0 + 128, w.rows) - 1);
    const int lo = a.lo & ~127, hi = max(z.hi, 0);
    const int all = (max(hi - lo, 0) + 127) >> 7, per = (all + p.splits - 1) / p.splits;
    w.first = a.lo;
    w.lo = lo + split * per * 128;
    w.hi = min(hi, w.lo + per * 128);
    w.tiles = w.hi > w.lo ? (w.hi - w.lo + 127) >> 7 : 0;
    w.need0 = min(w.tiles, (max(mid.hi - w.lo, 0) + 127) >> 7);
    w.need1 = w.rows - w.row0 > 128 ? w.tiles : 0;
    return w;
}

template <typename T, int DP>
__global__ void __launch_bounds__(UmmaConfig<DP>::THREADS, 1)
paged_attention_umma_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ UmmaMaps maps) {
    using C = UmmaConfig<DP>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[C::STAGES], empty[C::STAGES], q_full[2], s_full[2], p_full[2], o_full[2];
    __shared__ uint32_t tslot;
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sQ = base, *ring = base + 2 * C::TILE;
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned u = blockIdx.x;
    const int split = (int)blockIdx.y;
    const int kh = (int)(u % (unsigned)p.kv_heads);
    u /= (unsigned)p.kv_heads;
    const int tile0 = p.row_tiles - 1 - (int)(u % (unsigned)p.row_tiles);  // longest rows first
    const int b = (int)(u / (unsigned)p.row_tiles);
    const int start = __ldg(p.batch.q_starts + b), nq = __ldg(p.batch.q_starts + b + 1) - start;
    const int n = min(__ldg(p.batch.kv_lens + b), p.max_positions);
    if (n != __ldg(p.batch.kv_lens + b) && tid == 0 && p.batch.status) *p.batch.status = MGC_CUDA_GATHER_OOB;
    if (tile0 * 256 >= nq * p.group) return;

    if (tid == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&q_full[x], 128);
            mbar_init(&s_full[x], 1);
            mbar_init(&p_full[x], 128);
            mbar_init(&o_full[x], 1);
        }
        umma::fence_barrier_init();
        umma::prefetch_tmap(&maps.k);
        umma::prefetch_tmap(&maps.v);
    }
    if (warp == 8) umma::tmem_alloc(&tslot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tslot;
    // a warp's bounded wait; a wait that runs out ends its role, and every role that waits for it
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (__all_sync(0xFFFFFFFFu, mbar_wait(bar, parity))) return true;
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
            for (int tile = tile0; ok && tile * 256 < nq * p.group; tile += p.row_tiles) {
                const Item w = umma_item(p, n, nq, tile, split);
                // this lane's box of key tile j: page and first row in it; -1 if no row sees its keys
                auto box = [&](int j, int &row) {
                    const int at = w.lo + j * 128 + part * maps.box_rows;
                    row = at % p.batch.page_size;
                    if (lane >= boxes || j >= w.tiles || at >= w.hi || at + maps.box_rows <= w.first) return -1;
                    return page_of(p.batch, b, at / p.batch.page_size);
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
                                              kv ? &maps.v : &maps.k, &full[slot], half * 64, row, kh, page);
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
            int slot = 0;
            uint32_t lap = 0, q_phase = 0, p_phase = 0;  // p_phase: bit x of row tile x
            bool ok = true;
            constexpr uint32_t id_s = idesc_f16<T>(128, 0), id_o = idesc_f16<T>(DP, 1);
            auto step = [&]() {
                if (++slot == C::STAGES) {
                    slot = 0;
                    lap ^= 1u;
                }
            };
            auto scores = [&](int x, int stage) {
                uint64_t a = sw128_desc(smem_addr(sQ + x * C::TILE)), k = sw128_desc(smem_addr(ring + stage * C::TILE));
                asm volatile("" : "+l"(a), "+l"(k));  // computed here, not kept in registers around the loops
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) {
                    const uint32_t at = ((uint32_t)(ks >> 2) * C::HALF + (uint32_t)(ks & 3) * 32u) >> 4;
                    mma_f16_ss(tbase + C::S_COL + x * 128, a + at, k + at, id_s, ks > 0);
                }
                mma_commit(&s_full[x]);
            };
            for (int tile = tile0; ok && tile * 256 < nq * p.group; tile += p.row_tiles) {
                const Item w = umma_item(p, n, nq, tile, split);
                ok = ok && wait(&q_full[0], q_phase) && wait(&q_full[1], q_phase);
                q_phase ^= 1u;
                tc_fence_after();
                if (w.tiles > 0) {
                    ok = ok && wait(&full[slot], lap);
                    tc_fence_after();
                    if (ok && lane == 0) {
                        if (w.need0 > 0) scores(0, slot);
                        if (w.need1 > 0) scores(1, slot);
                        mma_commit(&empty[slot]);
                    }
                    __syncwarp();
                    step();
                }
                for (int j = 0; ok && j < w.tiles; ++j) {
                    const int vs = slot;
                    ok = ok && wait(&full[vs], lap);
                    step();
                    const int ks = slot;
                    const bool more = j + 1 < w.tiles;
                    if (more) {
                        ok = ok && wait(&full[ks], lap);
                        step();
                    }
                    // rows of V outside [first, hi): zeros
                    const int key0 = w.lo + j * 128;
                    if (ok && (key0 < w.first || key0 + 128 > w.hi)) {
                        const int r0 = max(w.first - key0, 0), r1 = min(w.hi - key0, 128);
#pragma unroll 1
                        for (int x = lane; x < 128 * C::HALVES * 8; x += 32) {
                            const int r = (x >> 3) & 127;
                            if (r < r0 || r >= r1)
                                *reinterpret_cast<uint4 *>(ring + vs * C::TILE + (x >> 10) * C::HALF + r * 128 + (x & 7) * 16) =
                                    make_uint4(0, 0, 0, 0);
                        }
                        umma::fence_proxy_async_smem();
                        __syncwarp();
                    }
#pragma unroll 1
                    for (int x = 0; x < 2; ++x) {
                        if (ok && j < w.need(x)) {
                            ok = wait(&p_full[x], (p_phase >> x) & 1u);
                            p_phase ^= 1u << x;
                            tc_fence_after();
                            if (ok && lane == 0) {
                                uint64_t v = mn128_desc(smem_addr(ring + vs * C::TILE), C::HALF);
                                asm volatile("" : "+l"(v));
#pragma unroll
                                for (int kk = 0; kk < 8; ++kk)
                                    mma_f16_ts(tbase + C::O_COL + x * DP, tbase + C::S_COL + x * 128 + kk * 8, v + kk * (2048 >> 4),
                                               id_o, j > 0 || kk > 0);
                                if (x == 1 || j >= w.need1) mma_commit(&empty[vs]);
                                if (j + 1 < w.need(x)) scores(x, ks);
                                else mma_commit(&o_full[x]);
                            }
                            __syncwarp();
                        } else if (ok && x == 1 && j >= w.need0 && lane == 0) {
                            mma_commit(&empty[vs]);  // no row tile used it
                        }
                    }
                    if (ok && more && lane == 0) mma_commit(&empty[ks]);
                    __syncwarp();
                }
            }
        }
    } else {
        // ---------------- softmax: one row per thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
        const int x = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tbase + lanes + C::S_COL + x * 128, to = tbase + lanes + C::O_COL + x * DP;
        uint32_t s_phase = 0, o_phase = 0;
        bool ok = true;
        for (int tile = tile0; ok && tile * 256 < nq * p.group; tile += p.row_tiles) {
            const Item w = umma_item(p, n, nq, tile, split);
            const int row = w.row0 + x * 128 + r;
            const bool live = row < w.rows;
            const int head = kh * p.group + row % p.group;
            const long long token = start + row / p.group;
            {
                uint8_t *q = sQ + x * C::TILE + r * 128;
                const T *src = static_cast<const T *>(p.q) + token * p.q_ts + (long long)head * p.q_hs;
#pragma unroll
                for (int c = 0; c < DP / 8; ++c) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (live && c * 8 < p.head_dim) v = *reinterpret_cast<const uint4 *>(src + c * 8);
                    *reinterpret_cast<uint4 *>(q + (c >> 3) * C::HALF + (((c & 7) ^ (r & 7)) << 4)) = v;
                }
                umma::fence_proxy_async_smem();
                mbar_arrive(&q_full[x]);
            }
            const RowRange see = row_range(p, n, nq, row);
            float m = -INFINITY, l = 0.0f;  // m: the (lazy) reference of the weights, scaled
            const int need = w.need(x);
            for (int j = 0; j < need; ++j) {
                ok = ok && wait(&s_full[x], s_phase);
                s_phase ^= 1u;
                if (!ok) break;
                tc_fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t t[32];
                    umma::tmem_ld32(ts + c * 32, t);
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[c * 32 + i] = __uint_as_float(t[i]);
                }
                umma::tmem_wait_ld();
                const int key0 = w.lo + j * 128;
                if (__any_sync(0xFFFFFFFFu, live && (key0 < see.lo || key0 + 128 > see.hi))) {
                    const int from = see.lo - key0, to_ = see.hi - key0;
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i < from || i >= to_) s[i] = -INFINITY;
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < 128; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
                const float mt = __fmul_rn(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), p.scale_log2);
                // grown by more than 2^8 (or the first finite maximum): move the reference
                const bool grow = mt > m + 8.0f;
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
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t t[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float a = ex2(fmaf(s[c * 64 + 2 * i], p.scale_log2, -y));
                        const float e = ex2(fmaf(s[c * 64 + 2 * i + 1], p.scale_log2, -y));
                        sum[i & 1] += a;
                        sum[2 + (i & 1)] += e;
                        t[i] = pack2<T>(a, e);
                    }
                    tmem_st32(ts + c * 32, t);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[x]);
            }
            if (need > 0) {
                ok = ok && wait(&o_full[x], o_phase);
                o_phase ^= 1u;
                tc_fence_after();
            }
            if (!ok) break;
            // ---- the row of O ----
            const long long at = ((long long)split * p.tokens + token) * p.q_heads + head;
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            T *out = static_cast<T *>(p.out) + token * p.o_ts + (long long)head * p.o_hs;
            if (p.splits > 1 && live) p.part_ml[at] = make_float2(m, l);
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                uint32_t t[32];
                if (need > 0) {
                    umma::tmem_ld32(to + c * 32, t);
                    umma::tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) t[i] = 0u;
                }
                if (!live) continue;
                if (p.splits > 1) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c * 32 + i * 4 < p.head_dim)
                            *reinterpret_cast<uint4 *>(p.part + at * p.head_dim + c * 32 + i * 4) =
                                make_uint4(t[4 * i], t[4 * i + 1], t[4 * i + 2], t[4 * i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c * 32 + i * 8 < p.head_dim) {
                            uint4 v;
                            uint32_t *q = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                q[e] = pack2<T>(__uint_as_float(t[8 * i + 2 * e]) * inv, __uint_as_float(t[8 * i + 2 * e + 1]) * inv);
                            *reinterpret_cast<uint4 *>(out + c * 32 + i * 8) = v;
                        }
                }
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
