// Paged attention on warp-level matrix instructions: decoding (few query rows, memory bound) and
// tiles of rows of any head width and page size.
//
// A CTA takes one (sequence, key head), a tile of R = 16 WM query rows (row = token * group + head
// of the group, so the heads that share a key head share its K and V loads) and a part of the
// tile's visible keys. WM x WN warps: warp (wm, wn) owns rows 16 wm .. 16 wm + 15 and the
// wn-th slice of every stage's BN keys, with its own running maximum, sum and output, so warps
// meet only at the end. K and V rows arrive by cp.async (16 bytes per thread, zero fill for keys
// that no row sees, so nothing there can reach a sum) into a ring of STAGES stages; rows are padded
// by 16 bytes to an odd number of 16-byte chunks, which keeps ldmatrix and the 32-bit fragment
// loads free of bank conflicts.
//
// 16-bit types: m16n8k16 products, the weights rounded to the type before the second one (as the
// type's own rounding of the output is of the same size). fp32: every operand x is split into
// h = x rounded to TF32 and x - h, and h h' + h l' + l h' are three m16n8k8 TF32 products into a
// fresh fp32 accumulator per tile that is added to the running one in fp32: the instruction
// truncates its sums, and a chain over the whole context would shrink the output by ~1e-8 per step.
//
// fp32 with few rows per key head (SIMT): the split products would cost the same for 1 row as for 16;
// up to 8 rows go through the FMA units instead, a key per lane for the scores and channels per lane
// for the output.
//
// When there are fewer units (row tiles of a sequence and key head) than the SMs hold CTAs, up to 8
// CTAs of a cluster take equal parts of a unit's keys and add their partial results through
// distributed shared memory. Else, or when 8 are not enough, every CTA takes an even share of all
// units' keys and pieces go through a workspace (paged_work.cuh). Partial sums are added in a fixed
// order, so a call repeats its bits.
//
// Decoding is bound by memory: 64 sequences of 8 key heads x 128 up to 8192 positions, bf16, 1.32 GB
// in 229 to 248 us (5.8 to 5.3 TB/s, 89 to 82 % of the copy bandwidth); one of 131071 positions 101 to 110 us
// (5.3 to 4.9 TB/s, the second kernel in it); 16 GPT-2 sequences up to 1024 positions, fp32, in clusters of
// two, 22.5 us (3.2 TB/s: the blocks' start, the first loads and the cluster's sum are half).
#pragma once

#include "paged_work.cuh"

namespace mgc {
namespace paged {

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes global -> shared; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, hi the nearest TF32 value; the instruction reads the upper 19 bits of lo.
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    lo = __float_as_uint(x - __uint_as_float(hi));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Word of the same shared address in CTA `rank` of the cluster.
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

constexpr int MAX_CLUSTER = 8;  // portable cluster size

// SIMT > 0: that many rows (fp32, at most 128 channels) on the FMA units, all four warps along the keys.
template <typename T, int DP, int WM, int WN, int SIMT> struct MmaConfig {
    static constexpr bool F32 = sizeof(T) == 4;
    // lanes that share a key of the plain form, each a part of its channels
    static constexpr int PARTS = DP <= 32 ? 1 : DP <= 64 ? 2 : 4;
    static constexpr int THREADS = 32 * WM * WN;
    static constexpr int R = SIMT ? SIMT : 16 * WM;
    static constexpr int BN = SIMT ? WN * 32 / PARTS : F32 ? 32 : 64;  // keys per stage
    static constexpr int KW = BN / WN;               // of them, a warp's
    static constexpr int KG = DP > 128 && KW > 32 ? 32 : KW;  // keys per softmax step (registers)
    // two for the plain form: more blocks an SM beat more stages a block (16 x 1024 fp32 24.8 -> 22.6 us)
    static constexpr int STAGES = DP > 128 || SIMT ? 2 : 3;
    // blocks that an SM is to hold (0: as it comes): even shares are cut for 4, and at 148 registers 3 fit, so
    // that a second round ran (64 x 4096, 16-bit, 8 key heads x 64: 116 us, at 128 registers 80 us)
    static constexpr int RESIDENT = !F32 && DP == 64 && WM == 1 ? 4 : 0;
    static constexpr int CH = 16 / (int)sizeof(T);   // elements of a 16-byte chunk
    static constexpr int ROW = DP * (int)sizeof(T) + 16;  // bytes of a padded K / V row
    static constexpr int STAGE = 2 * BN * ROW;
    static constexpr bool Q_REGS = !F32 && DP <= 128;     // Q fragments stay in registers
    static constexpr int Q_BYTES = Q_REGS ? 0 : R * ROW;
    static constexpr int ORED = DP + 4;              // floats of a row of the final reduction
    static constexpr int RED = WN * R * (ORED + 2) * 4;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int SMEM = Q_BYTES + (RING > RED ? RING : RED) + STAGES * BN * 8 + (SIMT ? WN * R * KW * 4 : 0);
};

// EVEN: the CTA takes an even share of all units' keys (paged_work.cuh); else one row tile's keys, or
// the part of them that its rank in a cluster names.
template <typename T, int DP, int WM, int WN, int SIMT, bool EVEN>
__global__ void __launch_bounds__(MmaConfig<T, DP, WM, WN, SIMT>::THREADS, MmaConfig<T, DP, WM, WN, SIMT>::RESIDENT * EVEN)
paged_attention_mma_kernel(const __grid_constant__ AttendParams p) {
    using C = MmaConfig<T, DP, WM, WN, SIMT>;
    constexpr int R = C::R, BN = C::BN, KW = C::KW, KG = C::KG, ROW = C::ROW, NB = KG / 8 ? KG / 8 : 1, DB = SIMT ? 1 : DP / 8;
    constexpr int CPR = DP / C::CH;  // 16-byte chunks of a padded row
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *sQ = smem;
    uint8_t *ring = smem + C::Q_BYTES;
    long long *sOff = reinterpret_cast<long long *>(smem + C::SMEM - C::STAGES * BN * 8 - (SIMT ? WN * R * KW * 4 : 0));
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int wm = warp % WM, wn = warp / WM;
    const int g4 = lane >> 2, t4 = lane & 3;
    const int chunks = p.head_dim / C::CH;

    const int split = EVEN ? 0 : (int)blockIdx.y;
    // one piece: rows row0 .. of (sequence b, key head kh) over keys [k_lo, k_hi)
    auto piece = [&](int b, int kh, const Sequence &seq, int row0, int k_lo, int k_hi, int slot) {
        const int rows = seq.nq * p.group, tiles = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
        const T *kp = static_cast<const T *>(p.k_pages) + kh * p.head_stride;
        const T *vp = static_cast<const T *>(p.v_pages) + kh * p.head_stride;
        // keys below first.lo no row sees; all rows see [all_lo, all_hi)
        const RowRange first = row_range(p, seq, row0), last = row_range(p, seq, min(row0 + R, rows) - 1);
        const int all_lo = last.lo, all_hi = first.hi;

        // Byte offset (of K and V alike) of key j of this thread's stage row, or -1: not loaded. In two
        // halves, the table's entry fetched a stage's work before it is looked at.
        const int ps = p.batch.page_size;
        bool bad_page = false;  // met by this thread
        auto fetch_page = [&](int j) {
            const int at = j / ps;
            return j < k_hi && j >= first.lo && at < p.batch.table_pages
                       ? __ldg(p.batch.table + (long long)b * p.batch.table_stride + at) : -1;
        };
        auto offset_of = [&](int j, int page) -> long long {
            if (j >= k_hi || j < first.lo) return -1;
            if (page < 0 || page >= p.batch.pages) {
                if (p.batch.status) *p.batch.status = MGC_CUDA_GATHER_OOB;
                bad_page = true;
                return -1;
            }
            return ((long long)page * p.page_stride + (long long)(j % ps) * p.token_stride) * (long long)sizeof(T);
        };
        auto load_stage = [&](int it) {
            uint8_t *st = ring + (it % C::STAGES) * C::STAGE;
            const long long *off = sOff + (it % C::STAGES) * BN;
#pragma unroll
            for (int x0 = 0; x0 < BN * CPR; x0 += C::THREADS) {
                const int r = (x0 + tid) / CPR, c = (x0 + tid) % CPR;
                if (c >= chunks || (BN * CPR % C::THREADS && r >= BN)) continue;
                const long long o = off[r];
                const long long at = o < 0 ? 0 : o + c * 16;
                const uint32_t dst = smem_u32(st + r * ROW + c * 16);
                cp_async16(dst, reinterpret_cast<const char *>(kp) + at, o < 0 ? 0 : 16);
                cp_async16(dst + BN * ROW, reinterpret_cast<const char *>(vp) + at, o < 0 ? 0 : 16);
            }
        };

        // Q: fragments in registers, or rows in shared memory
        auto q_ptr = [&](int row) {
            const int i = row / p.group, h = kh * p.group + row % p.group;
            return static_cast<const T *>(p.q) + (long long)(seq.start + i) * p.q_ts + (long long)h * p.q_hs;
        };
        uint32_t qf[C::Q_REGS ? DP / 16 : 1][4];
        if constexpr (C::Q_REGS) {
            const int ra = row0 + 16 * wm + g4, rb = ra + 8;
            const T *qa = ra < rows ? q_ptr(ra) : nullptr, *qb = rb < rows ? q_ptr(rb) : nullptr;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                const int c = ks * 16 + t4 * 2;
                qf[ks][0] = qa && c < p.head_dim ? *reinterpret_cast<const uint32_t *>(qa + c) : 0u;
                qf[ks][1] = qb && c < p.head_dim ? *reinterpret_cast<const uint32_t *>(qb + c) : 0u;
                qf[ks][2] = qa && c + 8 < p.head_dim ? *reinterpret_cast<const uint32_t *>(qa + c + 8) : 0u;
                qf[ks][3] = qb && c + 8 < p.head_dim ? *reinterpret_cast<const uint32_t *>(qb + c + 8) : 0u;
            }
        } else {
            for (int x = tid; x < R * (CPR); x += C::THREADS) {
                const int r = x / (CPR), c = x % (CPR);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row0 + r < rows && c < chunks) v = *reinterpret_cast<const uint4 *>(q_ptr(row0 + r) + c * C::CH);
                *reinterpret_cast<uint4 *>(sQ + r * ROW + c * 16) = v;
            }
        }

        const RowRange r0 = row_range(p, seq, row0 + 16 * wm + g4), r1 = row_range(p, seq, row0 + 16 * wm + g4 + 8);
        float o[DB][4], m0, m1, l0, l1;
        // plain form: every row's maximum, this lane's part of its sum, and CL channels of its output
        constexpr int SR = SIMT ? SIMT : 1, CL = DP / 32;
        float so[SR][CL], sm_[SR], sl_[SR];
        RowRange sr[SR];
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.0f;
        if constexpr (SIMT > 0) {
#pragma unroll
            for (int r = 0; r < SR; ++r) {
                sr[r] = row_range(p, seq, row0 + r);
                sm_[r] = -INFINITY;
                sl_[r] = 0.0f;
#pragma unroll
                for (int i = 0; i < CL; ++i) so[r][i] = 0.0f;
            }
        }

        // the first stages; a stage's offsets are looked up well before its loads
        for (int x = tid; x < C::STAGES * BN; x += C::THREADS) sOff[x] = offset_of(k_lo + x, fetch_page(k_lo + x));
        __syncthreads();
#pragma unroll
        for (int it = 0; it < C::STAGES - 1; ++it) {
            if (it < tiles) load_stage(it);
            cp_async_commit();
        }

        for (int it = 0; it < tiles; ++it) {
            cp_async_wait<C::STAGES - 2>();
            __syncthreads();
            if (it + C::STAGES - 1 < tiles) load_stage(it + C::STAGES - 1);
            cp_async_commit();
            const int j_next = k_lo + (it + C::STAGES) * BN + tid;
            const int page_next = tid < BN ? fetch_page(j_next) : -1;

            const uint8_t *st = ring + (it % C::STAGES) * C::STAGE;
            if constexpr (SIMT > 0) {
                // scores: lane (key, part) sums its part's channels of its key, the parts meet by
                // shuffles; output: lane owns channels CL lane .., weights broadcast from shared memory
                constexpr int PC = DP / C::PARTS / 4;  // 16-byte chunks of a part
                const int key = lane % KW, part = lane / KW;
                const int j0 = k_lo + it * BN + wn * KW, j = j0 + key;
                if (j0 < k_hi) {
                    float *sP = reinterpret_cast<float *>(smem + C::SMEM) - (wn + 1) * R * KW;
                    const float4 *kr = reinterpret_cast<const float4 *>(st + (wn * KW + key) * ROW) + part * PC;
                    float x[SR];
#pragma unroll
                    for (int r = 0; r < SR; ++r) x[r] = 0.0f;
#pragma unroll
                    for (int c = 0; c < PC; ++c) {
                        const float4 kv = kr[c];
#pragma unroll
                        for (int r = 0; r < SR; ++r) {
                            const float4 qv = reinterpret_cast<const float4 *>(sQ + r * ROW)[part * PC + c];
                            x[r] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, x[r]))));
                        }
                    }
#pragma unroll
                    for (int r = 0; r < SR; ++r) {
#pragma unroll
                        for (int d = KW; d < 32; d <<= 1) x[r] += __shfl_xor_sync(0xFFFFFFFFu, x[r], d);
                        if (j < sr[r].lo || j >= sr[r].hi || j >= k_hi) x[r] = -INFINITY;
                        float top = x[r];
#pragma unroll
                        for (int d = 1; d < KW; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                        top = fmaxf(top, sm_[r]);
                        const float y = top == -INFINITY ? 0.0f : __fmul_rn(top, p.scale_log2);
                        const float f = ex2(__fmul_rn(sm_[r], p.scale_log2) - y), wgt = ex2(fmaf(x[r], p.scale_log2, -y));
                        sm_[r] = top;
                        sl_[r] = sl_[r] * f + wgt;
#pragma unroll
                        for (int i = 0; i < CL; ++i) so[r][i] *= f;
                        if (part == 0) sP[r * KW + key] = wgt;
                    }
                    __syncwarp();
                    const float *vr = reinterpret_cast<const float *>(st + (BN + wn * KW) * ROW) + lane * CL;
#pragma unroll
                    for (int k4 = 0; k4 < KW; k4 += 4) {
                        float4 pw[SR];
#pragma unroll
                        for (int r = 0; r < SR; ++r) pw[r] = *reinterpret_cast<const float4 *>(sP + r * KW + k4);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float v[CL];
                            if constexpr (CL == 2) {
                                const float2 t = *reinterpret_cast<const float2 *>(vr + (k4 + k) * (ROW / 4));
                                v[0] = t.x;
                                v[1] = t.y;
                            } else if constexpr (CL == 4) {
                                const float4 t = *reinterpret_cast<const float4 *>(vr + (k4 + k) * (ROW / 4));
                                v[0] = t.x;
                                v[1] = t.y;
                                v[2] = t.z;
                                v[3] = t.w;
                            } else {
#pragma unroll
                                for (int i = 0; i < CL; ++i) v[i] = vr[(k4 + k) * (ROW / 4) + i];
                            }
#pragma unroll
                            for (int r = 0; r < SR; ++r) {
                                const float wgt = k == 0 ? pw[r].x : k == 1 ? pw[r].y : k == 2 ? pw[r].z : pw[r].w;
#pragma unroll
                                for (int i = 0; i < CL; ++i) so[r][i] = fmaf(wgt, v[i], so[r][i]);
                            }
                        }
                    }
                    __syncwarp();  // the weights are read before the next stage's are written
                }
            } else {
#pragma unroll
            for (int kg = 0; kg < KW / KG; ++kg) {
                const int kw = wn * KW + kg * KG;  // first of the warp's keys in the stage
                const int j0 = k_lo + it * BN + kw;
                if (j0 >= k_hi) break;
                const uint32_t ks_base = smem_u32(st + kw * ROW), vs_base = ks_base + BN * ROW;
                float s[NB][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.0f;
                if constexpr (!C::F32) {
                    const uint32_t kl = ks_base + ((lane & 7) + ((lane >> 4) & 1) * 8) * ROW + ((lane >> 3) & 1) * 16;
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ++ks) {
                        uint32_t qa[4];
                        if constexpr (C::Q_REGS) {
                            qa[0] = qf[ks][0]; qa[1] = qf[ks][1]; qa[2] = qf[ks][2]; qa[3] = qf[ks][3];
                        } else {
                            ldsm4(smem_u32(sQ + (16 * wm + (lane & 15)) * ROW + ks * 32 + (lane >> 4) * 16), qa);
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; nb += 2) {
                            uint32_t kb[4];
                            ldsm4(kl + nb * 8 * ROW + ks * 32, kb);
                            mma16<T>(s[nb], qa, kb[0], kb[1]);
                            mma16<T>(s[nb + 1], qa, kb[2], kb[3]);
                        }
                    }
                } else {
                    // the large products in chains of four steps and the small ones apart, added in
                    // fp32: each step of a chain truncates its sum
                    float big[NB][4], small[NB][4];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) big[nb][e] = small[nb][e] = 0.0f;
                    }
#pragma unroll 4
                    for (int ks = 0; ks < DP / 8; ++ks) {
                        uint32_t ah[4], al[4];
                        const float *qr = reinterpret_cast<const float *>(sQ + (16 * wm + g4) * ROW) + ks * 8 + t4;
                        split_tf32(qr[0], ah[0], al[0]);
                        split_tf32(qr[8 * ROW / 4], ah[1], al[1]);
                        split_tf32(qr[4], ah[2], al[2]);
                        split_tf32(qr[8 * ROW / 4 + 4], ah[3], al[3]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const float *kr = reinterpret_cast<const float *>(st + (kw + nb * 8 + g4) * ROW) + ks * 8 + t4;
                            uint32_t h0, q0, h1, q1;
                            split_tf32(kr[0], h0, q0);
                            split_tf32(kr[4], h1, q1);
                            mma8(small[nb], al, h0, h1);
                            mma8(small[nb], ah, q0, q1);
                            mma8(big[nb], ah, h0, h1);
                        }
                        if (ks % 4 == 3) {
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    s[nb][e] += big[nb][e];
                                    big[nb][e] = 0.0f;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[nb][e] += small[nb][e];
                    }
                }
                // infinite keys have no split (inf - inf): take such scores from plain products
                if constexpr (C::F32) {
                    bool odd = false;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) odd = odd || s[nb][e] != s[nb][e];
                    }
                    if (__any_sync(0xFFFFFFFFu, odd)) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (s[nb][e] == s[nb][e]) continue;
                                const float *qr = reinterpret_cast<const float *>(sQ + (16 * wm + g4 + (e < 2 ? 0 : 8)) * ROW);
                                const float *kr = reinterpret_cast<const float *>(st + (kw + nb * 8 + t4 * 2 + (e & 1)) * ROW);
                                float x = 0.0f;
                                for (int c = 0; c < p.head_dim; ++c) x += qr[c] * kr[c];
                                s[nb][e] = x;
                            }
                        }
                    }
                }
                // mask where some row of the tile does not see some key
                const bool whole = j0 >= all_lo && j0 + KG <= all_hi && j0 + KG <= k_hi;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (!whole) {
                            const int j = j0 + nb * 8 + t4 * 2 + (e & 1);
                            const RowRange &r = e < 2 ? r0 : r1;
                            if (j < r.lo || j >= r.hi || j >= k_hi) s[nb][e] = -INFINITY;
                        }
                    }
                }
                float x0 = m0, x1 = m1;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    x0 = fmaxf(x0, fmaxf(s[nb][0], s[nb][1]));
                    x1 = fmaxf(x1, fmaxf(s[nb][2], s[nb][3]));
                }
                x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, 1));
                x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, 1));
                x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, 2));
                x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, 2));
                // weights 2^(scale s - scale m), one rounding in the exponent; a row that has seen
                // nothing yet has the maximum -inf: subtract 0 instead. The products are rounded on their own:
                // contracted with the difference, a maximum that stays would rescale the row by its product's
                // rounding, 2^-24 of the exponent a tile, which adds up along a long context
                const float y0 = x0 == -INFINITY ? 0.0f : __fmul_rn(x0, p.scale_log2), y1 = x1 == -INFINITY ? 0.0f : __fmul_rn(x1, p.scale_log2);
                const float a0 = ex2(__fmul_rn(m0, p.scale_log2) - y0), a1 = ex2(__fmul_rn(m1, p.scale_log2) - y1);
                const float z0 = Weight<T>::LIFT - y0, z1 = Weight<T>::LIFT - y1;
                m0 = x0;
                m1 = x1;
                l0 *= a0;
                l1 *= a1;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    s[nb][0] = ex2(fmaf(s[nb][0], p.scale_log2, z0));
                    s[nb][1] = ex2(fmaf(s[nb][1], p.scale_log2, z0));
                    s[nb][2] = ex2(fmaf(s[nb][2], p.scale_log2, z1));
                    s[nb][3] = ex2(fmaf(s[nb][3], p.scale_log2, z1));
                    l0 += s[nb][0] + s[nb][1];
                    l1 += s[nb][2] + s[nb][3];
                }
                if (__any_sync(0xFFFFFFFFu, a0 != 1.0f || a1 != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        o[d][0] *= a0;
                        o[d][1] *= a0;
                        o[d][2] *= a1;
                        o[d][3] *= a1;
                    }
                }
                if constexpr (!C::F32) {
                    const uint32_t vl = vs_base + ((lane & 7) + ((lane >> 3) & 1) * 8) * ROW + ((lane >> 4) & 1) * 16;
#pragma unroll
                    for (int kb = 0; kb < KG / 16; ++kb) {
                        const uint32_t pa[4] = {pack2<T>(s[2 * kb][0], s[2 * kb][1]), pack2<T>(s[2 * kb][2], s[2 * kb][3]),
                                                pack2<T>(s[2 * kb + 1][0], s[2 * kb + 1][1]),
                                                pack2<T>(s[2 * kb + 1][2], s[2 * kb + 1][3])};
#pragma unroll
                        for (int d = 0; d < DB; d += 2) {
                            uint32_t vb[4];
                            ldsm4_t(vl + kb * 16 * ROW + d * 16, vb);
                            mma16<T>(o[d], pa, vb[0], vb[1]);
                            mma16<T>(o[d + 1], pa, vb[2], vb[3]);
                        }
                    }
                } else {
                    // the product's k index c stands for key 2 (c % 4) + c / 4 of its eight: the
                    // accumulator's own columns
                    uint32_t ph[NB][4], pl[NB][4];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        split_tf32(s[nb][0], ph[nb][0], pl[nb][0]);
                        split_tf32(s[nb][2], ph[nb][1], pl[nb][1]);
                        split_tf32(s[nb][1], ph[nb][2], pl[nb][2]);
                        split_tf32(s[nb][3], ph[nb][3], pl[nb][3]);
                    }
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f}, small[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const float *vr = reinterpret_cast<const float *>(st + (BN + kw + nb * 8 + 2 * t4) * ROW) + d * 8 + g4;
                            uint32_t h0, q0, h1, q1;
                            split_tf32(vr[0], h0, q0);
                            split_tf32(vr[ROW / 4], h1, q1);
                            mma8(small, pl[nb], h0, h1);
                            mma8(small, ph[nb], q0, q1);
                            mma8(t, ph[nb], h0, h1);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[d][e] += t[e] + small[e];
                    }
                }
            }
            }
            // the slot of this stage's own offsets is free
            if (tid < BN) sOff[(it % C::STAGES) * BN + tid] = offset_of(j_next, page_next);
        }
        cp_async_wait<0>();
        // The piece is computed again, row by row and only with the keys that a row sees, if it met a page
        // number out of range or if NaN came out that need not belong there (the row's sum is none): a
        // weight 0 of a key that a row does not see times a value that is not finite, or the split of an
        // infinite value. A single token's rows all see the same keys: there the 16-bit and the plain form
        // cannot have made one. (Looking at each stage cost 2 % of 64 x 8192 in bf16.)
        bool again = bad_page;
        const bool partly = rows > p.group;
        if constexpr (SIMT > 0) {
            if (partly) {
#pragma unroll
                for (int r = 0; r < SR; ++r) {
#pragma unroll
                    for (int i = 0; i < CL; ++i) again = again || (so[r][i] != so[r][i] && sl_[r] == sl_[r]);
                }
            }
        } else if (C::F32 || partly) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                again = again || (l0 == l0 && (o[d][0] != o[d][0] || o[d][1] != o[d][1]));
                again = again || (l1 == l1 && (o[d][2] != o[d][2] || o[d][3] != o[d][3]));
            }
        }
        again = __syncthreads_or(again);

        // ---- the warps' partial results, then the splits' ----
        float *red = reinterpret_cast<float *>(ring);
        float *sm = red + WN * R * C::ORED, *sl = sm + WN * R;
        if (again) {  // as the first slice's result, the others empty
            for (int r = warp; r < R; r += WM * WN) {
                RowSum<DP / 32> x;
                const RowRange see = row_range(p, seq, row0 + r);
                x.template over_keys<T>(p, b, kh, row0 + r < rows ? q_ptr(row0 + r) : nullptr, max(see.lo, k_lo), min(see.hi, k_hi), lane);
#pragma unroll 1
                for (int s = 0; s < WN; ++s) {
#pragma unroll
                    for (int c = 0; c < DP / 32; ++c) red[(s * R + r) * C::ORED + lane + 32 * c] = s ? 0.0f : x.o[c];
                    if (lane == 0) {
                        sm[s * R + r] = s ? -INFINITY : x.m;
                        sl[s * R + r] = s ? 0.0f : x.l;
                    }
                }
            }
            __syncthreads();
        } else if constexpr (SIMT > 0) {
#pragma unroll
            for (int r = 0; r < SR; ++r) {
#pragma unroll
                for (int d = 1; d < KW; d <<= 1) sl_[r] += __shfl_xor_sync(0xFFFFFFFFu, sl_[r], d);
#pragma unroll
                for (int i = 0; i < CL; ++i) red[(wn * R + r) * C::ORED + lane * CL + i] = so[r][i];
                if (lane == 0) {
                    sm[wn * R + r] = __fmul_rn(sm_[r], p.scale_log2);
                    sl[wn * R + r] = sl_[r];
                }
            }
            __syncthreads();
        } else {
            l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 1);
            l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 1);
            l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 2);
            l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 2);
            const int ra = wn * R + 16 * wm + g4;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                *reinterpret_cast<float2 *>(red + ra * C::ORED + d * 8 + t4 * 2) = make_float2(o[d][0], o[d][1]);
                *reinterpret_cast<float2 *>(red + (ra + 8) * C::ORED + d * 8 + t4 * 2) = make_float2(o[d][2], o[d][3]);
            }
            if (t4 == 0) {
                sm[ra] = __fmul_rn(m0, p.scale_log2);
                sm[ra + 8] = __fmul_rn(m1, p.scale_log2);
                sl[ra] = l0;
                sl[ra + 8] = l1;
            }
            __syncthreads();
        }
        const int quads = p.head_dim / 4;
        const int live = min(R, rows - row0);
        auto warps_sum = [&](int r, int c, float &m, float &l) {
            m = sm[r];
#pragma unroll
            for (int w = 1; w < WN; ++w) m = fmaxf(m, sm[w * R + r]);
            l = 0.0f;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WN; ++w) {
                const float f = m == -INFINITY ? 0.0f : ex2(sm[w * R + r] - m);
                const float4 x = *reinterpret_cast<const float4 *>(red + (w * R + r) * C::ORED + c * 4);
                l += f * sl[w * R + r];
                a.x += f * x.x;
                a.y += f * x.y;
                a.z += f * x.z;
                a.w += f * x.w;
            }
            return a;
        };
        auto put = [&](int r, int c, float4 a, float l) {
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            const int row = row0 + r, i = row / p.group, h = kh * p.group + row % p.group;
            T *out = static_cast<T *>(p.out) + (long long)(seq.start + i) * p.o_ts + (long long)h * p.o_hs + c * 4;
            Pack<4, T> v;
            v.e[0] = from_f<T>(a.x * inv);
            v.e[1] = from_f<T>(a.y * inv);
            v.e[2] = from_f<T>(a.z * inv);
            v.e[3] = from_f<T>(a.w * inv);
            v.store(out);
        };
        if (EVEN || p.splits == 1) {
            for (int x = tid; x < live * quads; x += C::THREADS) {
                const int r = x / quads, c = x - r * quads;
                float m, l;
                const float4 a = warps_sum(r, c, m, l);
                if (!EVEN || slot < 0) {
                    put(r, c, a, l);
                } else {
                    const long long at = ((long long)blockIdx.x * 2 + slot) * R + r;
                    *reinterpret_cast<float4 *>(p.part + at * p.head_dim + c * 4) = a;
                    if (c == 0) p.part_ml[at] = make_float2(m, l);
                }
            }
        } else {
            // this CTA's sum over its first warp slice's rows (each quad read and written by one thread)
            for (int x = tid; x < live * quads; x += C::THREADS) {
                const int r = x / quads, c = x - r * quads;
                float m, l;
                const float4 a = warps_sum(r, c, m, l);
                *reinterpret_cast<float4 *>(red + r * C::ORED + c * 4) = a;
            }
            __syncthreads();
            for (int r = tid; r < live; r += C::THREADS) {
                float m = sm[r], l = 0.0f;
#pragma unroll
                for (int w = 1; w < WN; ++w) m = fmaxf(m, sm[w * R + r]);
#pragma unroll
                for (int w = 0; w < WN; ++w) l += m == -INFINITY ? 0.0f : ex2(sm[w * R + r] - m) * sl[w * R + r];
                sm[r] = m;
                sl[r] = l;
            }
            cluster_barrier();
            const uint32_t a_red = smem_u32(red), a_m = smem_u32(sm), a_l = smem_u32(sl);
            for (int x = split * C::THREADS + tid; x < live * quads; x += p.splits * C::THREADS) {
                const int r = x / quads, c = x - r * quads;
                // every rank's loads in flight together
                float mk[MAX_CLUSTER], lk[MAX_CLUSTER];
                float4 vk[MAX_CLUSTER];
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) {
                    if (k >= p.splits) break;
                    mk[k] = ld_cluster(a_m + r * 4, k);
                    lk[k] = ld_cluster(a_l + r * 4, k);
                    vk[k] = ld_cluster4(a_red + (r * C::ORED + c * 4) * 4, k);
                }
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) m = k < p.splits ? fmaxf(m, mk[k]) : m;
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) {
                    if (k >= p.splits) break;
                    const float f = m == -INFINITY ? 0.0f : ex2(mk[k] - m);
                    l += f * lk[k];
                    a.x += f * vk[k].x;
                    a.y += f * vk[k].y;
                    a.z += f * vk[k].z;
                    a.w += f * vk[k].w;
                }
                put(r, c, a, l);
            }
            cluster_barrier();  // every partial read before the next tile or the exit reuses it
        }
        __syncthreads();
    };
    // channels past the head width: zero in every stage, never loaded over; the reduction at a piece's
    // end does write over them
    auto zero_padding = [&]() {
        if (chunks == CPR) return;
        const int pad = CPR - chunks;
        for (int x = tid; x < C::STAGES * 2 * BN * pad; x += C::THREADS) {
            const int r = x / pad, c = chunks + x % pad;
            *reinterpret_cast<uint4 *>(ring + (size_t)r * ROW + c * 16) = make_uint4(0, 0, 0, 0);
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
            zero_outside<T>(p, (int)blockIdx.x, (int)gridDim.x, warp - 1, WM * WN - 1, lane);
        }
        __syncthreads();
        asm volatile("griddepcontrol.launch_dependents;");  // the kernel that adds the pieces waits on its own
        Walk walk = stretch;
        Item w;
        CutUnit cut{0, 0, 0, 0};
        while (next_item<R, BN>(p, walk, w)) {
            zero_padding();
            if (w.slot == 1) cut = cut_of<R, BN>(p, walk, w);
            piece(w.b, w.h, w.seq, w.row0, w.lo, w.hi, w.slot);
        }
        if (tid == 0) p.cut[blockIdx.x] = cut;
    } else {
        // block -> (sequence, key head, row tile, split); the key heads of a token row, which lie side
        // by side in memory, run side by side
        unsigned u = blockIdx.x;
        const int kh = (int)(u % (unsigned)p.kv_heads);
        u /= (unsigned)p.kv_heads;
        const int tile0 = p.row_tiles - 1 - (int)(u % (unsigned)p.row_tiles);  // longest rows first
        const int b = (int)(u / (unsigned)p.row_tiles);
        const Sequence seq = load_sequence(p, b);
        if (tid == 0) check_sequence(p, b);
        zero_outside<T>(p, (int)(blockIdx.y * gridDim.x + blockIdx.x), (int)(gridDim.x * gridDim.y), warp, WM * WN, lane);
        for (int tile = tile0; tile * R < seq.nq * p.group; tile += p.row_tiles) {
            const RowRange z = row_range(p, seq, min(tile * R + R, seq.nq * p.group) - 1);
            const int lo = row_range(p, seq, tile * R).lo & ~15, hi = max(z.hi, 0);
            // this split's part of the keys that some row of the tile sees
            const int per = (max(hi - lo, 0) + p.splits * 16 - 1) / (p.splits * 16) * 16;
            const int k_lo = lo + split * per;
            zero_padding();
            piece(b, kh, seq, tile * R, k_lo, min(hi, k_lo + per), -1);
        }
    }
}

}  // namespace paged
}  // namespace mgc
