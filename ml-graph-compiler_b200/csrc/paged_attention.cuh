// Attention of new tokens over a paged cache: the kernel for unaligned operands, the choice of
// kernel and the launch.
#pragma once

#include "paged_umma.cuh"

namespace mgc {
namespace paged {

// One warp per (token, query head), lane l holding channels l, l + 32, ...: what the tiled kernels
// do not take (head widths that are no multiple of 16 bytes, unaligned rows).
template <typename T>
__global__ void __launch_bounds__(128) paged_attention_row_kernel(const __grid_constant__ AttendParams p) {
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
    const int n = __ldg(p.batch.kv_lens + b);
    int lo, hi;
    visible(p, min(n, p.max_positions), n - (end - t), lo, hi);
    RowSum<C> x;
    x.over_keys<T>(p, b, h / p.group, static_cast<const T *>(p.q) + t * p.q_ts + h * p.q_hs, lo, hi, lane);
    const float inv = x.l > 0.0f ? 1.0f / x.l : 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int d = lane + 32 * c;
        if (d < p.head_dim) out[d] = from_f<T>(x.o[c] * inv);
    }
}

// ---- host side ---------------------------------------------------------------------------------
// How a call runs: which kernel, its row tile and how its keys are shared out.
struct Plan {
    bool mma = false, umma = false, even = false;
    int wm = 1;         // 16-row warps of a row tile
    int simt = 0;       // rows of the plain fp32 form (0: matrix instructions)
    int row_tiles = 1, splits = 1;
    int unit_rows = 0, ctas = 0;  // even shares: rows of a unit, CTAs
    bool interleaved = false;
    int live_rows = 1;  // of a unit, going by max_q
    int64_t workspace = 0;
};

constexpr int MIN_SPLIT_KEYS = 128;  // below this a split's start and merge outweigh its loads

// CTAs of the tiled kernel (128 threads) that an SM holds by its shared memory. Registers are not counted:
// the even-share kernels of 16-bit types with 64 channels and more than 16 rows (168 registers), and of fp32
// with 96 channels and 8 rows, hold 3 where this says 4, so their last shares run in a second round.
inline int ctas_per_sm(int64_t dtype, int64_t head_dim, int wm, int simt) {
    const int dp = head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : head_dim <= 96 ? 96 : head_dim <= 128 ? 128 : 256;
    const bool f32 = dtype == MGC_F32;
    const int keys = !f32 ? 64 : !simt ? 32 : dp <= 32 ? 128 : dp <= 64 ? 64 : 32;
    const int row = dp * (f32 ? 4 : 2) + 16, ring = (dp > 128 || simt ? 2 : 3) * 2 * keys * row;
    const int bytes = ring + (!f32 && dp <= 128 ? 0 : (simt ? simt : 16 * wm) * row) + 3 * keys * 8 + 1024;
    const int fit = 232448 / bytes;
    return fit < 1 ? 1 : fit > 4 ? 4 : fit;
}

inline Plan plan_of(const mgc_cuda_paged_attention_args &a) {
    const mgc_cuda_paged &c = a.paged;
    Plan s;
    const int es = elem_size(c.dtype), chunk = 16 / es;
    auto rows16 = [&](const void *q, int64_t x, int64_t y, int64_t z) {
        return aligned(q, 16) && x * es % 16 == 0 && y * es % 16 == 0 && z * es % 16 == 0;
    };
    const int64_t group = a.q_heads / c.kv_heads;
    // 16-byte rows everywhere, and a sequence's rows (with those of its last tile) counted in 32 bits;
    // anything else takes the row kernel
    s.mma = c.head_dim % chunk == 0 && c.tokens * group < 0x80000000ll - 256 && rows16(c.k, c.page_stride, c.token_stride, c.head_stride) &&
            rows16(c.v, 0, 0, 0) && rows16(a.q, a.q_token_stride, a.q_head_stride, 0) &&
            rows16(a.out, a.o_token_stride, a.o_head_stride, 0);
    if (!s.mma) return s;
    int64_t max_q = a.max_q < 1 ? 1 : a.max_q > c.tokens ? c.tokens : a.max_q;
    const int64_t rows = max_q * group;
    auto even_shares = [&](int unit_rows, int ctas) {
        s.even = true;
        s.unit_rows = unit_rows;
        s.live_rows = (int)(rows < unit_rows ? rows : unit_rows);
        s.ctas = ctas;
        if (!s.umma && ctas >= c.kv_heads && ctas / c.kv_heads * c.kv_heads * 20 >= ctas * 19) {
            s.interleaved = true;
            s.ctas = (int)(ctas / c.kv_heads * c.kv_heads);
        }
        s.workspace = (int64_t)s.ctas * (2 * unit_rows * (c.head_dim * 4 + 8) + (int64_t)sizeof(CutUnit));
    };
    if (rows > 64 && umma_fits(c) && c.batch * ceil_div(rows, 256) < 0x7FFFFFFF) {
        s.umma = true;
        even_shares(256, sm_count());
        return s;
    }
    s.wm = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    // fp32 rows cost the FMA units ~200 instructions per 32 keys each; the split products cost ~3300
    // for 16 rows, used or not
    if (c.dtype == MGC_F32 && rows <= 8 && c.head_dim <= 128) s.simt = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
    s.unit_rows = s.simt ? s.simt : 16 * s.wm;
    s.row_tiles = (int)ceil_div(rows, s.unit_rows);
    const int64_t units = c.batch * c.kv_heads * s.row_tiles;
    int64_t most = a.max_kv;
    if (a.window > 0 && a.window + max_q < most) most = a.window + max_q;
    // CTAs that fit the GPU at once, going by shared memory
    const int64_t slots = (int64_t)sm_count() * ctas_per_sm(c.dtype, c.head_dim, s.wm, s.simt);
    int64_t splits = slots / units;
    if (splits > most / MIN_SPLIT_KEYS) splits = most / MIN_SPLIT_KEYS;
    if (splits < 1) splits = 1;
    // A cluster needs no second kernel (~1000 keys' worth of time); even shares leave no SM idle when
    // sequences differ or 8 parts are too few.
    const int64_t in_cluster = most / (splits < MAX_CLUSTER ? splits : MAX_CLUSTER), even = most * units / slots;
    if (in_cluster > even + 1024 || (units * 2 > slots && c.batch > 1)) {
        even_shares(s.unit_rows, (int)slots);
        return s;
    }
    if (splits > MAX_CLUSTER) splits = MAX_CLUSTER;
    s.splits = (int)splits;
    return s;
}

inline int64_t attend_workspace(const mgc_cuda_paged_attention_args &a) {
    if (check_attend(a, "mgc_cuda_paged_attention_workspace") != MGC_CUDA_OK) return -1;
    return a.paged.tokens == 0 || a.paged.batch == 0 ? 0 : plan_of(a).workspace;
}

template <typename T, typename O> inline int launch_umma(const AttendParams &p, const mgc_cuda_paged &c, int ctas, cudaStream_t stream) {
    UmmaMaps maps;
    memset(&maps, 0, sizeof maps);
    if (!umma_maps(&maps, c)) return fail(MGC_CUDA_UNSUPPORTED, "mgc_cuda_paged_attention: tensor map encoding failed");
    auto go = [&](auto kernel, uint32_t smem, int threads) -> int {
        MGC_CHECK(raise_smem_ceiling((const void *)kernel));
        kernel<<<(unsigned)ctas, threads, smem, stream>>>(p, maps);
        return check_launch("paged_attention_umma_kernel");
    };
    MGC_CHECK(p.head_dim <= 64 ? go(paged_attention_umma_kernel<T, 64, O>, UmmaConfig<64>::SMEM, UmmaConfig<64>::THREADS)
                               : go(paged_attention_umma_kernel<T, 128, O>, UmmaConfig<128>::SMEM, UmmaConfig<128>::THREADS));
    return launch_after(paged_combine_units_kernel<O, 256>, dim3((unsigned)ctas, 32), p, 1, stream);
}

template <typename T, int DP, int WM, int WN, int SIMT> inline int launch_mma(const AttendParams &p, const Plan &s, cudaStream_t stream) {
    using C = MmaConfig<T, DP, WM, WN, SIMT>;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    if (s.even) {
        auto kernel = paged_attention_mma_kernel<T, DP, WM, WN, SIMT, true>;
        MGC_CHECK(raise_smem_ceiling((const void *)kernel));
        cfg.gridDim = dim3((unsigned)s.ctas);
        MGC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
        return launch_after(paged_combine_units_kernel<T, C::R>, dim3((unsigned)s.ctas, (unsigned)s.live_rows), p, s.interleaved ? p.kv_heads : 1,
                            stream);
    }
    auto kernel = paged_attention_mma_kernel<T, DP, WM, WN, SIMT, false>;
    MGC_CHECK(raise_smem_ceiling((const void *)kernel));
    cfg.gridDim = dim3((unsigned)(p.batch.batch * p.kv_heads * p.row_tiles), (unsigned)p.splits);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
    attr[0].val.clusterDim.y = (unsigned)p.splits;
    cfg.attrs = attr;
    cfg.numAttrs = p.splits > 1 ? 1 : 0;
    MGC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return MGC_CUDA_OK;
}

template <typename T, int DP> inline int launch_mma_rows(const AttendParams &p, const Plan &s, cudaStream_t stream) {
    if constexpr (sizeof(T) == 4 && DP <= 128) {
        if (s.simt == 1) return launch_mma<T, DP, 1, 4, 1>(p, s, stream);
        if (s.simt == 2) return launch_mma<T, DP, 1, 4, 2>(p, s, stream);
        if (s.simt == 4) return launch_mma<T, DP, 1, 4, 4>(p, s, stream);
        if (s.simt == 8) return launch_mma<T, DP, 1, 4, 8>(p, s, stream);
    }
    if (s.wm == 1) return launch_mma<T, DP, 1, 4, 0>(p, s, stream);
    if (s.wm == 2) return launch_mma<T, DP, 2, 2, 0>(p, s, stream);
    return launch_mma<T, DP, 4, 1, 0>(p, s, stream);
}

// Head widths are padded to the next of these (zero channels).
template <typename T> inline int launch_mma_width(const AttendParams &p, const Plan &s, cudaStream_t stream) {
    if (p.head_dim <= 32) return launch_mma_rows<T, 32>(p, s, stream);
    if (p.head_dim <= 64) return launch_mma_rows<T, 64>(p, s, stream);
    if (p.head_dim <= 96) return launch_mma_rows<T, 96>(p, s, stream);
    if (p.head_dim <= 128) return launch_mma_rows<T, 128>(p, s, stream);
    return launch_mma_rows<T, 256>(p, s, stream);
}

int attend(const mgc_cuda_paged_attention_args &a, int64_t q_dtype, cudaStream_t stream) {
    const char *what = "mgc_cuda_paged_attention";
    const mgc_cuda_paged &c = a.paged;
    MGC_CHECK(check_attend(a, what));
    if (c.tokens == 0 || c.batch == 0) return MGC_CUDA_OK;
    AttendParams p = attend_params(a);
    const Plan s = plan_of(a);
    if (q_dtype != c.dtype && !(s.umma && c.dtype == MGC_F16 && q_dtype == MGC_BF16))
        return fail(MGC_CUDA_UNSUPPORTED, "%s: queries of type %d over pages of type %d", what, (int)q_dtype, (int)c.dtype);
    p.row_tiles = s.row_tiles; p.splits = s.splits; p.interleaved = s.interleaved;
    if (s.workspace) {
        if (!a.workspace || a.workspace_bytes < s.workspace || !aligned(a.workspace, 16))
            return fail(MGC_CUDA_NEEDS_WORKSPACE, "%s: needs %lld bytes of workspace (16-byte aligned), got %lld", what,
                        (long long)s.workspace, (long long)(a.workspace ? a.workspace_bytes : 0));
        p.part = static_cast<float *>(a.workspace);
        const int64_t rows = (int64_t)s.ctas * 2 * s.unit_rows;
        p.part_ml = reinterpret_cast<float2 *>(p.part + rows * p.head_dim);
        p.cut = reinterpret_cast<CutUnit *>(p.part_ml + rows);
    }
    if (s.mma) {
        const int64_t units = c.batch * c.kv_heads * s.row_tiles;
        if (units > 0x7FFFFFFF) return fail(MGC_CUDA_UNSUPPORTED, "%s: %lld row tiles", what, (long long)units);
        if (s.umma)
            return c.dtype != MGC_F16      ? launch_umma<__nv_bfloat16, __nv_bfloat16>(p, c, s.ctas, stream)
                   : q_dtype != MGC_F16 ? launch_umma<__half, __nv_bfloat16>(p, c, s.ctas, stream)
                                        : launch_umma<__half, __half>(p, c, s.ctas, stream);
        if (c.dtype == MGC_F32) return launch_mma_width<float>(p, s, stream);
        if (c.dtype == MGC_F16) return launch_mma_width<__half>(p, s, stream);
        return launch_mma_width<__nv_bfloat16>(p, s, stream);
    }
    const dim3 grid((unsigned)p.tokens, (unsigned)ceil_div(p.q_heads, 4));
    if (c.dtype == MGC_F32) paged_attention_row_kernel<float><<<grid, 128, 0, stream>>>(p);
    else if (c.dtype == MGC_F16) paged_attention_row_kernel<__half><<<grid, 128, 0, stream>>>(p);
    else paged_attention_row_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(p);
    return check_launch("paged_attention_row_kernel");
}

}  // namespace paged
}  // namespace mgc
