// Launches of the attention over codes, for the files that compile its kernels.
#pragma once

#include "quantized_attention.cuh"

namespace mgc {
namespace paged {

template <typename C> inline int launch_quantized(const QuantParams &p, const QuantPlan &s, C, cudaStream_t stream) {
    if (s.even) {
        auto kernel = quantized_attention_kernel<C, WORK_EVEN>;
        MGC_CHECK(raise_smem_ceiling((const void *)kernel));
        kernel<<<(unsigned)s.ctas, C::THREADS, C::SMEM, stream>>>(p);
        MGC_CHECK(check_launch("quantized_attention_kernel"));
        return launch_after(paged_combine_units_kernel<typename C::T, C::R>, dim3((unsigned)s.ctas, (unsigned)s.live_rows), p.a,
                            s.interleaved ? p.a.kv_heads : 1, stream);
    }
    const unsigned units = (unsigned)(p.a.batch.batch * p.a.kv_heads * s.row_tiles);
    if (s.splits == 1) {
        auto kernel = quantized_attention_kernel<C, WORK_UNIT>;
        MGC_CHECK(raise_smem_ceiling((const void *)kernel));
        kernel<<<units, C::THREADS, C::SMEM, stream>>>(p);
        return check_launch("quantized_attention_kernel");
    }
    auto kernel = quantized_attention_kernel<C, WORK_CLUSTER>;
    MGC_CHECK(raise_smem_ceiling((const void *)kernel));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(units, (unsigned)s.splits);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
    attr[0].val.clusterDim.y = (unsigned)s.splits;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MGC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return MGC_CUDA_OK;
}

template <int BITS> int launch_codes(const QuantParams &p, const QuantPlan &s, int64_t dtype, const mgc_cuda_quantized &z, cudaStream_t stream) {
    return with_config<BITS>(dtype, z, p.a.head_dim, s.nb, [&](auto config) { return launch_quantized(p, s, config, stream); });
}

}  // namespace paged
}  // namespace mgc
