// Entry points of the paged-cache operators (mgc_cuda_kv_append, mgc_cuda_paged_attention).
#include "kv_append.cuh"
#include "paged_attention.cuh"

extern "C" {

int mgc_cuda_kv_append(const mgc_cuda_kv_append_args *args, void *stream) {
    mgc::last_error().clear();
    if (!args) return mgc::fail(MGC_CUDA_BAD_ARGUMENT, "mgc_cuda_kv_append: args is NULL");
    return mgc::paged::append(*args, (cudaStream_t)stream);
}

int mgc_cuda_paged_attention(const mgc_cuda_paged_attention_args *args, void *stream) {
    mgc::last_error().clear();
    if (!args) return mgc::fail(MGC_CUDA_BAD_ARGUMENT, "mgc_cuda_paged_attention: args is NULL");
    return mgc::paged::attend(*args, (cudaStream_t)stream);
}

int64_t mgc_cuda_paged_attention_workspace(const mgc_cuda_paged_attention_args *args) {
    mgc::last_error().clear();
    if (!args) return mgc::fail(MGC_CUDA_BAD_ARGUMENT, "mgc_cuda_paged_attention_workspace: args is NULL"), -1;
    return mgc::paged::attend_workspace(*args);
}

}  // extern "C"
