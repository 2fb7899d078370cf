// Entry points of the quantised paged cache and of the append with head norms.
#include <string.h>

#include "kv_append_heads.cuh"
#include "kv_read.cuh"
#include "quantized_attention.cuh"

extern "C" {

int mgc_cuda_kv_append_heads(const mgc_cuda_kv_append_heads_args *args, void *stream) {
    mgc::last_error().clear();
    if (!args) return mgc::fail(MGC_CUDA_BAD_ARGUMENT, "mgc_cuda_kv_append_heads: args is NULL");
    return mgc::paged::append_heads(*args, (cudaStream_t)stream);
}

int mgc_cuda_kv_read(const mgc_cuda_kv_read_args *args, void *stream) {
    mgc::last_error().clear();
    if (!args) return mgc::fail(MGC_CUDA_BAD_ARGUMENT, "mgc_cuda_kv_read: args is NULL");
    return mgc::paged::read_back(*args, (cudaStream_t)stream);
}

int mgc_cuda_paged_attention_quantized(const mgc_cuda_paged_attention_quantized_args *args, void *stream) {
    mgc::last_error().clear();
    if (!args) return mgc::fail(MGC_CUDA_BAD_ARGUMENT, "mgc_cuda_paged_attention_quantized: args is NULL");
    return mgc::paged::attend_quantized(*args, (cudaStream_t)stream);
}

int64_t mgc_cuda_paged_attention_quantized_workspace(const mgc_cuda_paged_attention_quantized_args *args) {
    mgc::last_error().clear();
    if (!args) return mgc::fail(MGC_CUDA_BAD_ARGUMENT, "mgc_cuda_paged_attention_quantized_workspace: args is NULL"), -1;
    return mgc::paged::attend_quantized_workspace(*args);
}

}  // extern "C"
