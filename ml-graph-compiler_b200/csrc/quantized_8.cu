// The kernels of the attention over codes of 8 bits.
#include <string.h>

#include "quantized_launch.cuh"

namespace mgc {
namespace paged {

template int launch_codes<8>(const QuantParams &, const QuantPlan &, int64_t, const mgc_cuda_quantized &, cudaStream_t);

}  // namespace paged
}  // namespace mgc
