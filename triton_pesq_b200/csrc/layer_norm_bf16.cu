// The layer norm's kernels for inputs of __nv_bfloat16 and results of __nv_bfloat16.
#include "layer_norm_launch.cuh"

namespace pesq {
namespace lnorm {
template cudaError_t launch<__nv_bfloat16, __nv_bfloat16>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace lnorm
}  // namespace pesq
