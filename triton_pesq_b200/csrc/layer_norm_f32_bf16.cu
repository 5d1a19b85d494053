// The layer norm's kernels for inputs of float and results of __nv_bfloat16.
#include "layer_norm_launch.cuh"

namespace pesq {
namespace lnorm {
template cudaError_t launch<float, __nv_bfloat16>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace lnorm
}  // namespace pesq
