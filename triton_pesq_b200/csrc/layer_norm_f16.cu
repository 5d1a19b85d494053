// The layer norm's kernels for inputs of __half and results of __half.
#include "layer_norm_launch.cuh"

namespace pesq {
namespace lnorm {
template cudaError_t launch<__half, __half>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace lnorm
}  // namespace pesq
