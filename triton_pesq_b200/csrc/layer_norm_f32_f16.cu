// The layer norm's kernels for inputs of float and results of __half.
#include "layer_norm_launch.cuh"

namespace pesq {
namespace lnorm {
template cudaError_t launch<float, __half>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace lnorm
}  // namespace pesq
