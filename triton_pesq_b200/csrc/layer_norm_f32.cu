// The layer norm's kernels for inputs of float and results of float.
#include "layer_norm_launch.cuh"

namespace pesq {
namespace lnorm {
template cudaError_t launch<float, float>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace lnorm
}  // namespace pesq
