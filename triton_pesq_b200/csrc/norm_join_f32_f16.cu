// The join's kernels for a stream of float and blocks of __half.
#include "norm_join_launch.cuh"

namespace pesq {
namespace njoin {
template cudaError_t launch<float, __half>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace njoin
}  // namespace pesq
