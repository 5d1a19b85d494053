// The join's kernels for a stream of __half and blocks of __half.
#include "norm_join_launch.cuh"

namespace pesq {
namespace njoin {
template cudaError_t launch<__half, __half>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace njoin
}  // namespace pesq
