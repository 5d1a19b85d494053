// The linear attention's forward kernels for __half.
#include "linear_attention_launch.cuh"

namespace pesq {
namespace lattn {
template cudaError_t forward_of<__half>(const Args&, const Geometry&, Kind, cudaStream_t);
}  // namespace lattn
}  // namespace pesq
