// The linear attention's forward kernels for float.
#include "linear_attention_launch.cuh"

namespace pesq {
namespace lattn {
template cudaError_t forward_of<float>(const Args&, const Geometry&, Kind, cudaStream_t);
}  // namespace lattn
}  // namespace pesq
