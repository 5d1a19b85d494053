// The linear attention's backward kernels for float.
#include "linear_attention_launch.cuh"

namespace pesq {
namespace lattn {
template cudaError_t backward_of<float>(const Args&, const Geometry&, cudaStream_t);
}  // namespace lattn
}  // namespace pesq
