// The linear attention's backward kernels for __nv_bfloat16.
#include "linear_attention_launch.cuh"

namespace pesq {
namespace lattn {
template cudaError_t backward_of<__nv_bfloat16>(const Args&, const Geometry&, cudaStream_t);
}  // namespace lattn
}  // namespace pesq
