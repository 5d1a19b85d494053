// The linear attention's forward kernels for __nv_bfloat16.
#include "linear_attention_launch.cuh"

namespace pesq {
namespace lattn {
template cudaError_t forward_of<__nv_bfloat16>(const Args&, const Geometry&, Kind, cudaStream_t);
}  // namespace lattn
}  // namespace pesq
