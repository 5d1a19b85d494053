// Gated scan kernels for bf16 streams.
#include "gated_scan_launch.cuh"

namespace pesq {
namespace gscan {
template cudaError_t launch<__nv_bfloat16>(const Args&, const Maps&, const Geometry&, bool, bool, cudaStream_t);
}  // namespace gscan
}  // namespace pesq
