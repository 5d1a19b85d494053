// Gated scan kernels for f32 streams.
#include "gated_scan_launch.cuh"

namespace pesq {
namespace gscan {
template cudaError_t launch<float>(const Args&, const Maps&, const Geometry&, bool, bool, cudaStream_t);
}  // namespace gscan
}  // namespace pesq
