// Gated scan kernels for f16 streams.
#include "gated_scan_launch.cuh"

namespace pesq {
namespace gscan {
template cudaError_t launch<__half>(const Args&, const Maps&, const Geometry&, bool, bool, cudaStream_t);
}  // namespace gscan
}  // namespace pesq
