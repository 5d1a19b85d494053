// Instantiation of the gated scan kernels for one element type (one
// translation unit each, so that they compile in parallel).
#pragma once

#include "gated_scan.cuh"

namespace pesq {
namespace gscan {

template <class T, int V, int L>
cudaError_t launch_vl(const Args& p, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  const dim3 block(32, g.warps);
  const unsigned grid = (unsigned)g.blocks;
  if (!backward) {
    if (mask)
      forward_kernel<T, V, L, true><<<grid, block, 0, s>>>(p);
    else
      forward_kernel<T, V, L, false><<<grid, block, 0, s>>>(p);
  } else {
    if (mask)
      backward_kernel<T, V, L, true><<<grid, block, 0, s>>>(p);
    else
      backward_kernel<T, V, L, false><<<grid, block, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <class T>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  if (g.steps_per_thread == 1)
    return g.vec == 2 ? launch_vl<T, 2, 1>(p, g, backward, mask, s) : launch_vl<T, 1, 1>(p, g, backward, mask, s);
  return g.vec == 2 ? launch_vl<T, 2, kSteps>(p, g, backward, mask, s)
                    : launch_vl<T, 1, kSteps>(p, g, backward, mask, s);
}

}  // namespace gscan
}  // namespace pesq
