// Instantiation of the gated scan kernels for one element type (one
// translation unit each, so that they compile in parallel).
#pragma once

#include "gated_scan.cuh"

namespace pesq {
namespace gscan {

template <class T, int V, int L, bool kMask>
cudaError_t launch_vl(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  const int warps = g.strips < kStrips ? g.strips : kStrips;
  const dim3 grid((unsigned)(g.ctiles * ((g.strips + warps - 1) / warps)), (unsigned)p.batch), block(32, warps);
  if (g.strips > 1) {
    if (backward)
      backward_maps_kernel<T, V, L, kMask><<<grid, block, 0, s>>>(p);
    else
      forward_maps_kernel<T, V, L, kMask><<<grid, block, 0, s>>>(p);
  }
  if (backward)
    backward_kernel<T, V, L, kMask><<<grid, block, 0, s>>>(p);
  else
    forward_kernel<T, V, L, kMask><<<grid, block, 0, s>>>(p);
  return cudaGetLastError();
}

template <class T, int V>
cudaError_t launch_v(const Args& p, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  if (g.chunk == 1)
    return mask ? launch_vl<T, V, 1, true>(p, g, backward, s) : launch_vl<T, V, 1, false>(p, g, backward, s);
  return mask ? launch_vl<T, V, kChunk, true>(p, g, backward, s) : launch_vl<T, V, kChunk, false>(p, g, backward, s);
}

template <class T>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  return g.vec == 2 ? launch_v<T, 2>(p, g, backward, mask, s) : launch_v<T, 1>(p, g, backward, mask, s);
}

}  // namespace gscan
}  // namespace pesq
