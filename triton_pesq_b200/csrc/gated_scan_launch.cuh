// Instantiation of the gated scan kernels for one element type (one
// translation unit each, so that they compile in parallel).
#pragma once

#include "gated_scan.cuh"

namespace pesq {
namespace gscan {

template <class K>
cudaError_t start(K kernel, const Args& p, const Maps& m, const Geometry& g, size_t warp_smem, cudaStream_t s) {
  const int warps = g.strips < kStrips ? g.strips : kStrips;
  const size_t smem = warps * warp_smem;
  if (smem > 40 << 10) {  // beside the static part, more than a kernel gets without asking
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  const dim3 grid((unsigned)(g.ctiles * ((g.strips + warps - 1) / warps)), (unsigned)p.batch);
  kernel<<<grid, dim3(32, warps), smem, s>>>(p, m);
  return cudaGetLastError();
}

template <class T, int V, int L, bool kMask, bool kBulk>
cudaError_t launch_vl(const Args& p, const Maps& m, const Geometry& g, bool backward, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (!backward) {
    const size_t smem = kBulk ? Ring<T, 3, false>::kBytes : 0;
    if (g.strips > 1) e = start(forward_maps_kernel<T, V, L, kMask, kBulk>, p, m, g, smem, s);
    return e != cudaSuccess ? e : start(forward_kernel<T, V, L, kMask, kBulk>, p, m, g, smem, s);
  }
  if (g.strips > 1)
    e = start(backward_maps_kernel<T, V, L, kMask, kBulk>, p, m, g, kBulk ? Ring<T, 2, false>::kBytes : 0, s);
  return e != cudaSuccess
             ? e
             : start(backward_kernel<T, V, L, kMask, kBulk>, p, m, g, kBulk ? Ring<T, 4, true>::kBytes : 0, s);
}

template <class T, int V, int L, bool kBulk>
cudaError_t launch_m(const Args& p, const Maps& m, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  return mask ? launch_vl<T, V, L, true, kBulk>(p, m, g, backward, s)
              : launch_vl<T, V, L, false, kBulk>(p, m, g, backward, s);
}

template <class T>
cudaError_t launch(const Args& p, const Maps& m, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  if (g.bulk) return launch_m<T, 2, kChunk, true>(p, m, g, backward, mask, s);
  if (g.chunk == 1)
    return g.vec == 2 ? launch_m<T, 2, 1, false>(p, m, g, backward, mask, s)
                      : launch_m<T, 1, 1, false>(p, m, g, backward, mask, s);
  return g.vec == 2 ? launch_m<T, 2, kChunk, false>(p, m, g, backward, mask, s)
                    : launch_m<T, 1, kChunk, false>(p, m, g, backward, mask, s);
}

}  // namespace gscan
}  // namespace pesq
