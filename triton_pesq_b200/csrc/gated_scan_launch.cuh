// Instantiation of the gated scan kernels for one element type (one
// translation unit each, so that they compile in parallel).
#pragma once

#include "gated_scan.cuh"

namespace pesq {
namespace gscan {

// `after`: the kernel waits by itself for the one launched before it
template <class K>
cudaError_t start(K kernel, const Args& p, const Maps& m, const Geometry& g, size_t warp_smem, bool after,
                  cudaStream_t s) {
  const int warps = g.warps;
  const size_t smem = warps * warp_smem;
  if (smem > 40 << 10) {  // beside the static part, more than a kernel gets without asking
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  const int tiles = g.chunk == 1 ? (g.ctiles + warps - 1) / warps : g.ctiles * ((g.strips + warps - 1) / warps);
  c.gridDim = dim3((unsigned)tiles, (unsigned)p.batch);
  c.blockDim = dim3(32, warps);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  c.attrs = &at;
  c.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, p, m);
}

template <class T, int V, int L, bool kMask, bool kBulk>
cudaError_t launch_vl(const Args& p, const Maps& m, const Geometry& g, bool backward, cudaStream_t s) {
  constexpr bool kCuts = V == 1 && L > 1;  // only such rows are cut
  const bool cut = kCuts && g.strips > 1;
  cudaError_t e = cudaSuccess;
  if (!backward) {
    const size_t smem = kBulk ? Ring<T, V, L, 3, false, true>::kBytes : 0;
    if constexpr (kCuts) {
      if (g.row) return start(forward_row_kernel<T, L, kMask, kBulk>, p, m, g, smem, false, s);
      if (cut) e = start(forward_maps_kernel<T, L, kMask, kBulk>, p, m, g, smem, false, s);
    }
    return e != cudaSuccess ? e : start(forward_kernel<T, V, L, kMask, kBulk>, p, m, g, smem, cut, s);
  }
  if constexpr (kCuts) {
    if (cut)
      e = start(backward_maps_kernel<T, L, kMask, kBulk>, p, m, g, kBulk ? Ring<T, 1, L, 2, false, false>::kBytes : 0,
                false, s);
  }
  return e != cudaSuccess ? e
                          : start(backward_kernel<T, V, L, kMask, kBulk>, p, m, g,
                                  kBulk ? Ring<T, V, L, 4, true, true>::kBytes : 0, cut, s);
}

template <class T, int V>
cudaError_t launch_v(const Args& p, const Maps& m, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  if (g.chunk == 1)
    return mask ? launch_vl<T, V, 1, true, false>(p, m, g, backward, s)
                : launch_vl<T, V, 1, false, false>(p, m, g, backward, s);
  if (g.bulk)
    return mask ? launch_vl<T, V, chunk_steps(V, true), true, true>(p, m, g, backward, s)
                : launch_vl<T, V, chunk_steps(V, true), false, true>(p, m, g, backward, s);
  return mask ? launch_vl<T, V, chunk_steps(V, false), true, false>(p, m, g, backward, s)
              : launch_vl<T, V, chunk_steps(V, false), false, false>(p, m, g, backward, s);
}

template <class T>
cudaError_t launch(const Args& p, const Maps& m, const Geometry& g, bool backward, bool mask, cudaStream_t s) {
  return g.vec == 2 ? launch_v<T, 2>(p, m, g, backward, mask, s) : launch_v<T, 1>(p, m, g, backward, mask, s);
}

}  // namespace gscan
}  // namespace pesq
