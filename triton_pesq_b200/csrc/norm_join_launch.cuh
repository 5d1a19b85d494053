// Instantiation of the join's kernels for one pair of types of stream and
// block (one translation unit each, so that they compile in parallel).
#pragma once

#include "norm_join.cuh"

namespace pesq {
namespace njoin {

template <class K>
cudaError_t start(K kernel, const Args& p, unsigned grid, int threads, size_t smem, cudaStream_t s) {
  if (smem > 40 << 10) {  // beside the static part, more than a kernel gets without asking
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kernel<<<grid, threads, smem, s>>>(p);
  return cudaGetLastError();
}

template <class TS, class TB, int TEAM>
cudaError_t launch_team(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  const unsigned grid = (unsigned)g.blocks;
  constexpr int threads = TEAM > kThreads ? TEAM : kThreads;
  if (!backward)
    return g.wide ? start(forward_kernel<TS, TB, TEAM, true>, p, grid, threads, 0, s)
                  : start(forward_kernel<TS, TB, TEAM, false>, p, grid, threads, 0, s);
  constexpr size_t sums = kLeanRow<TEAM> ? 3 * kEach * sizeof(float) * threads : 0;
  return g.wide ? start(backward_kernel<TS, TB, TEAM, true>, p, grid, threads, sums, s)
                : start(backward_kernel<TS, TB, TEAM, false>, p, grid, threads, sums, s);
}

template <class TS, class TB>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  switch (g.team) {
    case 4: return launch_team<TS, TB, 4>(p, g, backward, s);
    case 8: return launch_team<TS, TB, 8>(p, g, backward, s);
    case 16: return launch_team<TS, TB, 16>(p, g, backward, s);
    case 32: return launch_team<TS, TB, 32>(p, g, backward, s);
    case 64: return launch_team<TS, TB, 64>(p, g, backward, s);
    case 128: return launch_team<TS, TB, 128>(p, g, backward, s);
    case 256: return launch_team<TS, TB, 256>(p, g, backward, s);
    case 512: return launch_team<TS, TB, 512>(p, g, backward, s);
    default: return launch_team<TS, TB, 1024>(p, g, backward, s);
  }
}

}  // namespace njoin
}  // namespace pesq
