// Instantiation of the layer norm's kernels for one pair of types of its input and
// output (one translation unit each, so that they compile in parallel).
#pragma once

#include "layer_norm.cuh"

namespace pesq {
namespace lnorm {

template <class TX, class TY, int TEAM, int GROUPS>
cudaError_t launch_team(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  const unsigned grid = (unsigned)g.blocks;
  constexpr int threads = TEAM > kThreads ? TEAM : kThreads;
  if (backward)
    g.wide ? backward_kernel<TX, TY, TEAM, GROUPS, true><<<grid, threads, 0, s>>>(p)
           : backward_kernel<TX, TY, TEAM, GROUPS, false><<<grid, threads, 0, s>>>(p);
  else
    g.wide ? forward_kernel<TX, TY, TEAM, GROUPS, true><<<grid, threads, 0, s>>>(p)
           : forward_kernel<TX, TY, TEAM, GROUPS, false><<<grid, threads, 0, s>>>(p);
  return cudaGetLastError();
}

template <class TX, class TY>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  switch (g.team) {
    case 4: return launch_team<TX, TY, 4, 1>(p, g, backward, s);
    case 8: return launch_team<TX, TY, 8, 1>(p, g, backward, s);
    case 16: return launch_team<TX, TY, 16, 1>(p, g, backward, s);
    case 32:
      return g.groups == 1   ? launch_team<TX, TY, 32, 1>(p, g, backward, s)
             : g.groups == 2 ? launch_team<TX, TY, 32, 2>(p, g, backward, s)
                             : launch_team<TX, TY, 32, 4>(p, g, backward, s);
    case 64: return launch_team<TX, TY, 64, 4>(p, g, backward, s);
    case 128: return launch_team<TX, TY, 128, 4>(p, g, backward, s);
    default: return launch_team<TX, TY, 256, 4>(p, g, backward, s);
  }
}

}  // namespace lnorm
}  // namespace pesq
