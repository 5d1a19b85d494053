// Instantiation of the layer norm's kernels for one pair of types of its input and
// output (one translation unit each, so that they compile in parallel).
#pragma once

#include "layer_norm.cuh"

namespace pesq {
namespace lnorm {

template <class TX, class TY, int TEAM, int GROUPS, bool kWide>
cudaError_t launch_team(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  constexpr int threads = threads_of(TEAM);
  if (backward)
    backward_kernel<TX, TY, TEAM, GROUPS, kWide><<<(unsigned)g.blocks, threads, 0, s>>>(p);
  else
    forward_kernel<TX, TY, TEAM, GROUPS, kWide><<<(unsigned)g.blocks, threads, 0, s>>>(p);
  return cudaGetLastError();
}

template <class TX, class TY, bool kWide>
cudaError_t launch_width(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  constexpr int kMost = most_groups(kWide);
  switch (g.team) {
    case 4: return launch_team<TX, TY, 4, 1, kWide>(p, g, backward, s);
    case 8: return launch_team<TX, TY, 8, 1, kWide>(p, g, backward, s);
    case 16: return launch_team<TX, TY, 16, 1, kWide>(p, g, backward, s);
    case 32:
      if (g.groups == 1) return launch_team<TX, TY, 32, 1, kWide>(p, g, backward, s);
      if (g.groups == 2) return launch_team<TX, TY, 32, 2, kWide>(p, g, backward, s);
      return launch_team<TX, TY, 32, kMost, kWide>(p, g, backward, s);
    case 64: return launch_team<TX, TY, 64, kMost, kWide>(p, g, backward, s);
    case 96:
      if (g.groups == 2) return launch_team<TX, TY, 96, 2, kWide>(p, g, backward, s);
      return launch_team<TX, TY, 96, kMost, kWide>(p, g, backward, s);
    case 128: return launch_team<TX, TY, 128, kMost, kWide>(p, g, backward, s);
    case 160: return launch_team<TX, TY, 160, kMost, kWide>(p, g, backward, s);
    case 192: return launch_team<TX, TY, 192, kMost, kWide>(p, g, backward, s);
    case 256: return launch_team<TX, TY, 256, kMost, kWide>(p, g, backward, s);
    default:
      if constexpr (kMost < 4) {
        if (g.team == 384) return launch_team<TX, TY, 384, kMost, kWide>(p, g, backward, s);
        return launch_team<TX, TY, 512, kMost, kWide>(p, g, backward, s);
      }
      return cudaErrorInvalidConfiguration;
  }
}

template <class TX, class TY>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  return g.wide ? launch_width<TX, TY, true>(p, g, backward, s) : launch_width<TX, TY, false>(p, g, backward, s);
}

}  // namespace lnorm
}  // namespace pesq
