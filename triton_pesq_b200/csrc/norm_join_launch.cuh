// Instantiation of the join's kernels for one pair of types of stream and
// block (one translation unit each, so that they compile in parallel).
#pragma once

#include "norm_join.cuh"

namespace pesq {
namespace njoin {

template <class TS, class TB, int TEAM>
void launch_team(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  const unsigned grid = (unsigned)g.blocks;
  constexpr int threads = TEAM > kThreads ? TEAM : kThreads;
  if (g.wide) {
    if (backward)
      backward_kernel<TS, TB, TEAM, true><<<grid, threads, 0, s>>>(p);
    else
      forward_kernel<TS, TB, TEAM, true><<<grid, threads, 0, s>>>(p);
  } else {
    if (backward)
      backward_kernel<TS, TB, TEAM, false><<<grid, threads, 0, s>>>(p);
    else
      forward_kernel<TS, TB, TEAM, false><<<grid, threads, 0, s>>>(p);
  }
}

template <class TS, class TB>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, cudaStream_t s) {
  switch (g.team) {
    case 4: launch_team<TS, TB, 4>(p, g, backward, s); break;
    case 16: launch_team<TS, TB, 16>(p, g, backward, s); break;
    case 32: launch_team<TS, TB, 32>(p, g, backward, s); break;
    case 64: launch_team<TS, TB, 64>(p, g, backward, s); break;
    case 128: launch_team<TS, TB, 128>(p, g, backward, s); break;
    case 256: launch_team<TS, TB, 256>(p, g, backward, s); break;
    case 512: launch_team<TS, TB, 512>(p, g, backward, s); break;
    default: launch_team<TS, TB, 1024>(p, g, backward, s); break;
  }
  return cudaGetLastError();
}

}  // namespace njoin
}  // namespace pesq
