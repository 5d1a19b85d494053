// Instantiation of the linear attention's kernels for one type (the forward and the backward of each in a translation
// unit of its own, so that they compile in parallel).
#pragma once

#include "linear_attention.cuh"

namespace pesq {
namespace lattn {

// close: to the kernel before, whose results it waits for itself
inline cudaError_t start(void (*kernel)(Args), const Args& p, int64_t grid, int threads, int smem, bool close, cudaStream_t s) {
  if (smem > 48 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = close;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)grid);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = (size_t)smem;
  c.stream = s;
  c.attrs = &at;
  c.numAttrs = close ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, p);
}

template <class T, int DK, int DV, int C, bool kWhole>
cudaError_t launch_forward(const Args& p, const Geometry& g, Kind kind, cudaStream_t s) {
  switch (kind) {
    case kForward: return start(forward_kernel<T, DK, DV, C, kWhole>, p, g.blocks, 128, ForwardShared<T, DK, DV, C>::kBytes, p.parts > 1, s);
    case kSweep: return start(sweep_kernel<T, DK, DV, C, kWhole, false>, p, g.blocks, 128, SweepShared<T, DK, DV, C>::kBytes, false, s);
    default: return start(sweep_kernel<T, DK, DV, C, kWhole, true>, p, g.blocks, 128, SweepShared<T, DK, DV, C>::kBytes, false, s);
  }
}

// Whether the padding is worked on too: where the widths fill it, and of bfloat16, whose instructions are too few for its
// tests to pay (a forward of 40 x 512 x 16 rows' steps of 12 x 20: 70 us with the padding, 74 without; float32 150 and 115.  Of backwards
// padded to 128 x 128 it depends: 192 rows of 1000 steps of 72 x 72 take 599 and 522, of 100 x 100 612 and 719)
template <class T>
constexpr bool kAlwaysWhole = std::is_same<T, __nv_bfloat16>::value;

template <class T, int DK, int DV, int C>
cudaError_t launch_forward(const Args& p, const Geometry& g, Kind kind, cudaStream_t s) {
  if constexpr (!kAlwaysWhole<T>) {
    if (p.key <= DK - 16 || p.value <= DV * p.slices - 16) return launch_forward<T, DK, DV, C, false>(p, g, kind, s);
  }
  return launch_forward<T, DK, DV, C, true>(p, g, kind, s);
}

template <class T, int DK>
cudaError_t forward_width(const Args& p, const Geometry& g, Kind kind, cudaStream_t s) {
  if (kind == kSteps) return start(steps_kernel<T, DK>, p, g.blocks, 128, 0, false, s);
  if constexpr (std::is_same<T, float>::value && DK == 128) {
    if (g.chunk == 32) return launch_forward<T, DK, 64, 32>(p, g, kind, s);
  }
  return g.dv == 32 ? launch_forward<T, DK, 32, 64>(p, g, kind, s) : launch_forward<T, DK, 64, 64>(p, g, kind, s);
}

// the forward, the sweeps of both directions and single steps
template <class T>
cudaError_t forward_of(const Args& p, const Geometry& g, Kind kind, cudaStream_t s) {
  return g.dk == 32   ? forward_width<T, 32>(p, g, kind, s)
         : g.dk == 64 ? forward_width<T, 64>(p, g, kind, s)
                      : forward_width<T, 128>(p, g, kind, s);
}

template <class T, int DK, int DV>
cudaError_t launch_backward(const Args& p, const Geometry& g, cudaStream_t s) {
  constexpr int dtype = std::is_same<T, float>::value ? PESQ_F32 : PESQ_BF16, C = chunk_of(dtype, DK, DV);
  constexpr int kThreads = 64 * kSide<T, DK, DV>, kBytes = BackwardShared<T, DK, DV, C>::kBytes;
  if constexpr (!kAlwaysWhole<T>) {
    if (p.key <= DK - 16 || p.value <= DV - 16) return start(backward_kernel<T, DK, DV, C, false>, p, g.blocks, kThreads, kBytes, p.parts > 1, s);
  }
  return start(backward_kernel<T, DK, DV, C, true>, p, g.blocks, kThreads, kBytes, p.parts > 1, s);
}
template <class T, int DK>
cudaError_t backward_width(const Args& p, const Geometry& g, cudaStream_t s) {
  return g.dv == 32   ? launch_backward<T, DK, 32>(p, g, s)
         : g.dv == 64 ? launch_backward<T, DK, 64>(p, g, s)
                      : launch_backward<T, DK, 128>(p, g, s);
}
template <class T>
cudaError_t backward_of(const Args& p, const Geometry& g, cudaStream_t s) {
  return g.dk == 32   ? backward_width<T, 32>(p, g, s)
         : g.dk == 64 ? backward_width<T, 64>(p, g, s)
                      : backward_width<T, 128>(p, g, s);
}

}  // namespace lattn
}  // namespace pesq
