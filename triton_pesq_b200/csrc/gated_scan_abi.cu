// C ABI of the gated linear recurrence: checks, geometry, workspace, and the
// sum of the decay gradient's partial sums.
#include <cuda_runtime.h>

#include <algorithm>

#include "gated_scan.cuh"

using namespace pesq::gscan;
using pesq::set_error;

namespace pesq {
namespace gscan {
extern template cudaError_t launch<float>(const Args&, const Geometry&, bool, bool, cudaStream_t);
extern template cudaError_t launch<__nv_bfloat16>(const Args&, const Geometry&, bool, bool, cudaStream_t);
extern template cudaError_t launch<__half>(const Args&, const Geometry&, bool, bool, cudaStream_t);
}  // namespace gscan
}  // namespace pesq

namespace {

// ddecay[c] = -rate sigmoid(decay[c]) sum over the rows of part, in a fixed
// order: 32 columns a block, every thread a stride of the rows, then a tree.
constexpr int kSumRows = 16;
__global__ void __launch_bounds__(32 * kSumRows) decay_sum_kernel(const float* part, int64_t rows, int64_t width,
                                                                  const float* decay, float rate, float* out) {
  __shared__ float s[kSumRows][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < width) {
    int64_t r = threadIdx.y;
    for (; r + 3 * kSumRows < rows; r += 4 * kSumRows) {
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += part[(r + k * kSumRows) * width + c];
    }
    for (; r < rows; r += kSumRows) acc[0] += part[r * width + c];
  }
  s[threadIdx.y][threadIdx.x] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    float v = 0.0f;
    for (int k = 0; k < kSumRows; ++k) v += s[k][threadIdx.x];
    out[c] = -rate / (1.0f + expf(-decay[c])) * v;
  }
}

size_t element(int dtype) { return dtype == PESQ_F32 ? 4 : 2; }

bool even(const pesq_stream& s, const pesq_gated_scan_desc& d) {
  return reinterpret_cast<uintptr_t>(s.data) % (2 * element(d.dtype)) == 0 &&
         (d.batch == 1 || s.batch_stride % 2 == 0) && (d.steps == 1 || s.step_stride % 2 == 0);
}

int check(const pesq_gated_scan_desc* d) {
  if (!d) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL descriptor");
  if (d->batch < 1 || d->steps < 1 || d->width < 1)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "batch, steps and width must be at least 1");
  if (d->dtype < PESQ_F32 || d->dtype > PESQ_F16) return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown element type");
  if (!(d->rate > 0.0f) || d->rate > 1e6f) return set_error(PESQ_ERR_INVALID_ARGUMENT, "rate must be positive");
  const int64_t most = INT64_C(0x7fffffff);
  if (d->batch > most || d->width > most || d->steps > (most << 4) ||
      (double)d->batch * (double)((d->width + 31) / 32) * (double)((d->steps + kTile - 1) / kTile) > (double)most)
    return set_error(PESQ_ERR_UNSUPPORTED, "too many tiles for one launch");
  return PESQ_OK;
}

// Vector width and tile of a call.  Pairs of channels when everything allows
// it.  A row of at most kWarps steps gives each its own warp; a longer one
// goes by tiles of kWarps * kSteps steps.
Geometry geometry(const pesq_gated_scan_desc& d, int vec) {
  Geometry g{};
  g.vec = vec;
  g.ctiles = (int)((d.width + 32 * vec - 1) / (32 * vec));
  g.steps_per_thread = d.steps <= kWarps ? 1 : kSteps;
  const int64_t warps = (d.steps + g.steps_per_thread - 1) / g.steps_per_thread;
  g.warps = (int)std::min<int64_t>(warps, kWarps);
  g.tiles = (int)((d.steps + (int64_t)g.warps * g.steps_per_thread - 1) / ((int64_t)g.warps * g.steps_per_thread));
  g.blocks = d.batch * g.ctiles * g.tiles;
  return g;
}

int64_t row_tiles(const pesq_gated_scan_desc& d) { return d.steps <= kTile ? 1 : (d.steps + kTile - 1) / kTile; }

// [ticket, 16 bytes][end words][pair words][backward: partial decay sums]
size_t words(const pesq_gated_scan_desc& d) {
  const int64_t t = row_tiles(d);
  return t == 1 ? 0 : (size_t)(d.batch * t * d.width) * 8;
}
size_t chain_bytes(const pesq_gated_scan_desc& d) {
  const size_t w = words(d);
  return w ? 16 + 2 * w : 0;
}
size_t need(const pesq_gated_scan_desc& d, bool backward) {
  return chain_bytes(d) + (backward ? (size_t)(d.batch * row_tiles(d) * d.width) * 4 : 0);
}

int prepare(const pesq_gated_scan_desc& d, void* ws, size_t ws_bytes, bool backward, cudaStream_t stream, Args& a) {
  if (!d.x.data || !d.input_gate.data || !d.decay_gate.data || !d.decay)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL input");
  const size_t bytes = need(d, backward);
  if (bytes && (!ws || ws_bytes < bytes || reinterpret_cast<uintptr_t>(ws) % 16))
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  a.x = {d.x.data, d.x.batch_stride, d.x.step_stride};
  a.ig = {d.input_gate.data, d.input_gate.batch_stride, d.input_gate.step_stride};
  a.rg = {d.decay_gate.data, d.decay_gate.batch_stride, d.decay_gate.step_stride};
  a.decay = d.decay;
  a.state = d.state;
  a.reset = d.reset;
  a.reset_b = d.reset_batch_stride;
  a.reset_t = d.reset_step_stride;
  a.lengths = d.lengths;
  a.batch = d.batch;
  a.steps = d.steps;
  a.width = d.width;
  a.reverse = d.reverse != 0;
  a.rate = d.rate;
  a.spin_limit = d.spin_limit ? d.spin_limit : kSpinLimit;
  const size_t w = words(d);
  if (w) {
    if (!d.error) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL error word");
    a.error = d.error;
    a.ticket = static_cast<unsigned*>(ws);
    a.end = reinterpret_cast<unsigned long long*>(static_cast<char*>(ws) + 16);
    a.pair = a.end + w / 8;
    if (cudaMemsetAsync(ws, 0, 16 + 2 * w, stream) != cudaSuccess)
      return set_error(PESQ_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
  }
  return PESQ_OK;
}

int run(const pesq_gated_scan_desc& d, Args& a, const Geometry& g, bool backward, cudaStream_t s) {
  a.tiles = g.tiles;
  a.ctiles = g.ctiles;
  const bool mask = d.reset || d.lengths;
  const cudaError_t e = d.dtype == PESQ_F32    ? launch<float>(a, g, backward, mask, s)
                        : d.dtype == PESQ_BF16 ? launch<__nv_bfloat16>(a, g, backward, mask, s)
                                               : launch<__half>(a, g, backward, mask, s);
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

bool aligned(const void* p, const pesq_gated_scan_desc& d) {
  return reinterpret_cast<uintptr_t>(p) % (2 * element(d.dtype)) == 0;
}

}  // namespace

extern "C" {

int pesq_gated_scan_workspace(const pesq_gated_scan_desc* d, int backward, size_t* bytes) {
  if (!bytes) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check(d)) return status;
  *bytes = need(*d, backward != 0);
  return PESQ_OK;
}

int pesq_gated_scan_forward(const pesq_gated_scan_desc* d, void* stream, void* y, float* last, void* workspace,
                            size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (!y || !last) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL output");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  Args a{};
  if (const int status = prepare(*d, workspace, workspace_bytes, false, s, a)) return status;
  a.y = y;
  a.last = last;
  const bool pairs = d->width % 2 == 0 && even(d->x, *d) && even(d->input_gate, *d) && even(d->decay_gate, *d) &&
                     aligned(y, *d);
  return run(*d, a, geometry(*d, pairs ? 2 : 1), false, s);
}

int pesq_gated_scan_backward(const pesq_gated_scan_desc* d, void* stream, const void* saved, size_t saved_bytes,
                             pesq_stream dy, const float* dlast, void* dx, void* dinput_gate, void* ddecay_gate,
                             float* ddecay, float* dstate, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (!dx || !dinput_gate || !ddecay_gate || !ddecay) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL output");
  if (chain_bytes(*d) && (!saved || saved_bytes < chain_bytes(*d) || reinterpret_cast<uintptr_t>(saved) % 16))
    return set_error(PESQ_ERR_WORKSPACE, "the forward's workspace is missing or too small");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  Args a{};
  if (const int status = prepare(*d, workspace, workspace_bytes, true, s, a)) return status;
  a.dy = {dy.data, dy.batch_stride, dy.step_stride};
  a.dlast = dlast;
  a.dx = dx;
  a.dig = dinput_gate;
  a.drg = ddecay_gate;
  a.dstate = dstate;
  a.dpart = reinterpret_cast<float*>(static_cast<char*>(workspace) + chain_bytes(*d));
  if (words(*d)) a.start = reinterpret_cast<const unsigned long long*>(static_cast<const char*>(saved) + 16);
  const bool pairs = d->width % 2 == 0 && even(d->x, *d) && even(d->input_gate, *d) && even(d->decay_gate, *d) &&
                     (!dy.data || even(dy, *d)) && aligned(dx, *d) && aligned(dinput_gate, *d) &&
                     aligned(ddecay_gate, *d);
  const Geometry g = geometry(*d, pairs ? 2 : 1);
  if (const int status = run(*d, a, g, true, s)) return status;
  decay_sum_kernel<<<(unsigned)((d->width + 31) / 32), dim3(32, kSumRows), 0, s>>>(
      a.dpart, d->batch * g.tiles, d->width, d->decay, d->rate, ddecay);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
