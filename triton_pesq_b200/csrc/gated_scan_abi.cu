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

int check(const pesq_gated_scan_desc* d) {
  if (!d) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL descriptor");
  if (d->batch < 1 || d->steps < 1 || d->width < 1)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "batch, steps and width must be at least 1");
  if (d->dtype < PESQ_F32 || d->dtype > PESQ_F16) return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown element type");
  if (!(d->rate > 0.0f) || d->rate > 1e6f) return set_error(PESQ_ERR_INVALID_ARGUMENT, "rate must be positive");
  if (d->batch > 65535 || d->width > (1 << 24) || d->steps > INT32_MAX - kChunk)
    return set_error(PESQ_ERR_UNSUPPORTED, "more than 65535 rows, 2^24 channels or 2^31 steps in one call");
  return PESQ_OK;
}

bool fits(const void* p, int vec, const pesq_gated_scan_desc& d) {
  return reinterpret_cast<uintptr_t>(p) % (vec * element(d.dtype)) == 0;
}
bool fits(const pesq_stream& s, int vec, const pesq_gated_scan_desc& d) {
  return fits(s.data, vec, d) && (d.batch == 1 || s.batch_stride % vec == 0) &&
         (d.steps == 1 || s.step_stride % vec == 0);
}

// Warps that fill the device, and the fewest chunks of a strip
constexpr int64_t kWarpsWanted = 148 * 8;
constexpr int64_t kWarpsEnough = 148 * 4;
constexpr int kFewestChunks = 4;

// Pairs of channels where everything allows it (a backward call has its
// forward's inputs, so takes its forward's).  One strip a row once rows and
// channels make kWarpsEnough warps; otherwise as many as make kWarpsWanted.
Geometry geometry(const pesq_gated_scan_desc& d) {
  Geometry g{};
  g.vec = d.width % 2 == 0 && fits(d.x, 2, d) && fits(d.input_gate, 2, d) && fits(d.decay_gate, 2, d) ? 2 : 1;
  g.ctiles = (int)((d.width + 32 * g.vec - 1) / (32 * g.vec));
  g.chunk = d.steps == 1 ? 1 : kChunk;
  const int64_t chunks = (d.steps + g.chunk - 1) / g.chunk, warps = d.batch * g.ctiles;
  int64_t strips = 1;
  if (warps < kWarpsEnough)
    strips = std::max<int64_t>(1, std::min((kWarpsWanted + warps - 1) / warps, chunks / kFewestChunks));
  const int64_t per = (chunks + strips - 1) / strips;
  g.strips = (int)((chunks + per - 1) / per);
  g.strip = (int)(per * g.chunk);
  return g;
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }
// maps of strips and of CTAs of strips
size_t map_bytes(const pesq_gated_scan_desc& d, const Geometry& g) {
  return g.strips == 1 ? 0 : round16((size_t)(d.batch * (g.strips + (g.strips + kStrips - 1) / kStrips) * d.width) * 8);
}
size_t kept_bytes(const pesq_gated_scan_desc& d, const Geometry& g) {
  return round16((size_t)(d.batch * ((d.steps + g.chunk - 1) / g.chunk) * d.width) * 4);
}
size_t part_bytes(const pesq_gated_scan_desc& d, const Geometry& g) {
  return round16((size_t)(d.batch * g.strips * d.width) * 4);
}

// [partial decay sums][maps][a row of zeros]
size_t back_bytes(const pesq_gated_scan_desc& d, const Geometry& g) {
  return part_bytes(d, g) + map_bytes(d, g) + round16(d.width * element(d.dtype));
}

// A step stride as the kernels take it: in bytes, 32 bits
int narrow_stride(const pesq_stream& s, const pesq_gated_scan_desc& d, Stream& out) {
  const int64_t bytes = d.steps == 1 ? 0 : s.step_stride * (int64_t)element(d.dtype);
  if (bytes > INT32_MAX || bytes < -INT32_MAX)
    return set_error(PESQ_ERR_UNSUPPORTED, "steps lie more than 2 GiB apart");
  out = {s.data, s.batch_stride, (int)bytes};
  return PESQ_OK;
}

int prepare(const pesq_gated_scan_desc& d, const Geometry& g, char* maps, Args& a) {
  if (!d.x.data || !d.input_gate.data || !d.decay_gate.data || !d.decay)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL input");
  if (const int status = narrow_stride(d.x, d, a.x)) return status;
  if (const int status = narrow_stride(d.input_gate, d, a.ig)) return status;
  if (const int status = narrow_stride(d.decay_gate, d, a.rg)) return status;
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
  a.ctiles = g.ctiles;
  a.strips = g.strips;
  a.strip = g.strip;
  if (g.strips > 1) {
    a.before = reinterpret_cast<float2*>(maps);
    a.total = a.before + d.batch * g.strips * d.width;
  }
  return PESQ_OK;
}

bool missing(const void* p, size_t have, size_t want) {
  return want && (!p || have < want || reinterpret_cast<uintptr_t>(p) % 16);
}

int run(const pesq_gated_scan_desc& d, const Args& a, const Geometry& g, bool backward, cudaStream_t s) {
  const bool mask = d.reset || d.lengths;
  const cudaError_t e = d.dtype == PESQ_F32    ? launch<float>(a, g, backward, mask, s)
                        : d.dtype == PESQ_BF16 ? launch<__nv_bfloat16>(a, g, backward, mask, s)
                                               : launch<__half>(a, g, backward, mask, s);
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int pesq_gated_scan_sizes(const pesq_gated_scan_desc* d, size_t* forward, size_t* kept, size_t* backward) {
  if (!forward || !kept || !backward) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check(d)) return status;
  const Geometry g = geometry(*d);
  *forward = map_bytes(*d, g);
  *kept = kept_bytes(*d, g);
  *backward = back_bytes(*d, g);
  return PESQ_OK;
}

int pesq_gated_scan_forward(const pesq_gated_scan_desc* d, void* stream, void* y, float* last, void* kept,
                            size_t kept_size, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (!y || !last) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL output");
  const Geometry g = geometry(*d);
  if (!fits(y, g.vec, *d)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "y is less aligned than the inputs");
  if (missing(workspace, workspace_bytes, map_bytes(*d, g)) || (kept && missing(kept, kept_size, kept_bytes(*d, g))))
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  Args a{};
  if (const int status = prepare(*d, g, static_cast<char*>(workspace), a)) return status;
  a.y = y;
  a.last = last;
  a.kept = static_cast<float*>(kept);
  return run(*d, a, g, false, static_cast<cudaStream_t>(stream));
}

int pesq_gated_scan_backward(const pesq_gated_scan_desc* d, void* stream, const void* kept, size_t kept_size,
                             pesq_stream dy, const float* dlast, void* dx, void* dinput_gate, void* ddecay_gate,
                             float* ddecay, float* dstate, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (!dx || !dinput_gate || !ddecay_gate || !ddecay) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL output");
  const Geometry g = geometry(*d);
  if ((dy.data && !fits(dy, g.vec, *d)) || !fits(dx, g.vec, *d) || !fits(dinput_gate, g.vec, *d) ||
      !fits(ddecay_gate, g.vec, *d))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "a gradient is less aligned than the inputs");
  if (missing(kept, kept_size, kept_bytes(*d, g)))
    return set_error(PESQ_ERR_WORKSPACE, "the states that the forward kept are missing");
  if (missing(workspace, workspace_bytes, back_bytes(*d, g)))
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  Args a{};
  char* ws = static_cast<char*>(workspace);
  if (const int status = prepare(*d, g, ws + part_bytes(*d, g), a)) return status;
  if (dy.data) {
    if (const int status = narrow_stride(dy, *d, a.dy)) return status;
  } else {  // one row of zeros for all steps
    char* zeros = ws + part_bytes(*d, g) + map_bytes(*d, g);
    if (cudaMemsetAsync(zeros, 0, d->width * element(d->dtype), s) != cudaSuccess)
      return set_error(PESQ_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
    a.dy = {zeros, 0, 0};
  }
  a.dlast = dlast;
  a.dx = dx;
  a.dig = dinput_gate;
  a.drg = ddecay_gate;
  a.dstate = dstate;
  a.dpart = reinterpret_cast<float*>(ws);
  a.kept = const_cast<float*>(static_cast<const float*>(kept));
  if (const int status = run(*d, a, g, true, s)) return status;
  decay_sum_kernel<<<(unsigned)((d->width + 31) / 32), dim3(32, kSumRows), 0, s>>>(
      a.dpart, d->batch * g.strips, d->width, d->decay, d->rate, ddecay);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
