// C ABI of the gated linear recurrence: checks, geometry, workspace, and the
// sum of the decay gradient's partial sums.
#include <cuda_runtime.h>

#include <algorithm>

#include "gated_scan.cuh"

using namespace pesq::gscan;
using pesq::set_error;

namespace pesq {
namespace gscan {
extern template cudaError_t launch<float>(const Args&, const Maps&, const Geometry&, bool, bool, cudaStream_t);
extern template cudaError_t launch<__nv_bfloat16>(const Args&, const Maps&, const Geometry&, bool, bool, cudaStream_t);
extern template cudaError_t launch<__half>(const Args&, const Maps&, const Geometry&, bool, bool, cudaStream_t);
}  // namespace gscan
}  // namespace pesq

namespace {

// Set by a kernel whose copies do not come; one a device
__device__ uint32_t g_error;

// ddecay[c] = -rate sigmoid(decay[c]) sum over the rows of part, in a fixed
// order: 32 columns a block, every thread a stride of the rows, then a tree.
constexpr int kSumRows = 32;
__global__ void __launch_bounds__(32 * kSumRows) decay_sum_kernel(const float* part, int64_t rows, int64_t width,
                                                                  const float* decay, float rate, float* out) {
  __shared__ float s[kSumRows][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  wait_for_last();
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
  if (!(d->rate > 0.0f) || d->rate > 1e6f) return set_error(PESQ_ERR_INVALID_ARGUMENT, "rate must lie above 0 and not above 1e6");
  if (d->batch > 65535 || d->width > (1 << 24) || d->steps > INT32_MAX - 64)
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

// Rows and channels that make this many warps are not cut: their cost is a row's walk, cut ones' the
// work of both kernels.  Forward and backward, whole / cut (us):
//   float32 in boxes    308 x 2000 steps: 122 / 132, 169 / 151;  448 x 2000: 122 / 155, 173 / 196
//   bfloat16 in boxes   448 x 2000: 128 / 124, 190 / 144;  672 x 2000: 148 / 151, 230 / 192;
//                       896 x 2000: 149 / 200, 232 / 243
//   float32 by lanes    520 x 2000: 204 / 175, 300 / 298;  624 x 2000: 212 / 224, 320 / 325
//   bfloat16 by lanes   624 x 2000: 196 / 194, 282 / 239;  832 x 2000: 201 / 222, 292 / 271
int64_t warps_enough(bool bulk, bool backward, int size) {
  return backward && size == 2 ? 148 * 5 : bulk && size == 4 ? 148 * 5 / 2 : 148 * 4;
}
// Short rows go through one CTA each up to so many warps; that / a warp a row, us:
//   float32 in boxes 308 x 500: 31 / 36, 448 x 500: 38 / 38;  bfloat16 448 x 500: 35 / 40, 560 x 500: 40 / 40
int64_t warps_for_rows(bool bulk, int size) { return bulk && size == 4 ? 148 * 3 : 148 * 4; }
// Rows and channel pairs that make so many warps take pairs of channels (forward and backward, pairs / single, us):
//   float32 in boxes    672 x 500: 73 / 69, 118 / 131;  768 x 512: 77 / 79, 138 / 146;  896 x 500: 81 / 91, 153 / 162;
//                       1232 x 500: 118 / 144, 227 / 214;  2240 x 500: 206 / 212, 347 / 374
//   float32 by lanes    1792 x 500: 202 / 175, 318 / 360;  2688 x 500: 259 / 255, 474 / 512
//   bfloat16 by lanes   1792 x 500: 156 / 144, 226 / 262;  2688 x 500: 177 / 200, 316 / 354
//   bfloat16 in boxes   4096 x 24: 23 / 27, 34 / 42;  4096 x 96: 49 / 52, 81 / 81;  4096 x 256: 111 / 113, 194 / 181;
//                       1792 x 500: 122 / 114, 210 / 181
int64_t warps_for_pairs(bool bulk, int size, int64_t steps) {
  return bulk && size == 4 ? 148 * 5 : !bulk || steps < 96 ? 148 * 12 : INT64_MAX;
}
// The fewest steps of a strip (2 x 256 x 512, backward: 13.4 us, 15.1 with 32), and of a row that is copied
// in boxes (512 x 24 x 512 bfloat16: 21.6 and 33.6 us, by lanes 25.6 and 37.9)
constexpr int kFewestSteps = 16;
constexpr int64_t kFewestBulk = 16;
// Single steps: more warps than this, what the device holds CTAs of at once, go in CTAs of eight (512 x 1 x 4096,
// forward: 20.5 us, 23.5 in CTAs of one); fewer in CTAs of one, which spread better
constexpr int64_t kWarpsAtOnce = 148 * 32;

// Whether boxes can be copied: 16-byte addresses and strides, which a tensor map asks for
bool boxes(const pesq_stream& s, const pesq_gated_scan_desc& d) {
  const int64_t e = element(d.dtype), most = INT64_C(1) << 39;
  return reinterpret_cast<uintptr_t>(s.data) % 16 == 0 && s.step_stride > 0 && s.step_stride < most &&
         s.step_stride * e % 16 == 0 &&
         (d.batch == 1 || (s.batch_stride > 0 && s.batch_stride < most && s.batch_stride * e % 16 == 0));
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

Geometry geometry(const pesq_gated_scan_desc& d, bool backward) {
  Geometry g{};
  const int size = (int)element(d.dtype);
  g.bulk = d.steps >= kFewestBulk && d.width * (int64_t)size % 16 == 0 && boxes(d.x, d) &&
           boxes(d.input_gate, d) && boxes(d.decay_gate, d);
  const bool pairs = d.width % 2 == 0 && fits(d.x, 2, d) && fits(d.input_gate, 2, d) && fits(d.decay_gate, 2, d);
  g.vec = pairs && d.batch * ((d.width + 63) / 64) >= warps_for_pairs(g.bulk, size, d.steps) ? 2 : 1;
  g.ctiles = (int)((d.width + 32 * g.vec - 1) / (32 * g.vec));
  g.chunk = d.steps == 1 ? 1 : chunk_steps(g.vec, g.bulk);
  const int64_t chunks = (d.steps + g.chunk - 1) / g.chunk, warps = d.batch * g.ctiles;
  int64_t strips = 1;
  g.row = !backward && g.vec == 1 && warps < warps_for_rows(g.bulk, size) && d.steps > kHeld &&
          d.steps <= kHeld * kRowWarps;
  if (!g.row && warps < warps_enough(g.bulk, backward, size)) {
    // one wave, in CTAs of four or eight strips: the more strips that gives, and eight where they are as many, since
    // a strip goes through all the CTAs before its own
    const bool mask = d.reset || d.lengths;
    for (int w = 4; w <= (backward ? backward_strips(g.bulk, mask, size) : 8); w *= 2) {
      const int ctas = backward ? backward_ctas(w, g.bulk, mask, size) : forward_ctas(w, g.bulk, size);
      const int64_t n = std::max<int64_t>(1, 148 * ctas / warps) * w;
      if (n >= strips) strips = n, g.warps = w;
    }
    strips = std::max<int64_t>(1, std::min(strips, (d.steps + kFewestSteps - 1) / kFewestSteps));
  }
  if (g.row) strips = (d.steps + kHeld - 1) / kHeld;
  const int64_t per = g.row ? kHeld / g.chunk : (chunks + strips - 1) / strips;
  g.strips = (int)((chunks + per - 1) / per);
  g.strip = (int)(per * g.chunk);
  g.warps = g.row                                     ? g.strips
            : d.steps == 1 && warps > kWarpsAtOnce ? std::min(g.ctiles, kStrips)
                                                   : std::max(1, std::min(g.strips, g.warps));
  return g;
}

// A result, dense: as aligned as its way out wants it
bool fits(const void* p, const Geometry& g, const pesq_gated_scan_desc& d) {
  return g.bulk ? reinterpret_cast<uintptr_t>(p) % 16 == 0 : fits(p, g.vec, d);
}

// (a step stride of 0: one row of zeros, and what lies outside a map reads as zero)
bool encode(CUtensorMap& m, const pesq_stream& s, const pesq_gated_scan_desc& d, const Geometry& g) {
  const bool one = s.step_stride == 0;
  const cuuint64_t e = element(d.dtype), step = (one ? d.width : s.step_stride) * e;
  const cuuint64_t dims[3] = {(cuuint64_t)d.width, one ? 1 : (cuuint64_t)d.steps, one ? 1 : (cuuint64_t)d.batch};
  const cuuint64_t strides[2] = {step, one || d.batch == 1 ? step : s.batch_stride * e};
  const cuuint32_t box[3] = {32u * g.vec, (cuuint32_t)g.chunk, 1}, unit[3] = {1, 1, 1};
  const CUtensorMapDataType type = d.dtype == PESQ_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : d.dtype == PESQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return encoder()(&m, type, 3, const_cast<void*>(s.data), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }
// maps of strips and of CTAs of strips
size_t map_bytes(const pesq_gated_scan_desc& d, const Geometry& g) {
  if (g.strips == 1 || g.row) return 0;
  return round16((size_t)(d.batch * (g.strips + (g.strips + g.warps - 1) / g.warps) * d.width) * 8);
}
size_t kept_bytes(const pesq_gated_scan_desc& d) {  // (of the sizes alone)
  return round16((size_t)(d.batch * ((d.steps + kKept - 1) / kKept) * d.width) * 4);
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
  if (g.strips > 1 && !g.row) {
    a.before = reinterpret_cast<float2*>(maps);
    a.total = a.before + d.batch * g.strips * d.width;
  }
  return PESQ_OK;
}

bool missing(const void* p, size_t have, size_t want) {
  return want && (!p || have < want || reinterpret_cast<uintptr_t>(p) % 16);
}

// The current device's error word
uint32_t* error_word() {
  static uint32_t* words[64] = {nullptr};  // by device; an address that does not change
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!words[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_error) != cudaSuccess) return nullptr;
    words[dev] = static_cast<uint32_t*>(p);
  }
  return words[dev];
}

int run(const pesq_gated_scan_desc& d, Args& a, const Geometry& g, const pesq_stream* dy, cudaStream_t s) {
  const bool backward = dy != nullptr, mask = d.reset || d.lengths;
  Maps m;
  if (g.bulk) {
    if (!encoder()) return set_error(PESQ_ERR_CUDA, "no cuTensorMapEncodeTiled");
    // the encoder is the driver's: it wants a context, which a thread that has not called the runtime yet lacks
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
      return set_error(PESQ_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
    a.error = error_word();
    if (!a.error) return set_error(PESQ_ERR_CUDA, "no error word");
    if (!encode(m.x, d.x, d, g) || !encode(m.ig, d.input_gate, d, g) || !encode(m.rg, d.decay_gate, d, g) ||
        (backward && !encode(m.dy, *dy, d, g)))
      return set_error(PESQ_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    void* out[3] = {a.drg, a.dig, backward ? a.dx : a.y};
    for (int i = backward ? 0 : 2; i < 3 && d.dtype != PESQ_F32 && !g.row; ++i)
      if (!encode(m.out[i], {out[i], d.steps * d.width, d.width}, d, g))
        return set_error(PESQ_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  }
  const cudaError_t e = d.dtype == PESQ_F32    ? launch<float>(a, m, g, backward, mask, s)
                        : d.dtype == PESQ_BF16 ? launch<__nv_bfloat16>(a, m, g, backward, mask, s)
                                               : launch<__half>(a, m, g, backward, mask, s);
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int pesq_gated_scan_sizes(const pesq_gated_scan_desc* d, size_t* forward, size_t* kept, size_t* backward) {
  if (!forward || !kept || !backward) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check(d)) return status;
  const Geometry g = geometry(*d, false);
  *forward = map_bytes(*d, g);
  *kept = kept_bytes(*d);
  *backward = back_bytes(*d, geometry(*d, true));
  return PESQ_OK;
}

int pesq_gated_scan_kept_steps(const pesq_gated_scan_desc* d, int32_t* here, int32_t* most) {
  if (!here || !most) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check(d)) return status;
  *here = geometry(*d, false).chunk;
  pesq_gated_scan_desc dense = *d;  // what tensor copies take is what has the longest chunks
  dense.x = dense.input_gate = dense.decay_gate = {reinterpret_cast<const void*>(256), d->steps * d->width, d->width};
  *most = std::max(*here, (int32_t)geometry(dense, false).chunk);
  return PESQ_OK;
}

int pesq_gated_scan_forward(const pesq_gated_scan_desc* d, void* stream, void* y, float* last, void* kept,
                            size_t kept_size, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (!y || !last) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL output");
  const Geometry g = geometry(*d, false);
  if (!fits(y, g, *d)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "y is less aligned than the inputs");
  if (missing(workspace, workspace_bytes, map_bytes(*d, g)) || (kept && missing(kept, kept_size, kept_bytes(*d))))
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  Args a{};
  if (const int status = prepare(*d, g, static_cast<char*>(workspace), a)) return status;
  a.y = y;
  a.last = last;
  a.kept = static_cast<float*>(kept);
  return run(*d, a, g, nullptr, static_cast<cudaStream_t>(stream));
}

int pesq_gated_scan_backward(const pesq_gated_scan_desc* d, void* stream, const void* kept, size_t kept_size,
                             pesq_stream dy, const float* dlast, void* dx, void* dinput_gate, void* ddecay_gate,
                             float* ddecay, float* dstate, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (!dx || !dinput_gate || !ddecay_gate || !ddecay) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL output");
  const Geometry g = geometry(*d, true);
  if ((dy.data && (g.bulk ? !boxes(dy, *d) : !fits(dy, g.vec, *d))) || !fits(dx, g, *d) || !fits(dinput_gate, g, *d) ||
      !fits(ddecay_gate, g, *d))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "a gradient is less aligned than the inputs");
  if (missing(kept, kept_size, kept_bytes(*d)))
    return set_error(PESQ_ERR_WORKSPACE, "the states that the forward kept are missing");
  if (d->kept_steps > g.chunk)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "the forward kept its states too far apart for streams laid out like these");
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
    dy = {zeros, 0, 0};
  }
  a.dlast = dlast;
  a.dx = dx;
  a.dig = dinput_gate;
  a.drg = ddecay_gate;
  a.dstate = dstate;
  a.dpart = reinterpret_cast<float*>(ws);
  a.kept = const_cast<float*>(static_cast<const float*>(kept));
  if (const int status = run(*d, a, g, &dy, s)) return status;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)((d->width + 31) / 32));
  c.blockDim = dim3(32, kSumRows);
  c.stream = s;
  c.attrs = &at;
  c.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&c, decay_sum_kernel, (const float*)a.dpart, (int64_t)(d->batch * g.strips),
                                           d->width, d->decay, d->rate, ddecay);
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

int pesq_gated_scan_check(void* stream, uint32_t* failed) {
  if (!failed) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  uint32_t* word = error_word();
  if (!word) return set_error(PESQ_ERR_CUDA, "no error word");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(failed, word, sizeof(uint32_t), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, sizeof(uint32_t), s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
