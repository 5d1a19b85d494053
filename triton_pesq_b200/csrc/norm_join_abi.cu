// C ABI of the norm-gate-residual join: checks, geometry, workspace, and the
// sums of the vectors' gradients.
#include <cuda_runtime.h>

#include <algorithm>

#include "norm_join.cuh"

using namespace pesq::njoin;
using pesq::set_error;

namespace pesq {
namespace njoin {
extern template cudaError_t launch<float, float>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<__nv_bfloat16, __nv_bfloat16>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<__half, __half>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<float, __nv_bfloat16>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<float, __half>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace njoin
}  // namespace pesq

namespace {

constexpr int kMaxWidth = 8192;  // one CTA of 1024 threads holds a row

// Columns of the CTAs' sums, in a fixed order: 32 columns a block, every thread a
// stride of the rows, then a tree.  first + blockIdx.y: 0 the pre vector, 1 the post and scale
// vectors, 2 + b the shared gate of batch item b.
struct SumArgs {
  const float *pre, *u, *gate, *post, *scale;
  float *dpre, *dpost, *dscale;
  void* dgate;
  int64_t rows, per_item, first;
  int width, dtype;
};
constexpr int kSumRows = 32, kMostSums = 65535;  // (of a launch)
__global__ void __launch_bounds__(32 * kSumRows) vectors_kernel(const __grid_constant__ SumArgs p) {
  __shared__ float s[kSumRows][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const int64_t which = p.first + blockIdx.y;
  const float* part = which == 0 ? p.pre : which == 1 ? p.u : p.gate + (which - 2) * p.per_item * p.width;
  const int64_t rows = which < 2 ? p.rows : p.per_item;
  if (!part) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the kernel before, which this one is launched close to
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < p.width) {
    int64_t r = threadIdx.y;
    for (; r + 3 * kSumRows < rows; r += 4 * kSumRows) {
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += part[(r + k * kSumRows) * p.width + c];
    }
    for (; r < rows; r += kSumRows) acc[0] += part[r * p.width + c];
  }
  s[threadIdx.y][threadIdx.x] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
  __syncthreads();
  if (threadIdx.y != 0 || c >= p.width) return;
  float v = 0.0f;
#pragma unroll
  for (int k = 0; k < kSumRows; ++k) v += s[k][threadIdx.x];
  if (which == 0) {
    p.dpre[c] = v;
  } else if (which == 1) {
    p.dpost[c] = p.scale ? v * p.scale[c] : v;
    if (p.dscale) p.dscale[c] = v * p.post[c];
  } else {
    const int64_t at = (which - 2) * p.width + c;
    if (p.dtype == PESQ_F32)
      static_cast<float*>(p.dgate)[at] = v;
    else if (p.dtype == PESQ_BF16)
      static_cast<__nv_bfloat16*>(p.dgate)[at] = __float2bfloat16_rn(v);
    else
      static_cast<__half*>(p.dgate)[at] = __float2half_rn(v);
  }
}

size_t element(int dtype) { return dtype == PESQ_F32 ? 4 : 2; }

int check(const pesq_norm_join_desc* d) {
  if (!d) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL descriptor");
  if (d->batch < 1 || d->steps < 1 || d->width < 1)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "batch, steps and width must be at least 1");
  if (d->width > kMaxWidth) return set_error(PESQ_ERR_UNSUPPORTED, "at most 8192 channels");
  if (d->stream_dtype < PESQ_F32 || d->stream_dtype > PESQ_F16 || d->dtype < PESQ_F32 || d->dtype > PESQ_F16 ||
      (d->stream_dtype != PESQ_F32 && d->stream_dtype != d->dtype))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "the stream is float32 or of the block's type");
  if (d->activation != PESQ_SIGMOID && d->activation != PESQ_SILU)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown activation");
  if (!(d->eps >= 0.0f)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "eps must not be negative");
  if (d->gate_shared && !d->gate.data) return set_error(PESQ_ERR_INVALID_ARGUMENT, "a shared gate that is NULL");
  if (!d->block.data && d->gate.data) return set_error(PESQ_ERR_INVALID_ARGUMENT, "a gate without a block");
  if (d->batch > INT32_MAX || d->steps > INT64_C(1) << 40)
    return set_error(PESQ_ERR_UNSUPPORTED, "too many rows for one launch");
  return PESQ_OK;
}

struct Plan {
  Geometry g;
  int64_t batch, steps;  // rows, batch items joined where their strides allow
  int units, span;
};

bool joined(const pesq_stream& s, const pesq_norm_join_desc& d) {
  return !s.data || d.batch == 1 || s.batch_stride == d.steps * s.step_stride;
}
bool wide(const pesq_stream& s, const pesq_norm_join_desc& d, int dtype) {
  const int64_t unit = 16 / element(dtype);
  return !s.data || (reinterpret_cast<uintptr_t>(s.data) % 16 == 0 && (d.batch == 1 || s.batch_stride % unit == 0) &&
                     (d.steps == 1 || s.step_stride % unit == 0));
}
bool wide(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// As many CTAs as the device holds at once, each with its share of the rows, but
// none with less than a row a team.
Plan plan(const pesq_norm_join_desc& d, bool backward, const pesq_stream* dstream, const pesq_stream* dnormed) {
  Plan q{};
  const pesq_stream none{nullptr, 0, 0};
  const pesq_stream &ds = dstream ? *dstream : none, &dn = dnormed ? *dnormed : none;
  const bool flat = joined(d.stream, d) && joined(d.block, d) && joined(ds, d) && joined(dn, d) &&
                    (d.gate_shared ? d.batch == 1 : joined(d.gate, d));
  q.batch = flat ? 1 : d.batch;
  q.steps = flat ? d.batch * d.steps : d.steps;
  q.g.team = 4;
  for (int t : {8, 16, 32, 64, 128, 256, 512, 1024})
    if (q.g.team * kEach < d.width) q.g.team = t;
  q.g.wide = d.width % kEach == 0 && wide(d.stream, d, d.stream_dtype) && wide(d.block, d, d.dtype) &&
             wide(d.gate, d, d.dtype) && wide(ds, d, d.stream_dtype) && wide(dn, d, d.dtype) && wide(d.post) &&
             wide(d.pre) && wide(d.scale);
  const int threads = std::max(q.g.team, kThreads), teams = threads / q.g.team;
  const int64_t most = std::max<int64_t>(1, 148 * ctas(backward, q.g.wide, q.g.team) / q.batch);
  const int64_t units = std::min<int64_t>(most, (q.steps + teams - 1) / teams);
  q.span = (int)std::min<int64_t>(INT32_MAX - 1024, (q.steps + units - 1) / units);
  q.units = (int)((q.steps + q.span - 1) / q.span);
  q.g.blocks = q.batch * q.units;
  return q;
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }
size_t part_bytes(const pesq_norm_join_desc& d) {
  // (whatever the gradients' strides, no more CTAs than this)
  const int64_t rows = std::max<int64_t>(d.batch, 148 * ctas(true, true, 1)) + d.batch;
  return round16((size_t)rows * d.width * 4);
}

Rows rows_of(const pesq_stream& s) {
  return {s.data, s.batch_stride, s.step_stride};
}

void fill(Args& a, const pesq_norm_join_desc& d, const Plan& q) {
  a.stream = rows_of(d.stream);
  a.block = rows_of(d.block);
  a.gate = rows_of(d.gate);
  if (d.gate_shared) a.gate.st = 0;
  a.post = d.post;
  a.pre = d.pre;
  a.scale = d.scale;
  a.batch = q.batch;
  a.steps = q.steps;
  a.width = (int)d.width;
  a.units = q.units;
  a.span = q.span;
  a.silu = d.activation == PESQ_SILU;
  a.eps = d.eps;
}

cudaError_t run(const Args& a, const Plan& q, const pesq_norm_join_desc& d, bool backward, cudaStream_t s) {
  if (d.stream_dtype == PESQ_F32)
    return d.dtype == PESQ_F32    ? launch<float, float>(a, q.g, backward, s)
           : d.dtype == PESQ_BF16 ? launch<float, __nv_bfloat16>(a, q.g, backward, s)
                                  : launch<float, __half>(a, q.g, backward, s);
  return d.dtype == PESQ_BF16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, q.g, backward, s)
                              : launch<__half, __half>(a, q.g, backward, s);
}

}  // namespace

extern "C" {

int pesq_norm_join_forward(const pesq_norm_join_desc* d, void* stream, void* out_stream, void* normed) {
  if (const int status = check(d)) return status;
  if (!d->stream.data || !d->pre || !normed || (d->block.data && (!d->post || !out_stream)))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL operand");
  Plan q = plan(*d, false, nullptr, nullptr);
  q.g.wide = q.g.wide && wide(out_stream) && wide(normed);
  Args a{};
  fill(a, *d, q);
  a.out_stream = out_stream;
  a.out_normed = normed;
  const cudaError_t e = run(a, q, *d, false, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

int pesq_norm_join_workspace(const pesq_norm_join_desc* d, size_t* bytes) {
  if (!bytes) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check(d)) return status;
  *bytes = part_bytes(*d) * 3;
  return PESQ_OK;
}

int pesq_norm_join_backward(const pesq_norm_join_desc* d, void* stream, pesq_stream dstream, pesq_stream dnormed,
                            void* dx, void* dblock, void* dgate, float* dpost, float* dpre, float* dscale,
                            void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (!d->stream.data || !d->pre || !dx || !dpre || (d->block.data && (!d->post || !dblock || !dpost)) ||
      (d->gate.data && !dgate) || (d->block.data && d->scale && !dscale))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL operand");
  if (!workspace || workspace_bytes < part_bytes(*d) * 3 || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  Plan q = plan(*d, true, &dstream, &dnormed);
  q.g.wide = q.g.wide && wide(dx) && wide(dblock) && wide(dgate);
  Args a{};
  fill(a, *d, q);
  a.dstream = rows_of(dstream);
  a.dnormed = rows_of(dnormed);
  a.dx = dx;
  a.dblock = d->block.data ? dblock : nullptr;
  a.dgate = d->gate.data && !d->gate_shared ? dgate : nullptr;
  char* ws = static_cast<char*>(workspace);
  a.part_pre = reinterpret_cast<float*>(ws);
  a.part_u = d->block.data ? reinterpret_cast<float*>(ws + part_bytes(*d)) : nullptr;
  a.part_gate = d->gate.data && d->gate_shared ? reinterpret_cast<float*>(ws + 2 * part_bytes(*d)) : nullptr;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = run(a, q, *d, true, s);
  if (e == cudaSuccess) {
    SumArgs t{};
    t.pre = a.part_pre;
    t.u = a.part_u;
    t.gate = a.part_gate;
    t.post = d->post;
    t.scale = d->scale;
    t.dpre = dpre;
    t.dpost = dpost;
    t.dscale = d->scale ? dscale : nullptr;
    t.dgate = dgate;
    t.rows = q.g.blocks;
    t.per_item = q.units;
    t.width = (int)d->width;
    t.dtype = d->dtype;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.blockDim = dim3(32, kSumRows);
    c.stream = s;
    c.attrs = &at;
    c.numAttrs = 1;
    const int64_t sums = 2 + (a.part_gate ? q.batch : 0);
    for (; e == cudaSuccess && t.first < sums; t.first += kMostSums) {
      c.gridDim = dim3((unsigned)((d->width + 31) / 32), (unsigned)std::min<int64_t>(sums - t.first, kMostSums));
      e = cudaLaunchKernelEx(&c, vectors_kernel, t);
    }
  }
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
