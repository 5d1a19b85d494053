// C ABI of the layer norm: checks, geometry, workspace, and the sums of the vectors' gradients.
#include <cuda_runtime.h>

#include <algorithm>

#include "layer_norm.cuh"

using namespace pesq::lnorm;
using pesq::set_error;

namespace pesq {
namespace lnorm {
extern template cudaError_t launch<float, float>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<__nv_bfloat16, __nv_bfloat16>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<__half, __half>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<float, __nv_bfloat16>(const Args&, const Geometry&, bool, cudaStream_t);
extern template cudaError_t launch<float, __half>(const Args&, const Geometry&, bool, cudaStream_t);
}  // namespace lnorm
}  // namespace pesq

namespace {

constexpr int kMaxWidth = 8192;          // one CTA of 256 threads holds a row
constexpr int64_t kMaxVector = 1 << 20;  // heads times channels

// Columns of the CTAs' sums, in a fixed order: 32 columns a block, every thread a stride of the rows, then a tree.
// blockIdx.y: the weight's, the bias'
struct SumArgs {
  const float* part[2];
  float* out[2];
  int64_t rows, columns;
};
constexpr int kSumRows = 32;
__global__ void __launch_bounds__(32 * kSumRows) sums_kernel(const __grid_constant__ SumArgs p) {
  __shared__ float s[kSumRows][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  const float* part = p.part[blockIdx.y];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the kernel before, which this one is launched close to
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < p.columns) {
    int64_t r = threadIdx.y;
    for (; r + 3 * kSumRows < p.rows; r += 4 * kSumRows) {
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += part[(r + k * kSumRows) * p.columns + c];
    }
    for (; r < p.rows; r += kSumRows) acc[0] += part[r * p.columns + c];
  }
  s[threadIdx.y][threadIdx.x] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
  __syncthreads();
  if (threadIdx.y != 0 || c >= p.columns) return;
  float v = 0.0f;
#pragma unroll
  for (int k = 0; k < kSumRows; ++k) v += s[k][threadIdx.x];
  p.out[blockIdx.y][c] = v;
}

int64_t element(int dtype) { return dtype == PESQ_F32 ? 4 : 2; }

int check(const pesq_layer_norm_desc* d) {
  if (!d) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL descriptor");
  if (d->batch < 1 || d->steps < 1 || d->heads < 1 || d->width < 1)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "batch, steps, heads and width must be at least 1");
  if (d->width > kMaxWidth) return set_error(PESQ_ERR_UNSUPPORTED, "at most 8192 channels");
  if (d->heads > kMaxVector / d->width) return set_error(PESQ_ERR_UNSUPPORTED, "at most 2^20 weights");
  if (d->dtype < PESQ_F32 || d->dtype > PESQ_F16 || d->out_dtype < PESQ_F32 || d->out_dtype > PESQ_F16 ||
      (d->dtype != PESQ_F32 && d->dtype != d->out_dtype))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "the result is of the input's type, or in 16 bits beside float32");
  if (!(d->eps >= 0.0f)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "eps must not be negative");
  if (d->batch > INT32_MAX || d->steps > INT64_C(1) << 31 || d->batch * d->steps > INT64_C(1) << 40)
    return set_error(PESQ_ERR_UNSUPPORTED, "too many rows for one launch");
  return PESQ_OK;
}

// To its type, which is all that channel by channel wants
bool aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % element(dtype) == 0; }
int check_operands(const pesq_layer_norm_desc* d) {
  if (!d->x.data || !d->weight) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL operand");
  if (!aligned(d->x.data, d->dtype) || !aligned(d->weight, PESQ_F32) || !aligned(d->bias, PESQ_F32))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "an operand that is not aligned to its type");
  return PESQ_OK;
}

bool joined(const pesq_heads& s, const pesq_layer_norm_desc& d) {
  return !s.data || d.batch == 1 || s.batch_stride == d.steps * s.step_stride;
}
bool wide(const pesq_heads& s, const pesq_layer_norm_desc& d, int dtype) {
  const int64_t unit = 16 / element(dtype);
  return !s.data || (reinterpret_cast<uintptr_t>(s.data) % 16 == 0 && (d.batch == 1 || s.batch_stride % unit == 0) &&
                     (d.steps == 1 || s.step_stride % unit == 0) && (d.heads == 1 || s.head_stride % unit == 0));
}
bool wide(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Threads of a row, and eights of channels of each.  Above a warp any number of warps that keeps few lanes idle, not a power of two
// (24006 x 1155 float32 to float16: three warps 40 us forward and 60 backward, four 47 and 74; 1160, of 16 bytes: three warps of two
// eights 38 and 55, two of four 39 and 63)
void team_of(int64_t width, Geometry& g) {
  const int most = most_groups(g.wide);
  g.team = 4, g.groups = 1;
  while (g.team * g.groups * kEach < width && (g.team < 32 || g.groups < most)) (g.team < 32 ? g.team : g.groups) *= 2;
  if (g.team * g.groups * kEach >= width) return;
  for (const int warps : {2, 3, 4, 5, 6, 8, 12, 16}) {
    g.team = 32 * warps;
    if (g.team * g.groups * kEach >= width) break;
  }
  if (g.groups == 4 && width <= 3 * 32 * 2 * kEach) g.team = 96, g.groups = 2;
}

struct Plan {
  Geometry g;
  int64_t batch, steps, units, span;
  int block_heads, head_blocks;
};

// As many CTAs as the device holds at once, each with its share of the rows, but none with less than a row a team.
// A CTA's teams take the heads side by side: of the numbers of heads that leave the fewest teams idle the largest, so that
// neighbouring heads, whose rows are neighbours in memory, are read together.
void share(const pesq_layer_norm_desc& d, bool backward, Plan& q) {
  team_of(d.width, q.g);
  const int threads = threads_of(q.g.team), teams = threads / q.g.team;
  double best = -1.0;
  for (int h = 1; h <= std::min<int64_t>(teams, d.heads); ++h) {
    const int64_t blocks = (d.heads + h - 1) / h;
    const double busy = (double)(teams / h * h) / teams * (double)d.heads / (double)(blocks * h);
    if (busy >= best - 1e-9) best = busy, q.block_heads = h, q.head_blocks = (int)blocks;
  }
  const int slots = teams / q.block_heads;
  const int64_t rows = d.batch * d.steps;
  const int64_t most = std::max<int64_t>(1, 148 * ctas(backward, q.g.wide, q.g.team, q.g.groups) / q.head_blocks);
  const int64_t units = std::min<int64_t>(most, (rows + slots - 1) / slots);
  q.span = (rows + units - 1) / units;
  q.units = (rows + q.span - 1) / q.span;
  q.g.blocks = q.units * q.head_blocks;
}

Plan plan(const pesq_layer_norm_desc& d, bool backward, const pesq_heads* dy, const void* result) {
  Plan q{};
  const pesq_heads none{nullptr, 0, 0, 0};
  const pesq_heads& g = dy ? *dy : none;
  const bool flat = joined(d.x, d) && joined(g, d);
  q.batch = flat ? 1 : d.batch;
  q.steps = flat ? d.batch * d.steps : d.steps;
  q.g.wide = d.width % kEach == 0 && wide(d.x, d, d.dtype) && wide(g, d, d.out_dtype) && wide(d.weight) && wide(d.bias) &&
             wide(result);
  share(d, backward, q);
  return q;
}

// of the CTAs' sums of one vector, however the operands lie
size_t part_bytes(const pesq_layer_norm_desc& d) {
  int64_t units = 0;
  for (const bool wide : {false, true}) {
    Plan q{};
    q.g.wide = wide;
    share(d, true, q);
    units = std::max(units, q.units);
  }
  return ((size_t)units * d.heads * d.width * 4 + 15) / 16 * 16;
}

Strided rows_of(const pesq_heads& s) { return {s.data, s.batch_stride, s.step_stride, s.head_stride}; }

Args arguments(const pesq_layer_norm_desc& d, const Plan& q) {
  Args a{};
  a.x = rows_of(d.x);
  a.weight = d.weight;
  a.bias = d.bias;
  a.batch = q.batch;
  a.steps = q.steps;
  a.heads = (int)d.heads;
  a.width = (int)d.width;
  a.block_heads = q.block_heads;
  a.head_blocks = q.head_blocks;
  a.units = q.units;
  a.span = q.span;
  a.eps = d.eps;
  return a;
}

cudaError_t run(const Args& a, const Plan& q, const pesq_layer_norm_desc& d, bool backward, cudaStream_t s) {
  if (d.dtype == PESQ_F32)
    return d.out_dtype == PESQ_F32    ? launch<float, float>(a, q.g, backward, s)
           : d.out_dtype == PESQ_BF16 ? launch<float, __nv_bfloat16>(a, q.g, backward, s)
                                      : launch<float, __half>(a, q.g, backward, s);
  return d.dtype == PESQ_BF16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, q.g, backward, s)
                              : launch<__half, __half>(a, q.g, backward, s);
}

}  // namespace

extern "C" {

int pesq_layer_norm_forward(const pesq_layer_norm_desc* d, void* stream, void* y) {
  if (const int status = check(d)) return status;
  if (const int status = check_operands(d)) return status;
  if (!y) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL result");
  if (!aligned(y, d->out_dtype)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "a result that is not aligned to its type");
  const Plan q = plan(*d, false, nullptr, y);
  Args a = arguments(*d, q);
  a.y = y;
  const cudaError_t e = run(a, q, *d, false, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

int pesq_layer_norm_workspace(const pesq_layer_norm_desc* d, size_t* bytes) {
  if (!bytes) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check(d)) return status;
  *bytes = part_bytes(*d) * 2;
  return PESQ_OK;
}

int pesq_layer_norm_backward(const pesq_layer_norm_desc* d, void* stream, pesq_heads dy, void* dx, float* dweight,
                             float* dbias, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (const int status = check_operands(d)) return status;
  if (!dy.data || !dx || !dweight || (d->bias && !dbias)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL operand");
  if (!aligned(dy.data, d->out_dtype) || !aligned(dx, d->dtype) || !aligned(dweight, PESQ_F32) || !aligned(dbias, PESQ_F32))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "a gradient that is not aligned to its type");
  if (!workspace || workspace_bytes < part_bytes(*d) * 2 || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  const Plan q = plan(*d, true, &dy, dx);
  Args a = arguments(*d, q);
  a.dy = rows_of(dy);
  a.dx = dx;
  a.part_weight = static_cast<float*>(workspace);
  a.part_bias = d->bias ? reinterpret_cast<float*>(static_cast<char*>(workspace) + part_bytes(*d)) : nullptr;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = run(a, q, *d, true, s);
  if (e == cudaSuccess) {
    SumArgs t{};
    t.part[0] = a.part_weight;
    t.part[1] = a.part_bias;
    t.out[0] = dweight;
    t.out[1] = dbias;
    t.rows = q.units;
    t.columns = d->heads * d->width;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)((t.columns + 31) / 32), d->bias ? 2 : 1);
    c.blockDim = dim3(32, kSumRows);
    c.stream = s;
    c.attrs = &at;
    c.numAttrs = 1;
    e = cudaLaunchKernelEx(&c, sums_kernel, t);
  }
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
