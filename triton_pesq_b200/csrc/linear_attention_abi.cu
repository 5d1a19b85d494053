// C ABI of the linear attention: checks, geometry, workspace, and the sums of the decays' gradients.
#include <cuda_runtime.h>

#include <algorithm>

#include "linear_attention.cuh"

using namespace pesq::lattn;
using pesq::set_error;

namespace pesq {
namespace lattn {
extern template cudaError_t forward_of<float>(const Args&, const Geometry&, Kind, cudaStream_t);
extern template cudaError_t forward_of<__nv_bfloat16>(const Args&, const Geometry&, Kind, cudaStream_t);
extern template cudaError_t forward_of<__half>(const Args&, const Geometry&, Kind, cudaStream_t);
extern template cudaError_t backward_of<float>(const Args&, const Geometry&, cudaStream_t);
extern template cudaError_t backward_of<__nv_bfloat16>(const Args&, const Geometry&, cudaStream_t);
extern template cudaError_t backward_of<__half>(const Args&, const Geometry&, cudaStream_t);
}  // namespace lattn
}  // namespace pesq

namespace {

constexpr int kMaxWidth = 128;  // of keys and of values
constexpr int kFewSteps = 8;    // that single steps take, where no backward follows
constexpr int kFewChunks = 6;   // that are not cut in parts
constexpr int kRagged = 4;
constexpr int kFewParts = 4;    // that make the states they begin from themselves, without a join
constexpr int kJoinThreads = 256;

// The decay's gradient of a head: the chunks' sums of its rows, in a fixed order
constexpr int kSumThreads = 256;
__global__ void __launch_bounds__(kSumThreads) decay_kernel(const double* parts, float* out, int64_t batch, int heads, int chunks) {
  __shared__ double s[kSumThreads];
  const int head = blockIdx.x;
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < batch * chunks; i += kSumThreads) {
    const int64_t b = i / chunks;
    v += parts[(b * heads + head) * chunks + (i - b * chunks)];
  }
  s[threadIdx.x] = v;
  __syncthreads();
  for (int n = kSumThreads / 2; n > 0; n >>= 1) {
    if (threadIdx.x < n) s[threadIdx.x] += s[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[head] = (float)s[0];
}

int64_t element(int dtype) { return dtype == PESQ_F32 ? 4 : 2; }
int padded(int64_t n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }

int check(const pesq_linear_attention_desc* d) {
  if (!d) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL descriptor");
  if (d->batch < 1 || d->steps < 1 || d->heads < 1 || d->key < 1 || d->value < 1)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "batch, steps, heads, key and value must be at least 1");
  if (d->key > kMaxWidth || d->value > kMaxWidth)
    return set_error(PESQ_ERR_UNSUPPORTED, "keys and values of at most 128 channels");
  if (d->dtype < PESQ_F32 || d->dtype > PESQ_F16) return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown type");
  if (!(d->scale - d->scale == 0.0f)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (d->batch > INT32_MAX || d->heads > INT32_MAX || d->batch * d->heads > 1 << 22 || d->steps > INT32_MAX)
    return set_error(PESQ_ERR_UNSUPPORTED, "more than 2^22 rows or 2^31 - 1 steps in a call");
  return PESQ_OK;
}

struct Plan {
  Geometry g;
  int chunks, parts, part_chunks, slices;
  int64_t rows, whole;  // of them not cut
  size_t starts, factors, sums;  // bytes of the workspace's pieces
  size_t bytes() const { return starts + factors + sums; }
};

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// CTAs of a kernel that an SM holds: what their shared memory leaves, and their registers
int resident(int dtype, const Geometry& g, bool backward) {
  const int size = (int)element(dtype), pad = size == 2 ? 8 : 4;
  const bool planes = dtype == PESQ_BF16 && !(backward && g.dk * g.dv == 128 * 128);
  const int state = planes ? (backward ? 3 : 2) * g.dk * (g.dv + 8) * 2 : g.dk * (g.dv + 4) * 4, sums = 60 * g.chunk;
  const int wide = g.dk > 64 || (backward && g.dv > 64);
  int bytes;
  if (backward) {
    bytes = 2 * g.chunk * (g.dk + g.dv + 2 * pad) * size + 2 * state + sums;
  } else {
    const int tiles = g.chunk * (2 * g.dk + g.dv + 3 * pad) * size;
    bytes = (2 * tiles + state + 40 * g.chunk <= 75 << 10 ? 2 : 1) * tiles + state + 40 * g.chunk;
  }
  return std::max(1, std::min((228 << 10) / (bytes + 1024), (backward ? 2 : 3) - wide));
}

// Rows are cut in parts, as many as the device holds at once, where that is four times the rows or more forward
// and twice backward: the parts' sweep and join take about 0.6 of a forward's time and 0.3 of a backward's, and some
// 10 us (12 x 8 rows of 500 steps of 64 x 64 in bfloat16: one part 43 us, four 42; 128 rows: 43 and three 58; 16: 41 and eight 24).
// Rows beyond full rounds of the device are cut by the same rule, and the others walked whole beside them (896 rows are six a SM
// and eight more, bfloat16: a round of their own takes 8 % longer forward and 7 % backward than cut).
// Rows of different lengths are cut four times as often, since parts past a row's end leave their place to others (30
// rows of up to 4001 steps of 96 x 128 in float16, trained: parts for one filling 953 us, for four 594).
Plan plan(const pesq_linear_attention_desc& d, bool backward) {
  Plan q{};
  q.rows = d.batch * d.heads;
  const int dk = padded(d.key), dv = padded(d.value);
  q.g.dk = dk;
  q.g.dv = backward ? dv : std::min(dv, 64);
  q.slices = dv / q.g.dv;
  q.g.chunk = chunk_of(d.dtype, dk, dv);
  q.chunks = (int)((d.steps + q.g.chunk - 1) / q.g.chunk);
  const int64_t hold = 148 * resident(d.dtype, q.g, backward) / q.slices;  // rows that the device holds at once
  int64_t last = q.rows < hold ? q.rows : d.lengths ? 0 : q.rows % hold;
  int64_t parts = 1;
  if (q.chunks >= kFewChunks && last > 0 && hold / last >= (backward ? 2 : 4))
    parts = std::min<int64_t>((d.lengths ? kRagged : 1) * (hold / last), q.chunks);
  q.part_chunks = (int)((q.chunks + parts - 1) / parts);
  q.parts = (q.chunks + q.part_chunks - 1) / q.part_chunks;
  if (q.parts == 1) last = 0;
  q.whole = q.rows - last;
  q.g.blocks = (q.whole + last * q.parts) * q.slices;
  if (q.parts > 1) {
    q.starts = round16((size_t)last * q.parts * dk * dv * 4);
    q.factors = round16((size_t)last * q.parts * 4);
  }
  if (backward && d.decay_shared) q.sums = round16((size_t)q.rows * q.chunks * 8);
  return q;
}

size_t kept_size(const pesq_linear_attention_desc& d) {
  const Plan q = plan(d, false);
  return (size_t)q.rows * q.chunks * kept_bytes(padded(d.key), padded(d.value));
}

Operand operand(const pesq_heads& s, const pesq_linear_attention_desc& d, int64_t width) {
  Operand o{s.data, s.batch_stride, s.step_stride, s.head_stride, 0};
  const int64_t size = element(d.dtype);
  const int64_t all = (int64_t)reinterpret_cast<uintptr_t>(s.data) | width * size | (d.batch > 1 ? s.batch_stride * size : 0) |
                      (d.steps > 1 ? s.step_stride * size : 0) | (d.heads > 1 ? s.head_stride * size : 0);
  o.unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
  return o;
}

Args arguments(const pesq_linear_attention_desc& d, const Plan& q, void* workspace) {
  Args a{};
  a.q = operand(d.q, d, d.key);
  a.k = operand(d.k, d, d.key);
  a.v = operand(d.v, d, d.value);
  a.decay = d.log_decay;
  a.decay_sb = d.decay_shared ? 0 : d.decay_batch_stride;
  a.decay_st = d.decay_shared ? 0 : d.decay_step_stride;
  a.decay_sh = d.decay_head_stride;
  a.reset = d.reset;
  a.reset_sb = d.reset_batch_stride;
  a.reset_st = d.reset_step_stride;
  a.lengths = d.lengths;
  a.state = d.state;
  a.steps = d.steps;
  a.heads = (int)d.heads;
  a.key = (int)d.key;
  a.value = (int)d.value;
  a.reverse = d.reverse != 0;
  a.scale = d.scale;
  a.chunks = q.chunks;
  a.parts = q.parts;
  a.part_chunks = q.part_chunks;
  a.whole = q.whole;
  a.slices = q.slices;
  a.joined = q.parts > kFewParts;
  char* ws = static_cast<char*>(workspace);
  a.starts = reinterpret_cast<float*>(ws);
  a.factors = reinterpret_cast<float*>(ws + q.starts);
  a.chunk_ddecay = q.sums ? reinterpret_cast<double*>(ws + q.starts + q.factors) : nullptr;
  return a;
}

cudaError_t forward(const Args& a, const Geometry& g, int dtype, Kind kind, cudaStream_t s) {
  return dtype == PESQ_F32    ? forward_of<float>(a, g, kind, s)
         : dtype == PESQ_BF16 ? forward_of<__nv_bfloat16>(a, g, kind, s)
                              : forward_of<__half>(a, g, kind, s);
}

// the states that the parts begin from
cudaError_t sweep(Args a, const Plan& q, int dtype, bool backward, cudaStream_t s) {
  Geometry g = q.g;
  const int dv = q.g.dv * q.slices;
  g.dv = std::min(dv, 64);
  a.slices = dv / g.dv;
  g.blocks = (q.rows - q.whole) * q.parts * a.slices;
  cudaError_t e = forward(a, g, dtype, backward ? kSweepBackward : kSweep, s);
  if (e != cudaSuccess) return e;
  if (!a.joined) return cudaSuccess;
  const int64_t per = ((int64_t)g.dk * dv + kJoinThreads - 1) / kJoinThreads;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)((q.rows - q.whole) * per));
  c.blockDim = dim3(kJoinThreads);
  c.stream = s;
  c.attrs = &at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, join_kernel<kJoinThreads>, a, g.dk, dv, (int)backward);
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
int check_operands(const pesq_linear_attention_desc* d) {
  if (!d->q.data || !d->k.data || !d->v.data || !d->log_decay) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL operand");
  const int64_t size = element(d->dtype);
  if (!aligned(d->q.data, size) || !aligned(d->k.data, size) || !aligned(d->v.data, size) || !aligned(d->log_decay, 4) ||
      !aligned(d->state, 4) || !aligned(d->lengths, 8))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "an operand that is not aligned to its type");
  return PESQ_OK;
}
// A dense result, whose rows of even width are stored two elements at a time
bool fits(const void* result, const pesq_linear_attention_desc& d, int64_t width) {
  return aligned(result, element(d.dtype) * (width % 2 == 0 ? 2 : 1));
}
int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  return PESQ_OK;
}

}  // namespace

extern "C" {

int pesq_linear_attention_sizes(const pesq_linear_attention_desc* d, size_t* forward, size_t* kept, size_t* backward) {
  if (!forward || !kept || !backward) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check(d)) return status;
  *forward = plan(*d, false).bytes();
  *kept = kept_size(*d);
  *backward = plan(*d, true).bytes();
  return PESQ_OK;
}

int pesq_linear_attention_forward(const pesq_linear_attention_desc* d, void* stream, void* y, float* last, void* kept,
                                  size_t kept_bytes, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (const int status = check_operands(d)) return status;
  if (!y) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL result");
  if (!fits(y, *d, d->value))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "y has to be aligned to its type, and where its width is even to two elements");
  if (!aligned(last, 4)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "the last state is not aligned to its type");
  if (kept && (kept_bytes < kept_size(*d) || reinterpret_cast<uintptr_t>(kept) % 16))
    return set_error(PESQ_ERR_WORKSPACE, "room for the kept states too small or not 16-byte aligned");
  Plan q = plan(*d, false);
  if (const int status = check_workspace(workspace, workspace_bytes, q.bytes())) return status;
  Args a = arguments(*d, q, workspace);
  a.y = y;
  a.last = last;
  a.kept = kept;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (!kept && d->steps <= kFewSteps) {
    Geometry g = q.g;
    g.blocks = q.rows * ((d->value + kStepColumns - 1) / kStepColumns);
    e = forward(a, g, d->dtype, kSteps, s);
  } else {
    if (q.parts > 1) e = sweep(a, q, d->dtype, false, s);
    if (e == cudaSuccess) e = forward(a, q.g, d->dtype, kForward, s);
  }
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

int pesq_linear_attention_backward(const pesq_linear_attention_desc* d, void* stream, const void* kept, size_t kept_bytes,
                                   pesq_heads dy, const float* dlast, void* dq, void* dk, void* dv, float* ddecay,
                                   float* dstate, void* workspace, size_t workspace_bytes) {
  if (const int status = check(d)) return status;
  if (const int status = check_operands(d)) return status;
  if (!dy.data || !dq || !dk || !dv || !ddecay) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL operand");
  if (!aligned(dy.data, element(d->dtype)) || !aligned(dlast, 4) || !aligned(ddecay, 4) || !aligned(dstate, 4))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "an operand that is not aligned to its type");
  if (!fits(dq, *d, d->key) || !fits(dk, *d, d->key) || !fits(dv, *d, d->value))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "a gradient has to be aligned to its type, and where its width is even to two elements");
  if (!kept || kept_bytes < kept_size(*d) || reinterpret_cast<uintptr_t>(kept) % 16)
    return set_error(PESQ_ERR_WORKSPACE, "kept states missing, too small or not 16-byte aligned");
  Plan q = plan(*d, true);
  if (const int status = check_workspace(workspace, workspace_bytes, q.bytes())) return status;
  Args a = arguments(*d, q, workspace);
  a.dy = operand(dy, *d, d->value);
  a.kept = const_cast<void*>(kept);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.ddecay = d->decay_shared ? nullptr : ddecay;
  a.dlast = dlast;
  a.dstate = dstate;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = q.parts > 1 ? sweep(a, q, d->dtype, true, s) : cudaSuccess;
  if (e == cudaSuccess)
    e = d->dtype == PESQ_F32    ? backward_of<float>(a, q.g, s)
        : d->dtype == PESQ_BF16 ? backward_of<__nv_bfloat16>(a, q.g, s)
                                : backward_of<__half>(a, q.g, s);
  if (e == cudaSuccess && d->decay_shared) {
    decay_kernel<<<(unsigned)d->heads, kSumThreads, 0, s>>>(a.chunk_ddecay, ddecay, d->batch, (int)d->heads, q.chunks);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
