// Orthogonalised updates of matrices (Muon), all matrices together.
//
// With g the gradient (times grad_scale) of a matrix p:
//   m = b m + (1 - b) g,   U = b m + (1 - b) g (or m),   X = U / max(|U|, eps)
//   `steps` times:  A = X X^T,  X = a X + (b A + c A A) X = (a + b A + c A A) X
//   p = p (1 - lr wd) - lr adjust X
// on the shorter side of the matrix first (X is n x m, n <= m), so that A is small.
//
// Numbers.  The iteration is meant for 3.4 times as large small singular values a step, 485 times in five, and with
// them whatever rounding added to them: operands of 8 or 11 bits would leave percents in the result.  So every operand is two float16
// terms, hi + lo (22 bits, 2^-23 off), and every product three instructions (hi hi, hi lo, lo hi) into one float32
// accumulator.  Values are kept times 2^10: elements of X and A are at most about 1.2, those of the polynomial about 8, for the
// usual coefficients, far from float16's largest, and the lo term of an element of 2^-10 still has its bits.
// The accumulator of the instruction cuts off what it does not hold instead of rounding it, which adds up over a long
// contraction (2.3e-5 of the result of a 385 x 1155 matrix, 5.0e-5 of 1280 x 3840).  So it sums 64 columns alone (of narrow matrices
// 32 or 16), and the warps that read it add those sums in registers, rounded (2.5e-6 and 1.5e-6; with 128 columns 4.3e-6 and 2.8e-6 in
// 4 % less time, with 32 1.6e-6 of 385 x 1155 in 20 % more; float32 products 2.8e-6 and 3.6e-6).
//
// Products run on tcgen05 with the accumulator in tensor memory, in tiles of 128 x 128.  Matrices lie in the workspace as the
// tiles that the instruction reads from shared memory: 128 rows of 64 columns in the 128-byte swizzle, hi and lo
// behind each other, zeros past the matrix' edge.  So an operand is a plain bulk copy of 32 KB, odd sizes need nothing
// anywhere, and the one layout serves X X^T (64 columns of the contraction side by side) and B X (X's rows are the contraction:
// the same bytes read as a transposed operand).  A and the polynomial are symmetric: the tiles below and on the diagonal are
// computed, and written mirrored too, which takes 10 n^3 operations of a square matrix' step instead of 14.  Beside A goes
// b + c A, so that the polynomial but for its a on the diagonal is one product of the two.
//
// A CTA takes tiles in turn: a thread issues copies three stages ahead, a thread issues products, sixteen warps
// empty the accumulators, of which there are two, so that a tile's end overlaps the next one's products (each a quarter of
// the columns: four warps with all of them took twice as long over a small model's tiles).  All products of
// a call are one cooperative launch, whose CTAs wait for one another between the products of a step (15 launches of a
// small model's step took 230 us of the host's time).  The bound is what a product's operands take: 128 x 128 x 16
// reads 8 KB of shared memory in its 64 cycles, all that it gives, while 64 KB are copied in for a stage's 3 x 2.1 MFLOP beside.
// 4096 x 4096 alone runs at 990 TFLOP/s of the three products, 10 TB/s out of the L2 cache; pairs of CTAs on 256 x 256, with half of those
// copies, at 1030, but slower in all of a model's sizes (3.08 ms for 2.53).  All waits are
// bounded; one that runs out sets an error word and the CTA returns.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <utility>
#include <vector>

#include "../../include/pesq_cuda.h"
#include "common.cuh"
#include "train.cuh"

namespace {

using namespace pesq::train;
using pesq::bulk_g2s;
using pesq::mbar_arrive_expect_tx;
using pesq::mbar_wait;
using pesq::set_error;
using pesq::smem_u32;

constexpr int kTile = 128, kDepth = 64;               // rows of a tile, columns of the contraction in a stage
constexpr int kPlane = kTile * kDepth * 2;            // bytes of a tile's hi or lo terms
constexpr int kPair = 2 * kPlane;
constexpr int kStages = 3, kStage = 2 * kPair;        // both operands
constexpr int kReaders = 16;                          // warps of results: four for each quarter of the columns
constexpr int kThreads = 64 + 32 * kReaders;          // copies, products, results
constexpr int kShared = kStages * kStage + 1024;      // (aligned to 1024 in the kernel)
constexpr float kScale = 1024.0f;                     // of what is kept
constexpr int kMost = 32768;                          // rows or columns
constexpr int kItems = 128;                           // matrices of a launch
constexpr int kNarrowStages = 3;                      // of one operand, beside two squares, of the narrow kernel
constexpr int kNarrowShared = 4 * kPair + kNarrowStages * kPair + 1024;
constexpr int kNarrowTiles = 8;                       // across, of the matrices that it takes
constexpr int64_t kGroupBytes = INT64_C(256) << 20;   // of their workspace, where there are several
constexpr int kNormValues = 8192;                     // of a block of the first pass
constexpr int kPrepThreads = 256;

enum Mode { kGram, kPolynomial, kUpdate, kLast };

struct Item {
  float* param;      // Muon; null where X itself is the result
  float* momentum;
  const void* grad;  // or the matrix to orthogonalise
  void* out;         // the parameter's copy in the gradient's type, or the result, or null
  int64_t x[2], a, c, b;  // workspace offsets of X (before and after a step), A, what it is multiplied with, the polynomial
  int rows, cols;
  int n, m, nt, mt;    // shorter and longer side, in tiles of 128
  int flipped;         // X is the matrix' transpose
  int first_norm, norms;                     // of the blocks, of the first pass
  int first_prep, first_square, first_wide;  // tile, of the second pass, of symmetric products, of updates
  float step;          // lr times adjust
};
struct Call {
  int count, dtype, nesterov, steps;
  int squares, wides;  // tiles of symmetric products, of updates
  char* ws;
  double* norms;       // sums of squares of the first pass' blocks
  uint32_t* arrived;   // CTAs at the ends of the products so far
  const float* grad_scale;
  float beta, rest, decay;  // momentum, 1 - momentum, 1 - lr wd
  float eps, ca, cb, cc;
  uint32_t* error;
};
// Kernel parameters; a launch of few matrices takes the short table
template <int N>
struct Args : Call {
  Item item[N];
};
constexpr int kShort = 16;
static_assert(sizeof(Args<kItems>) < 32000, "kernel parameters");

__device__ uint32_t g_error;

// f(a value of the gradients' type)
template <class F>
__device__ __forceinline__ void with_type(int dtype, F f) {
  if (dtype == PESQ_F32)
    f(float{});
  else if (dtype == PESQ_BF16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}
// the last item whose first is not above at
template <int Item::*kFirst, int N>
__device__ __forceinline__ int find(const Args<N>& p, int at) {
  int lo = 0, hi = p.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.item[mid].*kFirst <= at) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// the factor of the gradients; `skip` where it is not finite
__device__ __forceinline__ float scale_of(const Call& p, bool& skip) {
  const float s = p.grad_scale ? *p.grad_scale : 1.0f;
  skip = !(s - s == 0.0f);
  return s;
}
__device__ __forceinline__ void dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void depend() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------------------- momentum and its norm

// the matrix that is orthogonalised
__device__ __forceinline__ float update_of(const Call& p, float m, float g) { return p.nesterov ? fmaf(p.beta, m, p.rest * g) : m; }

template <int N>
__global__ void __launch_bounds__(kPrepThreads) momentum_kernel(const __grid_constant__ Args<N> p) {
  constexpr int kTogether = 8;  // values of a thread whose loads are on their way together
  __shared__ double s_sum[kPrepThreads / 32];
  dependents();
  depend();
  const Item& it = p.item[find<&Item::first_norm>(p, blockIdx.x)];
  const int64_t numel = (int64_t)it.rows * it.cols, first = (int64_t)(blockIdx.x - it.first_norm) * kNormValues;
  bool skip;
  const float s = scale_of(p, skip);
  double sum = 0.0;
  with_type(p.dtype, [&](auto zero) {
    using G = decltype(zero);
    const G* grad = static_cast<const G*>(it.grad) + first + threadIdx.x;
    float* momentum = it.momentum ? it.momentum + first + threadIdx.x : nullptr;
    const int left = (int)min((int64_t)kNormValues, numel - first) - (int)threadIdx.x;
#pragma unroll 1
    for (int i0 = 0; i0 < kNormValues / kPrepThreads; i0 += kTogether) {
      float g[kTogether], m[kTogether];
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const int at = (i0 + k) * kPrepThreads;
        g[k] = at < left ? widen(grad[at]) : 0.0f;
        m[k] = at < left && momentum ? momentum[at] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const int at = (i0 + k) * kPrepThreads;
        float u = g[k];
        if (momentum) {
          g[k] *= s;
          m[k] = fmaf(p.beta, m[k], p.rest * g[k]);
          if (at < left && !skip) momentum[at] = m[k];
          u = update_of(p, m[k], g[k]);
        }
        if (at < left) sum = fma((double)u, (double)u, sum);
      }
    }
  });
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPrepThreads / 32; ++w) sum += s_sum[w];
    p.norms[blockIdx.x] = sum;
    if (blockIdx.x == 0) *p.arrived = 0;
  }
}

struct alignas(16) Eight {
  uint32_t w[4];  // two float16 each
};
// Eight values as their terms.  The upper term's value is the value's own bits rounded to 11, half away from zero, which a conversion back
// would take twice as long for (conversions are what bounds this); below 2^-14, where float16 holds fewer, the terms are off by up to 2^-25.
__device__ __forceinline__ void split8(const float (&v)[8], Eight& hi, Eight& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = v[2 * j], b = v[2 * j + 1];
    const float x = __uint_as_float((__float_as_uint(a) + 0x1000u) & 0xffffe000u), y = __uint_as_float((__float_as_uint(b) + 0x1000u) & 0xffffe000u);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi.w[j]) : "f"(y), "f"(x));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo.w[j]) : "f"(b - y), "f"(a - x));
  }
}
// where columns 8 chunk .. of a row of a tile's plane lie
__device__ __forceinline__ int at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// X in tiles; a block takes one
template <int N>
__global__ void __launch_bounds__(kPrepThreads) prepare_kernel(const __grid_constant__ Args<N> p) {
  __shared__ double s_sum[kPrepThreads];
  dependents();
  const int index = find<&Item::first_prep>(p, blockIdx.x);
  const Item& it = p.item[index];
  const int tile = blockIdx.x - it.first_prep, rt = tile / (2 * it.mt), ct = tile % (2 * it.mt);
  depend();
  double sum = 0.0;
  for (int i = threadIdx.x; i < it.norms; i += kPrepThreads) sum += p.norms[it.first_norm + i];
  s_sum[threadIdx.x] = sum;
  __syncthreads();
  for (int n = kPrepThreads / 2; n > 0; n >>= 1) {
    if (threadIdx.x < n) s_sum[threadIdx.x] += s_sum[threadIdx.x + n];
    __syncthreads();
  }
  bool skip;
  const float s = scale_of(p, skip);
  const double norm = sqrt(s_sum[0]);
  const float inverse = (float)(1.0 / (norm > p.eps || norm != norm ? norm : (double)p.eps));  // (times 2^10 it may be past float32)
  char* to = p.ws + it.x[0] + (int64_t)tile * kPair;
  with_type(p.dtype, [&](auto zero) {
    using G = decltype(zero);
    const G* grad = static_cast<const G*>(it.grad);
    // neighbouring threads: rows of a flipped matrix, chunks of a row of another
#pragma unroll 2
    for (int i = threadIdx.x; i < kTile * 8; i += kPrepThreads) {
      const int row = it.flipped ? i % kTile : i / 8, chunk = it.flipped ? i / kTile : i % 8;
      const int r = rt * kTile + row, c = ct * kDepth + chunk * 8;
      const int64_t first = it.flipped ? (int64_t)c * it.cols + r : (int64_t)r * it.cols + c, apart = it.flipped ? it.cols : 1;
      float g[8], m[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = r < it.n && c + j < it.m;
        g[j] = in ? widen(grad[first + j * apart]) : 0.0f;
        m[j] = in && it.momentum ? it.momentum[first + j * apart] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = (it.momentum ? update_of(p, m[j], s * g[j]) : g[j]) * inverse * kScale;
        if (!(r < it.n && c + j < it.m)) v[j] = 0.0f;
      }
      Eight hi, lo;
      split8(v, hi, lo);
      *reinterpret_cast<Eight*>(to + at(row, chunk)) = hi;
      *reinterpret_cast<Eight*>(to + kPlane + at(row, chunk)) = lo;
    }
  });
}

// ------------------------------------------------------------------------------------------ products

// An operand in shared memory, 128-byte swizzle.  Rows of 64 columns of the contraction (8 rows are 1024 bytes), or,
// transposed, rows of the contraction of 64 columns each (8 rows are 1024 bytes, the next 64 columns 8192 further).
__device__ __forceinline__ uint64_t descriptor(uint32_t address, bool transposed) {
  const uint64_t leading = transposed ? 8192 >> 4 : 1, stride = 1024 >> 4;
  return (uint64_t)((address & 0x3ffff) >> 4) | leading << 16 | stride << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// f16 operands, f32 accumulator, 128 x 128
constexpr uint32_t kInstruction = 1u << 4 | (kTile / 8) << 17 | (kTile / 16) << 24;
constexpr uint32_t kTransposedB = 1u << 16;

__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void load32(uint32_t (&v)[32], uint32_t address) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(address));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// A tile of a launch: its matrix, its place, and how long its contraction is
struct Tile {
  int index, i, j, depth;
  template <int N>
  __device__ __forceinline__ Tile(const Args<N>& p, int mode, int t) {
    if (mode < kUpdate) {
      index = find<&Item::first_square>(p, t);
      const Item& it = p.item[index];
      t -= it.first_square;
      i = 0;
      while (t > i) t -= ++i;  // rows of 1, 2, 3, ... tiles
      j = t;
      depth = ((mode == kGram ? it.m : it.n) + kDepth - 1) / kDepth;
    } else {
      index = find<&Item::first_wide>(p, t);
      const Item& it = p.item[index];
      t -= it.first_wide;
      i = t % it.nt;
      j = t / it.nt;
      depth = (it.n + kDepth - 1) / kDepth;
    }
  }
};

// Eight columns of a row to a tile, and where mirrored to the tile across the diagonal too, whose rows are the columns here:
// neighbouring lanes, which hold neighbouring rows, exchange halves, so that each stores two columns of one row
__device__ __forceinline__ void put(char* to, char* over, bool mirrored, int row, int col, const float (&v)[8]) {
  Eight plane[2];
  split8(v, plane[0], plane[1]);
  const int lane = threadIdx.x & 31, chunk = col % kDepth / 8, column = row % kDepth & ~1;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    *reinterpret_cast<Eight*>(to + q * kPlane + at(row, chunk)) = plane[q];
    if (!mirrored) continue;
    const uint32_t* words = plane[q].w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, words[j], 1);
      const uint32_t pair = lane & 1 ? __byte_perm(other, words[j], 0x7632) : __byte_perm(words[j], other, 0x5410);
      *reinterpret_cast<uint32_t*>(over + q * kPlane + at(col + 2 * j + (lane & 1), column / 8) + column % 8 * 2) = pair;
    }
  }
}

__device__ __forceinline__ void add_diagonal(float (&v)[8], int at, float x) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j == at) v[j] += x;
}

// What a warp makes of 32 columns of a tile's accumulators: a thread has a row
__device__ __forceinline__ void finish(const Call& p, int mode, int from, const Item& it, const Tile& t, int row, int col,
                                       const float (&acc)[32], bool skip) {
  const int r = t.i * kTile + row, c0 = t.j * kTile + col;
  if (mode == kLast) {
    // (X is the result or its transpose.  All loads before all stores, as they may be the same memory)
    if (r >= it.n || skip) return;
    const int64_t first = it.flipped ? (int64_t)c0 * it.cols + r : (int64_t)r * it.cols + c0, apart = it.flipped ? it.cols : 1;
    const int left = it.m - c0;
    float v[32];
    if (it.param) {
      float* param = it.param + first;
      const bool fours = !it.flipped && left >= 32 && reinterpret_cast<uintptr_t>(param) % 16 == 0;
      if (fours) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 f = *reinterpret_cast<const float4*>(param + k);
          v[k] = f.x, v[k + 1] = f.y, v[k + 2] = f.z, v[k + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = k < left ? param[k * apart] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = fmaf(-it.step, acc[k] * (1.0f / (kScale * kScale)), v[k] * p.decay);
      if (fours) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(param + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (k < left) param[k * apart] = v[k];
      }
      if (!it.out) return;
    } else {
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = acc[k] * (1.0f / (kScale * kScale));
    }
    with_type(p.dtype, [&](auto zero) {
      using G = decltype(zero);
      G* out = static_cast<G*>(it.out) + first;
      if (apart == 1 && left >= 32 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
        constexpr int kEach = 16 / sizeof(G);
#pragma unroll
        for (int k = 0; k < 32; k += kEach) {
          Pack<G, kEach> q;
#pragma unroll
          for (int j = 0; j < kEach; ++j) q.v[j] = narrow<G>(v[k + j]);
          *reinterpret_cast<Pack<G, kEach>*>(out + k) = q;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (k < left) out[k * apart] = narrow<G>(v[k]);
      }
    });
    return;
  }
  const int tiles = mode == kUpdate ? 2 * it.mt : 2 * it.nt;  // side by side
  const int64_t place = ((int64_t)t.i * tiles + t.j * 2 + col / kDepth) * kPair;
  const int64_t across = ((int64_t)t.j * tiles + t.i * 2 + row / kDepth) * kPair;
  const bool mirrored = mode < kUpdate && t.i != t.j;
  char* const to = p.ws + (mode == kGram ? it.a : mode == kPolynomial ? it.b : it.x[from ^ 1]);
  const bool diagonal = mode < kUpdate && t.i == t.j && col == row / 32 * 32 && r < it.n;
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = acc[k + j] * (1.0f / kScale);
    if (mode == kPolynomial && diagonal) add_diagonal(v, row % 32 - k, p.ca * kScale);
    put(to + place, to + across, mirrored, row, col + k, v);
    if (mode == kGram) {  // and what A is multiplied with: b + c A, so that the polynomial's tiles are products alone
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= p.cc;
      if (diagonal) add_diagonal(v, row % 32 - k, p.cb * kScale);
      put(p.ws + it.c + place, p.ws + it.c + across, mirrored, row, col + k, v);
    }
  }
}

// The three products of kCount sixteens of a stage's columns from `first`, to a sum of their own
template <int kCount>
__device__ __forceinline__ void products_of(uint32_t to, uint32_t a, uint32_t b, bool transposed, int first) {
  const uint32_t instruction = kInstruction | (transposed ? kTransposedB : 0);
  // (the lower terms first: what the accumulator cuts off is a share of what it holds)
#pragma unroll
  for (int pair = 0; pair < 3; ++pair) {
#pragma unroll
    for (int s = 0; s < kCount; ++s) {
      const uint32_t as = a + (first + s) * 32 + (pair == 0 ? kPlane : 0), bs = b + (first + s) * (transposed ? 2048 : 32) + (pair == 1 ? kPlane : 0);
      product(to, descriptor(as, false), descriptor(bs, transposed), instruction, pair > 0 || s > 0);
    }
  }
}

// All CTAs of the launch at the same point, what they wrote visible to the copies that they issue next.  False where some
// did not come in time
constexpr uint32_t kPolls = 1u << 21;  // (a second or two)
__device__ __forceinline__ bool meet(uint32_t* arrived, uint32_t want, volatile uint32_t& s_stop) {
  asm volatile("fence.proxy.async;" ::: "memory");
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0 && !s_stop) {
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(arrived) : "memory");
    uint32_t seen = 0;
    for (uint32_t i = 0; i < kPolls; ++i) {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(arrived) : "memory");
      if (seen >= want) break;
    }
    if (seen < want) s_stop = 1;
  }
  __syncthreads();
  asm volatile("fence.proxy.async;" ::: "memory");
  return !s_stop;
}

template <int N>
__global__ void __launch_bounds__(kThreads, 1) products_kernel(const __grid_constant__ Args<N> p) {
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], ready[2], spent[2], drained;
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_stop;
  char* const tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) init(full + s, 1), init(empty + s, 1);
    for (int s = 0; s < 2; ++s) init(ready + s, 1), init(spent + s, kReaders);
    init(&drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_stop = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s_tmem;
  // where the role of this thread is in its ring: copies or products of stages, accumulators
  int stage = 0, half = 0;
  uint32_t parity = warp == 0 ? 1 : 0, half_parity = warp == 1 ? 1 : 0;
  int issued = 0;
  bool good = true, skip;
  scale_of(p, skip);
  uint32_t met = 0;
#pragma unroll 1
  for (int product_index = 0; product_index < 3 * p.steps; ++product_index) {
    const int step = product_index / 3, from = step & 1;
    const int mode = product_index % 3 < 2 ? product_index % 3 : step + 1 < p.steps ? kUpdate : kLast;
    const int total = mode < kUpdate ? p.squares : p.wides;
    const bool wide = mode >= kUpdate;
    if (warp == 0) {
      if (lane == 0) {
        for (int t = blockIdx.x; t < total && good; t += gridDim.x) {
          const Tile tile(p, mode, t);
          const Item& it = p.item[tile.index];
          const bool same = mode == kGram && tile.i == tile.j;
          const int64_t left = mode == kGram ? it.x[from] : mode == kPolynomial ? it.a : it.b;
          const int across = mode == kGram ? 2 * it.mt : 2 * it.nt;
          const char* a = p.ws + left + (int64_t)tile.i * across * kPair;
          const char* b = p.ws + (mode == kPolynomial ? it.c : left) + (int64_t)tile.j * across * kPair;
          for (int k = 0; k < tile.depth; ++k) {
            if (!mbar_wait(empty + stage, parity)) {
              good = false;
              break;
            }
            char* to = tiles + stage * kStage;
            mbar_arrive_expect_tx(full + stage, same ? kPair : 2 * kPair);
            bulk_g2s(to, a + (int64_t)k * kPair, kPair, full + stage);
            if (wide) {
              // 64 rows of two tiles of X side by side
              const char* x = p.ws + it.x[from] + ((int64_t)(k / 2) * 2 * it.mt + tile.j * 2) * kPair + (k & 1) * (kPlane / 2);
              for (int plane = 0; plane < 2; ++plane)
                for (int side = 0; side < 2; ++side)
                  bulk_g2s(to + kPair + plane * kPlane + side * (kPlane / 2), x + side * kPair + plane * kPlane, kPlane / 2, full + stage);
            } else if (!same) {
              bulk_g2s(to + kPair, b + (int64_t)k * kPair, kPair, full + stage);
            }
            if (issued < kStages) ++issued;
            if (++stage == kStages) stage = 0, parity ^= 1;
          }
        }
        if (!good) {  // (what is in flight lands before the CTA ends)
          atomicOr(p.error, 1u);
          s_stop = 1;
          for (int s = 1; s <= issued; ++s) {
            // the copies s stages back, whose phase is that of the parity they were issued with
            const int back = (stage + kStages - s) % kStages;
            mbar_wait(full + back, back < stage ? parity ^ 1 : parity);
          }
        }
      }
    } else if (warp == 1) {
      if (lane == 0) {
        for (int t = blockIdx.x; t < total && good; t += gridDim.x) {
          const Tile tile(p, mode, t);
          const bool same = mode == kGram && tile.i == tile.j;
          for (int k = 0; k < tile.depth; ++k) {
            if (!mbar_wait(spent + half, half_parity) || !mbar_wait(full + stage, parity)) {
              good = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t a = smem_u32(tiles + stage * kStage);
            products_of<kDepth / 16>(tmem + half * kTile, a, same ? a : a + kPair, wide, 0);
            commit(empty + stage);
            commit(ready + half);
            half ^= 1;
            if (half == 0) half_parity ^= 1;
            if (++stage == kStages) stage = 0, parity ^= 1;
          }
        }
        if (!good) {  // (what is issued ends before its memory goes)
          atomicOr(p.error, 2u);
          s_stop = 1;
          commit(&drained);
          mbar_wait(&drained, 0);
        }
      }
    } else {
      const int quarter = warp & 3, col = (warp - 2) / 4 * 32;  // its lanes of tensor memory, and columns
      for (int t = blockIdx.x; t < total && good; t += gridDim.x) {
        const Tile tile(p, mode, t);
        float acc[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[e] = 0.0f;
        for (int k = 0; k < tile.depth; ++k) {
          good = __all_sync(0xffffffffu, mbar_wait(ready + half, half_parity));
          if (!good) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          uint32_t part[32];
          load32(part, tmem + half * kTile + col + ((uint32_t)(quarter * 32) << 16));
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive(spent + half);
          half ^= 1;
          if (half == 0) half_parity ^= 1;
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[e] += __uint_as_float(part[e]);
        }
        if (!good) break;
        finish(p, mode, from, p.item[tile.index], tile, quarter * 32 + lane, col, acc, skip);
      }
      if (!good && lane == 0) {
        atomicOr(p.error, 4u);
        s_stop = 1;
      }
    }
    __syncwarp();
    met += gridDim.x;
    if (product_index + 1 < 3 * p.steps) {
      good = meet(p.arrived, met, s_stop) && good;
      if (s_stop) {
        if (threadIdx.x == 0) atomicOr(p.error, 8u);
        break;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
  }
}

// Eight columns of a row of a square in shared memory: two tiles of 64 columns
__device__ __forceinline__ void put_shared(char* square, int row, int col, const float (&v)[8]) {
  Eight hi, lo;
  split8(v, hi, lo);
  char* to = square + col / kDepth * kPair + at(row, col % kDepth / 8);
  *reinterpret_cast<Eight*>(to) = hi;
  *reinterpret_cast<Eight*>(to + kPlane) = lo;
}

// Sixteens of columns that a narrow matrix' products sum in tensor memory.  What the accumulator cuts off is of the sum's sign, and the
// fewer rows there are, the less of it averages out.  With a stage's four 37 x 225 is 3.4e-6 off (float32 products 1.6e-6), 52 x 725 3.5e-6
// (2.0e-6), 70 x 506 2.8e-6 (1.6e-6), 96 x 288 1.7e-6 (1.5e-6); with two 2.8e-6, 2.3e-6, 1.8e-6 and 1.1e-6, with one 2.0e-6, 1.7e-6, 1.3e-6
// and 8e-7.  A small model's step (96 wide) takes 116 us with four, 124 with two, 146 with one.
__device__ __forceinline__ int narrow_sum(const Item& it) { return it.n <= kDepth ? 1 : 2; }
// Such sums of a contraction over `width` columns: those past the edge are zeros, and not worked on
__device__ __forceinline__ int sums_of(int width, int each) { return (width + 16 * each - 1) / (16 * each); }

template <int N>
__global__ void __launch_bounds__(kThreads, 1) narrow_kernel(const __grid_constant__ Args<N> p) {
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t full[kNarrowStages], empty[kNarrowStages], ready[2], spent[2], made, drained;
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_stop;
  char* const squares = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);  // A, then the polynomial; b + c A
  char* const ring = squares + 4 * kPair;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kNarrowStages; ++s) init(full + s, 1), init(empty + s, 1);
    for (int s = 0; s < 2; ++s) init(ready + s, 1), init(spent + s, kReaders);
    init(&made, kReaders);
    init(&drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_stop = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s_tmem;
  int stage = 0, half = 0, issued = 0;
  uint32_t parity = warp == 0 ? 1 : 0, half_parity = warp == 1 ? 1 : 0, made_parity = 0, met = 0;
  bool good = true, skip;
  scale_of(p, skip);
#pragma unroll 1
  for (int step = 0; step < p.steps; ++step) {
    const int from = step & 1;
    if (warp == 0) {
      if (lane == 0) {
        for (int t = blockIdx.x; t < p.wides && good; t += gridDim.x) {
          const Tile tile(p, kUpdate, t);
          const Item& it = p.item[tile.index];
          const char* x = p.ws + it.x[from];
          const int gram = (it.m + kDepth - 1) / kDepth;
          for (int k = 0; k < gram + tile.depth; ++k) {
            if (!mbar_wait(empty + stage, parity)) {
              good = false;
              break;
            }
            char* to = ring + stage * kPair;
            mbar_arrive_expect_tx(full + stage, kPair);
            if (k < gram) {
              bulk_g2s(to, x + (int64_t)k * kPair, kPair, full + stage);
            } else {  // 64 rows of two tiles of X side by side
              const char* rows = x + (int64_t)tile.j * 2 * kPair + (k - gram) * (kPlane / 2);
              for (int plane = 0; plane < 2; ++plane)
                for (int side = 0; side < 2; ++side)
                  bulk_g2s(to + plane * kPlane + side * (kPlane / 2), rows + side * kPair + plane * kPlane, kPlane / 2, full + stage);
            }
            if (issued < kNarrowStages) ++issued;
            if (++stage == kNarrowStages) stage = 0, parity ^= 1;
          }
        }
        if (!good) {  // (what is in flight lands before the CTA ends)
          atomicOr(p.error, 1u);
          s_stop = 1;
          for (int s = 1; s <= issued; ++s) {
            const int back = (stage + kNarrowStages - s) % kNarrowStages;
            mbar_wait(full + back, back < stage ? parity ^ 1 : parity);
          }
        }
      }
    } else if (warp == 1) {
      if (lane == 0) {
        const uint32_t square = smem_u32(squares);
        for (int t = blockIdx.x; t < p.wides && good; t += gridDim.x) {
          const Tile tile(p, kUpdate, t);
          const Item& it = p.item[tile.index];
          const int each = narrow_sum(it), stage_sums = kDepth / 16 / each;
          // A: X X^T, then the polynomial: A (b + c A), then X': the polynomial times X
          for (int part = 0; part < 3 && good; ++part) {
            const int sums = sums_of(part == 0 ? it.m : it.n, each);
            if (part > 0) {
              good = mbar_wait(&made, made_parity);
              made_parity ^= 1;
            }
            for (int c = 0; c < sums && good; ++c) {
              const int k = c / stage_sums, first = c % stage_sums * each;
              if (part != 1 && first == 0) good = mbar_wait(full + stage, parity);
              good = good && mbar_wait(spent + half, half_parity);
              if (!good) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              const uint32_t own = smem_u32(ring + stage * kPair);
              const uint32_t to = tmem + half * kTile, a = part == 0 ? own : square + k * kPair, b = part == 1 ? square + (2 + k) * kPair : own;
              if (each == 1) products_of<1>(to, a, b, part == 2, first);
              else products_of<2>(to, a, b, part == 2, first);
              if (part != 1 && ((c + 1) % stage_sums == 0 || c + 1 == sums)) {
                commit(empty + stage);
                if (++stage == kNarrowStages) stage = 0, parity ^= 1;
              }
              commit(ready + half);
              half ^= 1;
              if (half == 0) half_parity ^= 1;
            }
          }
        }
        if (!good) {  // (what is issued ends before its memory goes)
          atomicOr(p.error, 2u);
          s_stop = 1;
          commit(&drained);
          mbar_wait(&drained, 0);
        }
      }
    } else {
      const int quarter = warp & 3, col = (warp - 2) / 4 * 32, row = quarter * 32 + lane;
      for (int t = blockIdx.x; t < p.wides && good; t += gridDim.x) {
        const Tile tile(p, kUpdate, t);
        const Item& it = p.item[tile.index];
#pragma unroll 1
        for (int part = 0; part < 3 && good; ++part) {
          const int sums = sums_of(part == 0 ? it.m : it.n, narrow_sum(it));
          float acc[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[e] = 0.0f;
          for (int c = 0; c < sums; ++c) {
            good = __all_sync(0xffffffffu, mbar_wait(ready + half, half_parity));
            if (!good) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            uint32_t sum[32];
            load32(sum, tmem + half * kTile + col + ((uint32_t)(quarter * 32) << 16));
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive(spent + half);
            half ^= 1;
            if (half == 0) half_parity ^= 1;
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[e] += __uint_as_float(sum[e]);
          }
          if (!good) break;
          if (part == 2) {
            finish(p, step + 1 < p.steps ? kUpdate : kLast, from, it, tile, row, col, acc, skip);
            break;
          }
          const float one = part == 0 ? 0.0f : p.ca * kScale;
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = acc[k + j] * (1.0f / kScale) + (col + k + j == row && row < it.n ? one : 0.0f);
            put_shared(squares, row, col + k, v);
            if (part == 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = p.cc * v[j] + (col + k + j == row && row < it.n ? p.cb * kScale : 0.0f);
              put_shared(squares + 2 * kPair, row, col + k, v);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive(&made);
        }
      }
      if (!good && lane == 0) {
        atomicOr(p.error, 4u);
        s_stop = 1;
      }
    }
    __syncwarp();
    met += gridDim.x;
    if (step + 1 < p.steps) {
      good = meet(p.arrived, met, s_stop) && good;
      if (s_stop) {
        if (threadIdx.x == 0) atomicOr(p.error, 8u);
        break;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
  }
}

// --------------------------------------------------------------------------------------------- launches

uint32_t* error_word() {
  void* at = nullptr;
  return cudaGetSymbolAddress(&at, g_error) == cudaSuccess ? static_cast<uint32_t*>(at) : nullptr;
}

int sms() {
  int dev = 0, n = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? n : 148;
}

// close behind the kernel before, or with all CTAs on the device at once
template <class A>
cudaError_t start(void (*kernel)(A), int grid, int threads, int smem, bool together, cudaStream_t s, const A& args) {
  cudaLaunchAttribute at{};
  if (together) {
    at.id = cudaLaunchAttributeCooperative;
    at.val.cooperative = 1;
  } else {
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)grid);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = (size_t)smem;
  c.stream = s;
  c.attrs = &at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args);
}

struct Matrix {
  float *param, *momentum;
  const void* grad;
  void* out;
  int64_t rows, cols;
  float step;
};

int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }
int64_t matrix_bytes(int64_t rows, int64_t cols) {
  const int64_t nt = tiles_of(std::min(rows, cols)), mt = tiles_of(std::max(rows, cols));
  return (2 * nt * mt + 3 * nt * nt) * 2 * kPair;
}
int64_t norm_blocks(int64_t rows, int64_t cols) { return (rows * cols + kNormValues - 1) / kNormValues; }

bool narrow(const Matrix& m) {
  return std::min(m.rows, m.cols) <= kTile && std::max(m.rows, m.cols) <= kNarrowTiles * kTile;
}

// Matrices that go together, narrow ones or others: as many as the table and the workspace's share hold
template <class F>
void groups(const std::vector<Matrix>& all, F f) {
  for (size_t first = 0; first < all.size();) {
    size_t n = 0;
    int64_t bytes = 0, norms = 0;
    while (first + n < all.size() && n < kItems) {
      const Matrix& m = all[first + n];
      const int64_t more = matrix_bytes(m.rows, m.cols);
      if (n > 0 && (bytes + more > kGroupBytes || narrow(m) != narrow(all[first]))) break;
      bytes += more;
      norms += norm_blocks(m.rows, m.cols);
      ++n;
    }
    f(first, n, bytes, norms);
    first += n;
  }
}
size_t workspace_of(const std::vector<Matrix>& all) {
  int64_t most = 0;
  groups(all, [&](size_t, size_t, int64_t bytes, int64_t norms) { most = std::max(most, bytes + norms * 8 + 16); });
  return (size_t)most;
}

template <int N>
cudaError_t run_group(const Call& call, const Matrix* all, int n, int64_t bytes, int64_t norm_count, cudaStream_t s) {
  Args<N> a{};
  static_cast<Call&>(a) = call;
  a.count = n;
  a.norms = reinterpret_cast<double*>(a.ws + bytes);
  a.arrived = reinterpret_cast<uint32_t*>(a.norms + norm_count);
  int64_t at = 0;
  int norms = 0, preps = 0;
  for (int k = 0; k < n; ++k) {
    const Matrix& m = all[k];
    Item& it = a.item[k];
    it.param = m.param;
    it.momentum = m.momentum;
    it.grad = m.grad;
    it.out = m.out;
    it.rows = (int)m.rows;
    it.cols = (int)m.cols;
    it.flipped = m.rows > m.cols;
    it.n = std::min(it.rows, it.cols);
    it.m = std::max(it.rows, it.cols);
    it.nt = (int)tiles_of(it.n);
    it.mt = (int)tiles_of(it.m);
    it.step = m.step;
    const int64_t x = (int64_t)it.nt * 2 * it.mt * kPair, square = (int64_t)it.nt * 2 * it.nt * kPair;
    it.x[0] = at;
    it.x[1] = at + x;
    it.a = at + 2 * x;
    it.c = it.a + square;
    it.b = it.c + square;
    at = it.b + square;
    it.first_norm = norms;
    it.norms = (int)norm_blocks(m.rows, m.cols);
    it.first_prep = preps;
    it.first_square = a.squares;
    it.first_wide = a.wides;
    norms += it.norms;
    preps += it.nt * 2 * it.mt;
    a.squares += it.nt * (it.nt + 1) / 2;
    a.wides += it.nt * it.mt;
  }
  const bool thin = narrow(all[0]);  // (all of them)
  void (*const kernel)(Args<N>) = thin ? narrow_kernel<N> : products_kernel<N>;
  const int shared = thin ? kNarrowShared : kShared, tiles = thin ? a.wides : std::max(a.squares, a.wides);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
  if (e == cudaSuccess) e = start(momentum_kernel<N>, norms, kPrepThreads, 0, false, s, a);
  if (e == cudaSuccess) e = start(prepare_kernel<N>, preps, kPrepThreads, 0, false, s, a);
  if (e == cudaSuccess) e = start(kernel, std::min(sms(), tiles), kThreads, shared, true, s, a);
  return e;
}

cudaError_t run(const std::vector<Matrix>& all, Call& call, void* workspace, cudaStream_t s) {
  call.ws = static_cast<char*>(workspace);
  cudaError_t e = cudaSuccess;
  groups(all, [&](size_t first, size_t n, int64_t bytes, int64_t norms) {
    if (e != cudaSuccess) return;
    e = n <= kShort ? run_group<kShort>(call, &all[first], (int)n, bytes, norms, s)
                    : run_group<kItems>(call, &all[first], (int)n, bytes, norms, s);
  });
  return e;
}

int check_iteration(int dtype, int steps, float eps, float a, float b, float c) {
  if (dtype < PESQ_F32 || dtype > PESQ_F16) return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown type");
  if (steps < 1 || steps > 100) return set_error(PESQ_ERR_INVALID_ARGUMENT, "between 1 and 100 steps");
  if (!(eps >= FLT_MIN) || !(eps - eps == 0.0f))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "eps must be positive, finite and no subnormal");
  for (float x : {a, b, c})
    if (!(std::fabs(x) <= 16.0f)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "coefficients must lie between -16 and 16");
  return PESQ_OK;
}
int check_sizes(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return set_error(PESQ_ERR_INVALID_ARGUMENT, "matrices need at least one row and column");
  if (rows > kMost || cols > kMost) return set_error(PESQ_ERR_UNSUPPORTED, "at most 32768 rows and columns");
  return PESQ_OK;
}
// (what lies at 16 bytes is read and written in fours, all else value by value)
bool aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == PESQ_F32 ? 4 : 2) == 0; }
int check_workspace(const void* workspace, size_t bytes, size_t need) {
  // (its tiles are read by bulk copies, and by instructions that want rows of eight in 1024 bytes, of the copy)
  if (!workspace || bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(PESQ_ERR_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  return PESQ_OK;
}

int muon_matrices(const pesq_muon_desc* d, const pesq_muon_tensor* tensors, int64_t count, std::vector<Matrix>& all) {
  if (!d || count < 0 || (count > 0 && !tensors)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (const int status = check_iteration(d->grad_dtype, d->steps, d->eps, d->a, d->b, d->c)) return status;
  if (!(d->momentum >= 0.0) || !(d->momentum < 1.0)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "momentum must lie in [0, 1)");
  if (!(d->lr >= 0.0f) || !(d->weight_decay >= 0.0f))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "lr and weight_decay must not be negative");
  if (!aligned(d->grad_scale, PESQ_F32)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "grad_scale is not aligned to its type");
  if (d->adjust != PESQ_MUON_ORIGINAL && d->adjust != PESQ_MUON_MATCH_RMS)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown adjustment");
  for (int64_t i = 0; i < count; ++i) {
    const pesq_muon_tensor& t = tensors[i];
    if (!t.grad) continue;
    if (!t.param || !t.momentum) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL parameter or momentum");
    if (t.copy && d->grad_dtype == PESQ_F32) return set_error(PESQ_ERR_INVALID_ARGUMENT, "copies are of 16-bit gradients' type");
    if (!aligned(t.param, PESQ_F32) || !aligned(t.momentum, PESQ_F32) || !aligned(t.grad, d->grad_dtype) || !aligned(t.copy, d->grad_dtype))
      return set_error(PESQ_ERR_INVALID_ARGUMENT, "a tensor that is not aligned to its type");
    if (const int status = check_sizes(t.rows, t.cols)) return status;
    const double ratio = (double)t.rows / (double)t.cols;
    const double adjust = d->adjust == PESQ_MUON_ORIGINAL ? std::sqrt(std::max(1.0, ratio))
                                                          : 0.2 * std::sqrt((double)std::max(t.rows, t.cols));
    all.push_back({t.param, t.momentum, t.grad, t.copy, t.rows, t.cols, (float)(d->lr * adjust)});
  }
  std::stable_partition(all.begin(), all.end(), narrow);
  return PESQ_OK;
}

// Whether two of what a step writes are the same memory, or some of it: matrices are worked on at the same time
bool overlap(const std::vector<Matrix>& all, int grad_dtype) {
  std::vector<std::pair<const char*, const char*>> written;
  written.reserve(3 * all.size());
  for (const Matrix& m : all) {
    const int64_t n = m.rows * m.cols;
    for (const float* p : {m.param, m.momentum}) written.push_back({reinterpret_cast<const char*>(p), reinterpret_cast<const char*>(p + n)});
    if (m.out) written.push_back({static_cast<const char*>(m.out), static_cast<const char*>(m.out) + n * (grad_dtype == PESQ_F32 ? 4 : 2)});
  }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].second) return true;
  return false;
}

int stack(const pesq_orthogonalize_desc* d, const void* x, void* out, std::vector<Matrix>& all) {
  if (!d) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL descriptor");
  if (const int status = check_iteration(d->dtype, d->steps, d->eps, d->a, d->b, d->c)) return status;
  if (const int status = check_sizes(d->rows, d->cols)) return status;
  if (!aligned(x, d->dtype) || !aligned(out, d->dtype)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "a stack that is not aligned to its type");
  if (d->count < 1 || d->count > 1 << 20) return set_error(PESQ_ERR_INVALID_ARGUMENT, "between 1 and 2^20 matrices");
  const int64_t bytes = d->rows * d->cols * (d->dtype == PESQ_F32 ? 4 : 2);
  for (int64_t i = 0; i < d->count; ++i)
    all.push_back({nullptr, nullptr, static_cast<const char*>(x) + i * bytes, static_cast<char*>(out) + i * bytes, d->rows,
                   d->cols, 0.0f});
  return PESQ_OK;
}

// (a vector or a launch's attributes may fail to find memory: no exception leaves a C entry)
template <class F>
int guarded(F f) {
  try {
    return f();
  } catch (...) {
    return set_error(PESQ_ERR_CUDA, "out of host memory");
  }
}

}  // namespace

extern "C" {

int pesq_muon_workspace(const pesq_muon_desc* d, const pesq_muon_tensor* tensors, int64_t count, size_t* bytes) {
  if (!bytes) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  return guarded([&] {
    std::vector<Matrix> all;
    if (const int status = muon_matrices(d, tensors, count, all)) return status;
    *bytes = workspace_of(all);
    return (int)PESQ_OK;
  });
}

int pesq_muon_step(const pesq_muon_desc* d, const pesq_muon_tensor* tensors, int64_t count, void* stream, void* workspace,
                   size_t workspace_bytes) {
  return guarded([&] {
    std::vector<Matrix> all;
    if (const int status = muon_matrices(d, tensors, count, all)) return status;
    if (all.empty()) return (int)PESQ_OK;
    if (const int status = check_workspace(workspace, workspace_bytes, workspace_of(all))) return status;
    if (overlap(all, d->grad_dtype)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "parameters, momenta and copies must not share memory");
    Call a{};
    a.dtype = d->grad_dtype;
    a.steps = d->steps;
    a.nesterov = d->nesterov != 0;
    a.grad_scale = d->grad_scale;
    a.beta = (float)d->momentum;
    a.rest = (float)(1.0 - d->momentum);
    a.decay = (float)(1.0 - (double)d->lr * d->weight_decay);
    a.eps = d->eps;
    a.ca = d->a, a.cb = d->b, a.cc = d->c;
    a.error = error_word();
    if (!a.error) return set_error(PESQ_ERR_CUDA, "no error word");
    const cudaError_t e = run(all, a, workspace, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? (int)PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
  });
}

int pesq_orthogonalize_workspace(const pesq_orthogonalize_desc* d, size_t* bytes) {
  if (!bytes) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  return guarded([&] {
    std::vector<Matrix> all;
    if (const int status = stack(d, nullptr, nullptr, all)) return status;
    *bytes = workspace_of(all);
    return (int)PESQ_OK;
  });
}

int pesq_orthogonalize(const pesq_orthogonalize_desc* d, void* stream, const void* x, void* out, void* workspace,
                       size_t workspace_bytes) {
  return guarded([&] {
    std::vector<Matrix> all;
    if (!x || !out) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL operand");
    if (const int status = stack(d, x, out, all)) return status;
    if (const int status = check_workspace(workspace, workspace_bytes, workspace_of(all))) return status;
    Call a{};
    a.dtype = d->dtype;
    a.steps = d->steps;
    a.eps = d->eps;
    a.ca = d->a, a.cb = d->b, a.cc = d->c;
    a.error = error_word();
    if (!a.error) return set_error(PESQ_ERR_CUDA, "no error word");
    const cudaError_t e = run(all, a, workspace, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? (int)PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
  });
}

int pesq_muon_check(void* stream, uint32_t* failed) {
  if (!failed) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  uint32_t* word = error_word();
  if (!word) return set_error(PESQ_ERR_CUDA, "no error word");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(failed, word, 4, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, 4, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e == cudaSuccess ? PESQ_OK : set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
