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
// contraction (2.3e-5 of the result of a 385 x 1155 matrix, 5.0e-5 of 1280 x 3840).  So it sums 128 columns alone, and the
// warps that read it add those sums in registers, rounded (7.1e-6 and 4.0e-6; float32 products 2.8e-6 and 3.6e-6).
//
// Products run on tcgen05 with the accumulator in tensor memory, in tiles of 128 x 128.  Matrices lie in the workspace as the
// tiles that the instruction reads from shared memory: 128 rows of 64 columns in the 128-byte swizzle, hi and lo
// behind each other, zeros past the matrix' edge.  So an operand is a plain bulk copy of 32 KB, odd sizes need nothing
// anywhere, and the one layout serves X X^T (64 columns of the contraction side by side) and B X (X's rows are the contraction:
// the same bytes read as a transposed operand).  A and the polynomial are symmetric: the tiles below and on the diagonal are
// computed, and written mirrored too, which takes 10 n^2 m products of a square matrix' step instead of 14.
//
// A CTA takes tiles in turn: a thread issues copies three stages ahead, a thread issues products, four warps
// empty the accumulators, of which there are two, so that a tile's end overlaps the next one's products.  All waits are
// bounded; one that runs out sets an error word and the CTA returns.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
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
constexpr int kThreads = 192;                         // copies, products, four warps of results
constexpr int kShared = kStages * kStage + 1024;      // (aligned to 1024 in the kernel)
constexpr int kSegment = 2;                           // stages whose products are summed in tensor memory
constexpr float kScale = 1024.0f;                     // of what is kept
constexpr int kMost = 32768;                          // rows or columns
constexpr int kItems = 128;                           // matrices of a launch
constexpr int64_t kGroupBytes = INT64_C(256) << 20;   // of their workspace, where there are several
constexpr int kNormValues = 8192;                     // of a block of the first pass
constexpr int kPrepThreads = 256;

enum Mode { kGram, kPolynomial, kUpdate, kLast };

struct Item {
  float* param;      // Muon; null where X itself is the result
  float* momentum;
  const void* grad;  // or the matrix to orthogonalise
  void* out;         // the parameter's copy in the gradient's type, or the result, or null
  int64_t x[2], a, b;  // workspace offsets of X (before and after a step), A, the polynomial
  int rows, cols;
  int n, m, nt, mt;    // shorter and longer side, in tiles of 128
  int flipped;         // X is the matrix' transpose
  int first_norm, norms;                     // of the blocks, of the first pass
  int first_prep, first_square, first_wide;  // tile, of the second pass, of symmetric products, of updates
  float step;          // lr times adjust
};
struct Args {
  int count, dtype, nesterov;
  int total;           // tiles, or blocks, of the launch
  int mode, from;      // of a product; which X it reads
  char* ws;
  double* norms;       // sums of squares of the first pass' blocks
  const float* grad_scale;
  float beta, rest, decay;  // momentum, 1 - momentum, 1 - lr wd
  float eps, ca, cb, cc;
  uint32_t* error;
  Item item[kItems];
};
static_assert(sizeof(Args) < 32000, "kernel parameters");

__device__ uint32_t g_error;

__device__ __forceinline__ float load(const void* p, int dtype, int64_t i) {
  return dtype == PESQ_F32    ? static_cast<const float*>(p)[i]
         : dtype == PESQ_BF16 ? widen(static_cast<const __nv_bfloat16*>(p)[i])
                              : widen(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store(void* p, int dtype, int64_t i, float v) {
  if (dtype == PESQ_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == PESQ_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = narrow<__nv_bfloat16>(v);
  else
    static_cast<__half*>(p)[i] = narrow<__half>(v);
}
// the last item whose first is not above at
template <int Item::*kFirst>
__device__ __forceinline__ int find(const Args& p, int at) {
  int lo = 0, hi = p.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.item[mid].*kFirst <= at) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// the factor of the gradients; `skip` where it is not finite
__device__ __forceinline__ float scale_of(const Args& p, bool& skip) {
  const float s = p.grad_scale ? *p.grad_scale : 1.0f;
  skip = !(s - s == 0.0f);
  return s;
}
__device__ __forceinline__ void dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void depend() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------------------- momentum and its norm

__device__ __forceinline__ float update_of(const Args& p, const Item& it, int64_t i, float s) {
  if (!it.momentum) return load(it.grad, p.dtype, i);
  const float m = it.momentum[i];
  return p.nesterov ? fmaf(p.beta, m, p.rest * (s * load(it.grad, p.dtype, i))) : m;
}

__global__ void __launch_bounds__(kPrepThreads) momentum_kernel(const __grid_constant__ Args p) {
  __shared__ double s_sum[kPrepThreads / 32];
  dependents();
  depend();
  const Item& it = p.item[find<&Item::first_norm>(p, blockIdx.x)];
  const int64_t numel = (int64_t)it.rows * it.cols, first = (int64_t)(blockIdx.x - it.first_norm) * kNormValues;
  const int64_t end = min(numel, first + kNormValues);
  bool skip;
  const float s = scale_of(p, skip);
  double sum = 0.0;
  for (int64_t i = first + threadIdx.x; i < end; i += kPrepThreads) {
    float u;
    if (it.momentum) {
      const float g = s * load(it.grad, p.dtype, i);
      const float m = fmaf(p.beta, it.momentum[i], p.rest * g);
      if (!skip) it.momentum[i] = m;
      u = p.nesterov ? fmaf(p.beta, m, p.rest * g) : m;
    } else {
      u = load(it.grad, p.dtype, i);
    }
    sum = fma((double)u, (double)u, sum);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPrepThreads / 32; ++w) sum += s_sum[w];
    p.norms[blockIdx.x] = sum;
  }
}

__device__ __forceinline__ void split(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}
struct alignas(16) Eight {
  __half h[8];
};
__device__ __forceinline__ void split8(const float (&v)[8], Eight& hi, Eight& lo) {
#pragma unroll
  for (int j = 0; j < 8; ++j) split(v[j], hi.h[j], lo.h[j]);
}
// where columns 8 chunk .. of a row of a tile's plane lie
__device__ __forceinline__ int at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// X in tiles; a block takes one
__global__ void __launch_bounds__(kPrepThreads) prepare_kernel(const __grid_constant__ Args p) {
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
  const float inverse = (float)(kScale / (norm > p.eps || norm != norm ? norm : (double)p.eps));
  char* to = p.ws + it.x[0] + (int64_t)tile * kPair;
  // neighbouring threads: rows of a flipped matrix, chunks of a row of another
  for (int i = threadIdx.x; i < kTile * 8; i += kPrepThreads) {
    const int row = it.flipped ? i % kTile : i / 8, chunk = it.flipped ? i / kTile : i % 8;
    const int r = rt * kTile + row, c = ct * kDepth + chunk * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = r < it.n && c + j < it.m;
      v[j] = in ? update_of(p, it, it.flipped ? (int64_t)(c + j) * it.cols + r : (int64_t)r * it.cols + c + j, s) * inverse : 0.0f;
    }
    Eight hi, lo;
    split8(v, hi, lo);
    *reinterpret_cast<Eight*>(to + at(row, chunk)) = hi;
    *reinterpret_cast<Eight*>(to + kPlane + at(row, chunk)) = lo;
  }
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
  __device__ __forceinline__ Tile(const Args& p, int t) {
    if (p.mode < kUpdate) {
      index = find<&Item::first_square>(p, t);
      const Item& it = p.item[index];
      t -= it.first_square;
      i = 0;
      while (t > i) t -= ++i;  // rows of 1, 2, 3, ... tiles
      j = t;
      depth = ((p.mode == kGram ? it.m : it.n) + kDepth - 1) / kDepth;
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

// What four warps make of 32 columns of a tile's accumulators
__device__ __forceinline__ void finish(const Args& p, const Item& it, const Tile& t, int row, int col, const float (&acc)[32],
                                       float s_decay, bool skip) {
  const int r = t.i * kTile + row, lane = threadIdx.x & 31;
  if (p.mode == kLast) {
    // (X is the result or its transpose: either way a thread has a row of X)
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const int c = t.j * kTile + col + k;
      if (r >= it.n || c >= it.m || skip) continue;
      const float x = acc[k] * (1.0f / (kScale * kScale));
      const int64_t to = it.flipped ? (int64_t)c * it.cols + r : (int64_t)r * it.cols + c;
      if (it.param) {
        const float v = fmaf(-it.step, x, it.param[to] * s_decay);
        it.param[to] = v;
        if (it.out) store(it.out, p.dtype, to, v);
      } else {
        store(it.out, p.dtype, to, x);
      }
    }
    return;
  }
  const int tiles = p.mode == kUpdate ? 2 * it.mt : 2 * it.nt;  // side by side
  const int64_t base = p.mode == kGram ? it.a : p.mode == kPolynomial ? it.b : it.x[p.from ^ 1];
  const int64_t place = ((int64_t)t.i * tiles + t.j * 2 + col / kDepth) * kPair;
  char* to = p.ws + base + place;
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    const int chunk = col % kDepth / 8 + k / 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = acc[k + j] * (1.0f / kScale);
    if (p.mode == kPolynomial) {
      const char* from = p.ws + it.a + place;
      const Eight hi = *reinterpret_cast<const Eight*>(from + at(row, chunk));
      const Eight lo = *reinterpret_cast<const Eight*>(from + kPlane + at(row, chunk));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = t.j * kTile + col + k + j;
        v[j] = fmaf(p.cc, v[j], p.cb * (__half2float(hi.h[j]) + __half2float(lo.h[j])));
        if (c == r && r < it.n) v[j] += p.ca * kScale;
      }
    }
    Eight hi, lo;
    split8(v, hi, lo);
    *reinterpret_cast<Eight*>(to + at(row, chunk)) = hi;
    *reinterpret_cast<Eight*>(to + kPlane + at(row, chunk)) = lo;
    if (p.mode < kUpdate && t.i != t.j) {
      // mirrored: rows are the columns here.  Neighbouring lanes, which hold neighbouring rows, exchange halves, so that each
      // stores two columns of one row
      char* over = p.ws + base + ((int64_t)t.j * tiles + t.i * 2 + row / kDepth) * kPair;
      const int column = row % kDepth & ~1;
#pragma unroll
      for (int plane = 0; plane < 2; ++plane) {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(plane ? lo.h : hi.h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, words[j], 1);
          const uint32_t pair = lane & 1 ? __byte_perm(other, words[j], 0x7632) : __byte_perm(words[j], other, 0x5410);
          const int mine = col + k + 2 * j + (lane & 1);
          *reinterpret_cast<uint32_t*>(over + plane * kPlane + at(mine, column / 8) + column % 8 * 2) = pair;
        }
      }
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1) products_kernel(const __grid_constant__ Args p) {
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], ready[2], spent[2], drained;
  __shared__ uint32_t s_tmem;
  char* const tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) init(full + s, 1), init(empty + s, 1);
    for (int s = 0; s < 2; ++s) init(ready + s, 1), init(spent + s, 4);
    init(&drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s_tmem;
  dependents();
  depend();
  bool good = true;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t parity = 1;
      for (int t = blockIdx.x; t < p.total && good; t += gridDim.x) {
        const Tile tile(p, t);
        const Item& it = p.item[tile.index];
        const bool wide = p.mode >= kUpdate, same = !wide && tile.i == tile.j;
        const int64_t left = p.mode == kGram ? it.x[p.from] : p.mode == kPolynomial ? it.a : it.b;
        const int across = p.mode == kGram ? 2 * it.mt : 2 * it.nt;
        const char *a = p.ws + left + (int64_t)tile.i * across * kPair, *b = p.ws + left + (int64_t)tile.j * across * kPair;
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
            const char* x = p.ws + it.x[p.from] + ((int64_t)(k / 2) * 2 * it.mt + tile.j * 2) * kPair + (k & 1) * (kPlane / 2);
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
        for (int s = 1; s <= issued; ++s) {
          // the copies s stages back, whose phase is that of the parity they were issued with
          const int back = (stage + kStages - s) % kStages;
          mbar_wait(full + back, back < stage ? parity ^ 1 : parity);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, half = 0;
      uint32_t parity = 0, spent_parity = 1;
      for (int t = blockIdx.x; t < p.total && good; t += gridDim.x) {
        const Tile tile(p, t);
        const bool wide = p.mode >= kUpdate, same = !wide && tile.i == tile.j;
        const uint32_t instruction = kInstruction | (wide ? kTransposedB : 0);
        for (int k = 0; k < tile.depth; ++k) {
          if (k % kSegment == 0 && !mbar_wait(spent + half, spent_parity) || !mbar_wait(full + stage, parity)) {
            good = false;
            break;
          }
          const uint32_t to = tmem + half * kTile;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a = smem_u32(tiles + stage * kStage), b = same ? a : a + kPair;
#pragma unroll
          for (int s = 0; s < kDepth / 16; ++s) {
            const uint32_t as = a + s * 32, bs = b + s * (wide ? 2048 : 32);
            const uint64_t a_hi = descriptor(as, false), a_lo = descriptor(as + kPlane, false);
            const uint64_t b_hi = descriptor(bs, wide), b_lo = descriptor(bs + kPlane, wide);
            product(to, a_lo, b_hi, instruction, k % kSegment > 0 || s > 0);
            product(to, a_hi, b_lo, instruction, true);
            product(to, a_hi, b_hi, instruction, true);
          }
          commit(empty + stage);
          if (++stage == kStages) stage = 0, parity ^= 1;
          if ((k + 1) % kSegment == 0 || k + 1 == tile.depth) {
            commit(ready + half);
            half ^= 1;
            if (half == 0) spent_parity ^= 1;
          }
        }
      }
      if (!good) {  // (what is issued ends before its memory goes)
        atomicOr(p.error, 2u);
        commit(&drained);
        mbar_wait(&drained, 0);
      }
    }
  } else {
    const int quarter = warp & 3;
    int half = 0;
    uint32_t parity = 0;
    bool skip;
    scale_of(p, skip);
    for (int t = blockIdx.x; t < p.total && good; t += gridDim.x) {
      const Tile tile(p, t);
      float acc[kTile / 32][32];
#pragma unroll
      for (int c = 0; c < kTile / 32; ++c)
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[c][e] = 0.0f;
      for (int k = 0; k < tile.depth; k += kSegment) {
        good = __all_sync(0xffffffffu, mbar_wait(ready + half, parity));
        if (!good) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c = 0; c < kTile / 32; ++c) {
          uint32_t part[32];
          load32(part, tmem + half * kTile + c * 32 + ((uint32_t)(quarter * 32) << 16));
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[c][e] += __uint_as_float(part[e]);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(spent + half);
        half ^= 1;
        if (half == 0) parity ^= 1;
      }
      if (!good) break;
#pragma unroll
      for (int c = 0; c < kTile / 32; ++c)
        finish(p, p.item[tile.index], tile, quarter * 32 + lane, c * 32, acc[c], p.decay, skip);
    }
    if (!good && lane == 0) atomicOr(p.error, 4u);
  }
  __syncwarp();
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

template <class... A>
cudaError_t start(void (*kernel)(A...), int grid, int threads, int smem, cudaStream_t s, const A&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)grid);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = (size_t)smem;
  c.stream = s;
  c.attrs = &at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
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
  return (2 * nt * mt + 2 * nt * nt) * 2 * kPair;
}
int64_t norm_blocks(int64_t rows, int64_t cols) { return (rows * cols + kNormValues - 1) / kNormValues; }

// Matrices that go together: as many as the table and the workspace's share hold
template <class F>
void groups(const std::vector<Matrix>& all, F f) {
  for (size_t first = 0; first < all.size();) {
    size_t n = 0;
    int64_t bytes = 0, norms = 0;
    while (first + n < all.size() && n < kItems) {
      const Matrix& m = all[first + n];
      const int64_t more = matrix_bytes(m.rows, m.cols);
      if (n > 0 && bytes + more > kGroupBytes) break;
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
  groups(all, [&](size_t, size_t, int64_t bytes, int64_t norms) { most = std::max(most, bytes + norms * 8); });
  return (size_t)most;
}

cudaError_t run(const std::vector<Matrix>& all, Args& a, int steps, void* workspace, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(products_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared);
  groups(all, [&](size_t first, size_t n, int64_t bytes, int64_t) {
    if (e != cudaSuccess) return;
    a.count = (int)n;
    a.ws = static_cast<char*>(workspace);
    a.norms = reinterpret_cast<double*>(a.ws + bytes);
    int64_t at = 0;
    int norms = 0, preps = 0, squares = 0, wides = 0;
    for (size_t k = 0; k < n; ++k) {
      const Matrix& m = all[first + k];
      Item& it = a.item[k];
      it = Item{};
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
      it.b = it.a + square;
      at = it.b + square;
      it.first_norm = norms;
      it.norms = (int)norm_blocks(m.rows, m.cols);
      it.first_prep = preps;
      it.first_square = squares;
      it.first_wide = wides;
      norms += it.norms;
      preps += it.nt * 2 * it.mt;
      squares += it.nt * (it.nt + 1) / 2;
      wides += it.nt * it.mt;
    }
    e = start(momentum_kernel, norms, kPrepThreads, 0, s, a);
    if (e == cudaSuccess) e = start(prepare_kernel, preps, kPrepThreads, 0, s, a);
    for (int step = 0; step < steps && e == cudaSuccess; ++step) {
      a.from = step & 1;
      for (int mode : {(int)kGram, (int)kPolynomial, step + 1 < steps ? (int)kUpdate : (int)kLast}) {
        a.mode = mode;
        a.total = mode < kUpdate ? squares : wides;
        if (e == cudaSuccess) e = start(products_kernel, std::min(sms(), a.total), kThreads, kShared, s, a);
      }
    }
  });
  return e;
}

int check_iteration(int dtype, int steps, float eps, float a, float b, float c) {
  if (dtype < PESQ_F32 || dtype > PESQ_F16) return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown type");
  if (steps < 1 || steps > 100) return set_error(PESQ_ERR_INVALID_ARGUMENT, "between 1 and 100 steps");
  if (!(eps > 0.0f) || !(eps - eps == 0.0f)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "eps must be positive and finite");
  for (float x : {a, b, c})
    if (!(std::fabs(x) <= 16.0f)) return set_error(PESQ_ERR_INVALID_ARGUMENT, "coefficients must lie between -16 and 16");
  return PESQ_OK;
}
int check_sizes(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return set_error(PESQ_ERR_INVALID_ARGUMENT, "matrices need at least one row and column");
  if (rows > kMost || cols > kMost) return set_error(PESQ_ERR_UNSUPPORTED, "at most 32768 rows and columns");
  return PESQ_OK;
}
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
  if (d->adjust != PESQ_MUON_ORIGINAL && d->adjust != PESQ_MUON_MATCH_RMS)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown adjustment");
  for (int64_t i = 0; i < count; ++i) {
    const pesq_muon_tensor& t = tensors[i];
    if (!t.grad) continue;
    if (!t.param || !t.momentum) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL parameter or momentum");
    if (t.copy && d->grad_dtype == PESQ_F32) return set_error(PESQ_ERR_INVALID_ARGUMENT, "copies are of 16-bit gradients' type");
    if (const int status = check_sizes(t.rows, t.cols)) return status;
    const double ratio = (double)t.rows / (double)t.cols;
    const double adjust = d->adjust == PESQ_MUON_ORIGINAL ? std::sqrt(std::max(1.0, ratio))
                                                          : 0.2 * std::sqrt((double)std::max(t.rows, t.cols));
    all.push_back({t.param, t.momentum, t.grad, t.copy, t.rows, t.cols, (float)(d->lr * adjust)});
  }
  return PESQ_OK;
}

int stack(const pesq_orthogonalize_desc* d, const void* x, void* out, std::vector<Matrix>& all) {
  if (!d) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL descriptor");
  if (const int status = check_iteration(d->dtype, d->steps, d->eps, d->a, d->b, d->c)) return status;
  if (const int status = check_sizes(d->rows, d->cols)) return status;
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
    Args a{};
    a.dtype = d->grad_dtype;
    a.nesterov = d->nesterov != 0;
    a.grad_scale = d->grad_scale;
    a.beta = (float)d->momentum;
    a.rest = (float)(1.0 - d->momentum);
    a.decay = (float)(1.0 - (double)d->lr * d->weight_decay);
    a.eps = d->eps;
    a.ca = d->a, a.cb = d->b, a.cc = d->c;
    a.error = error_word();
    if (!a.error) return set_error(PESQ_ERR_CUDA, "no error word");
    const cudaError_t e = run(all, a, d->steps, workspace, static_cast<cudaStream_t>(stream));
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
    Args a{};
    a.dtype = d->dtype;
    a.eps = d->eps;
    a.ca = d->a, a.cb = d->b, a.cc = d->c;
    a.error = error_word();
    if (!a.error) return set_error(PESQ_ERR_CUDA, "no error word");
    const cudaError_t e = run(all, a, d->steps, workspace, static_cast<cudaStream_t>(stream));
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
