// Linear attention with a decay for each head, per row (batch item and head) of
// [batch, step, head, channel] streams, in scan order:
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   y_t = scale S_t^T q_t
//
// In chunks of C steps, with G_i the sum of the chunk's g up to step i and L_ij = exp(G_i - G_j) for
// j <= i (0 elsewhere), this is matrix products:
//
//   Y  = scale ((Q K^T) o L) V + scale diag(e^G) Q S
//   S' = e^{G_C} S + (diag(e^{G_C - G}) K)^T V
//
// and, with dS the gradient of the state at the chunk's end,
//
//   dQ = scale ((dY V^T) o L) K + scale diag(e^G) dY S^T
//   dK = scale ((dY V^T) o L)^T Q + diag(e^{G_C - G}) V dS^T
//   dV = scale ((Q K^T) o L)^T dY + diag(e^{G_C - G}) K dS
//   dS' = e^{G_C} dS + scale (diag(e^G) Q)^T dY
//
// The gradient of g_t is what flows through step t from before it to it and later: with
// W = scale (Q K^T) o (dY V^T) o L without its diagonal,
//
//   dg_t = sum_{i >= t > j} W_ij + sum_{i >= t} scale e^{G_i} q_i S dy_i + sum_{j < t} e^{G_C - G_j} k_j dS v_j
//          + e^{G_C} <S, dS>
//
// in which the chunk's own sums alone are prefix sums, so that nothing large cancels over a long row.
//
// A CTA walks the chunks of a row, or of a part of a row where rows are few (or are the few that full rounds of the device leave
// over), with the state in the registers of its warps as 32-bit sums and a copy in shared memory as an operand of the next
// chunk's products.  Parts begin from states that a sweep over keys and values alone, and a join over the parts, made before
// (of up to four parts, each makes its own of the sweep's).  A forward that a
// backward follows keeps the state before every chunk, which the backward reads beside its own, the gradient of the
// state, that it carries from the row's end.  The backward forms (Q K^T) and (dY V^T) once by rows and once by columns,
// so that every product's left operand is in the registers of the warp that made it.
//
// Numbers.  All sums, the state and the decays are 32 bits; G is summed in 64 bits and kept as two floats, so that
// differences of it are as exact as the steps' own (a reset is a step of -200 in log2, which exp2 turns to 0).
// Products go through the matrix instructions in the operands' own type where both are inputs.  What is computed (the
// weighted products, the state, the decayed keys) goes in as terms.  Beside bfloat16: three of bfloat16, which hold all bits, for what
// becomes an output of 32 bits (states, and the products with a state or its gradient that a decay's gradient sums), two (2^-18 off at
// most) for what is rounded to bfloat16 itself: 1e-4 of such an output's norm is rounded the other way, 5e-5 with three terms, which
// take 16 % more time of both directions.  Two of tf32 (2^-22) beside float16, whose range the products and states exceed, and
// float32, whose inputs are also two terms, and whose sums are made apart and added rounded.
//
// Bound.  The bytes alone would take 36 us forward and 63 backward of 896 rows of 500 steps of 64 x 64 in bfloat16, which take 157
// and 405 (all other figures of this file are of its stages, and given as shares of the time then): neither memory (20 to 30 % of its rate)
// nor the matrix instructions (30 %) are full.  Shared memory's pipe is the fullest (60 %), since every warp reads the chunk's operands
// and the state for 16 rows, and the rest is latency between barriers with 12 to 16 warps an SM, whose registers are what holds the state.
// The backward is held to 128 registers by its 16 warps an SM, and spills: 504 bytes stored and 328 read a thread of 64 x 64 in
// bfloat16, 580 and 400 in float16, 1012 and 628 in float32, 1.5 to 2 KB and 0.9 to 1.5 of 128 x 128 (1 and 0.7 in float32).
// Of other splits none was faster: 32 rows a warp (a third slower forward), eight warps a chunk (a quarter), a quarter more CTAs with one
// set of tiles.
#pragma once

#include <type_traits>

#include "../../include/pesq_cuda.h"
#include "train.cuh"

namespace pesq {
namespace lattn {

using namespace train;

constexpr float kCut = -200.0f;  // log2 of a decay that is zero: exp2 of it and less is 0, and sums of it stay exact

// ------------------------------------------------------------------------------------------- arguments

struct Operand {
  const void* p;
  int64_t sb, st, sh;  // strides of batch, step and head, in elements
  int unit;            // bytes that a row's pieces are loaded in: 16, 8, 4 or 2
};

struct Args {
  Operand q, k, v, dy;
  const float* decay;  // log decays
  int64_t decay_sb, decay_st, decay_sh;
  const uint8_t* reset;
  int64_t reset_sb, reset_st;
  const int64_t* lengths;
  const float* state;  // [batch, heads, key, value], or null
  int64_t steps;
  int heads, key, value;
  int reverse;
  float scale;
  int chunks, parts, part_chunks, slices;  // of a row; of a row that is cut; chunks of a part; CTAs side by side over the values
  int64_t whole;            // the first rows, which are not cut
  float *starts, *factors;  // [cut rows, parts, DK, DV], [cut rows, parts]: of a sweep and its join
  int joined;               // a join has made the states that the parts begin from; else they are made from the sweep's
  void* kept;               // states before the chunks
  // results
  void* y;
  float* last;              // or null: not wanted
  void *dq, *dk, *dv;
  float* ddecay;            // [batch, step, heads], or
  double* chunk_ddecay;     // its sums over the steps of every chunk, [rows, chunks], where a head has one decay
  const float* dlast;
  float* dstate;
};

// ----------------------------------------------------------------------------------------- instructions

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

template <bool kTrans>
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], const void* p) {
  if (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_of(p)) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_of(p)) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// Sixteen columns of the contraction as two of eight.  A thread's pairs of columns 2c, 2c + 1 stand where the instruction has
// columns c and c + 4: in both operands, so that the sum is the same.
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[8], const uint32_t (&b)[4]) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[4 * s]), "r"(a[4 * s + 2]), "r"(a[4 * s + 1]), "r"(a[4 * s + 3]), "r"(b[2 * s]), "r"(b[2 * s + 1]));
}

// Both of two tf32 terms, as a sum of its own that is added rounded: the instruction cuts off what its accumulator does not hold
// (over 128 columns 1.2e-6 of a float32 result, 3e-7 so)
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&ahi)[8], const uint32_t (&alo)[8], const uint32_t (&bhi)[4],
                                         const uint32_t (&blo)[4]) {
  float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  mma_tf32(t, alo, bhi);
  mma_tf32(t, ahi, blo);
  mma_tf32(t, ahi, bhi);
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] += t[e];
}

// two values as bfloat16 terms hi + lo
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
  const float dx = x - __uint_as_float(hi << 16), dy = y - __uint_as_float(hi & 0xffff0000u);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(dy), "f"(dx));
}
// and the term that they leave: with it all bits of 32
__device__ __forceinline__ uint32_t least_bf16(float x, float y, uint32_t hi, uint32_t lo) {
  uint32_t least;
  const float dx = (x - __uint_as_float(hi << 16)) - __uint_as_float(lo << 16);
  const float dy = (y - __uint_as_float(hi & 0xffff0000u)) - __uint_as_float(lo & 0xffff0000u);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(least) : "f"(dy), "f"(dx));
  return least;
}
// a value as tf32 terms
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
__device__ __forceinline__ float2 floats_of(uint32_t pair, __nv_bfloat16) {
  return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
}
__device__ __forceinline__ float2 floats_of(uint32_t pair, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&pair));
}

__device__ __forceinline__ uint32_t narrow_pair(float x, float y, __nv_bfloat16) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t narrow_pair(float x, float y, __half) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}

// ------------------------------------------------------------------------------------------- operands
//
// A thread's share of a 16 x 16 left operand is four pairs of adjacent columns: rows g and g + 8 (g = lane / 4)
// of columns 2c, 2c + 1 (c = lane % 4), then the same rows of columns 2c + 8, 2c + 9.  Of a 16 x 8 right operand two
// pairs of adjacent rows of column g.  The same of every type; what is computed in a product's
// layout (rows g, g + 8 of columns 2c, 2c + 1 of eight) is two of these eighths of a left operand.

template <class T>
constexpr bool kHalfWord = sizeof(T) == 2;

// left operand: an input
template <class T>
struct InA {
  uint32_t x[4];
};
template <>
struct InA<float> {
  uint32_t hi[8], lo[8];
};
template <class T>
struct InB {
  uint32_t x[2];
};
template <>
struct InB<float> {
  uint32_t hi[4], lo[4];
};
// computed: of two terms
template <class T>
struct Made {
  uint32_t hi[8], lo[8];
};
template <>
struct Made<__nv_bfloat16> {
  uint32_t hi[4], lo[4];
};
// What goes into a state, which is an output in 32 bits: of three terms of bfloat16 (of two, 2.2e-6 of the last state are off instead of
// 1.2e-7, in 4 % less time)
template <class T>
struct Finest : Made<T> {};
template <>
struct Finest<__nv_bfloat16> : Made<__nv_bfloat16> {
  uint32_t least[4];
};
template <class T>
struct MadeB {
  uint32_t hi[4], lo[4];
};
template <>
struct MadeB<__nv_bfloat16> {
  uint32_t hi[2], lo[2], least[2];  // (the least where a product takes three)
};

template <class T>
__device__ __forceinline__ void make(Made<T>& m, const float (&x)[8]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) split_bf16(x[2 * i], x[2 * i + 1], m.hi[i], m.lo[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) split_tf32(x[i], m.hi[i], m.lo[i]);
  }
}

template <class T>
__device__ __forceinline__ void make(Finest<T>& m, const float (&x)[8]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      split_bf16(x[2 * i], x[2 * i + 1], m.hi[i], m.lo[i]);
      m.least[i] = least_bf16(x[2 * i], x[2 * i + 1], m.hi[i], m.lo[i]);
    }
  } else {
    make(static_cast<Made<T>&>(m), x);
  }
}

// The raw values of a left operand whose rows are a tile's rows (kTrans: columns)
template <class T, int LD, bool kTrans>
__device__ __forceinline__ void load_a(float (&x)[8], const T* tile, int m0, int k0) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  if constexpr (kHalfWord<T>) {
    uint32_t r[4];
    const T* at = kTrans ? tile + (k0 + (lane >> 4) * 8 + (lane & 7)) * LD + m0 + (lane >> 3 & 1) * 8
                         : tile + (m0 + (lane & 15)) * LD + k0 + (lane >> 4) * 8;
    ldmatrix<kTrans>(r, at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = floats_of(r[i], T{});
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + g + (i & 1) * 8, k = k0 + 2 * c + (i >> 1) * 8;
      if (kTrans) {
        x[2 * i] = tile[k * LD + m], x[2 * i + 1] = tile[(k + 1) * LD + m];
      } else {
        const float2 f = *reinterpret_cast<const float2*>(tile + m * LD + k);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  }
}
template <class T, int LD>
__device__ __forceinline__ void load_a(InA<T>& a, const T* tile, int m0, int k0) {
  if constexpr (kHalfWord<T>) {
    const int lane = threadIdx.x & 31;
    ldmatrix<false>(a.x, tile + (m0 + (lane & 15)) * LD + k0 + (lane >> 4) * 8);
  } else {
    float x[8];
    load_a<T, LD, false>(x, tile, m0, k0);
#pragma unroll
    for (int i = 0; i < 8; ++i) split_tf32(x[i], a.hi[i], a.lo[i]);
  }
}
// two right operands, of columns n0 .. n0 + 7 and n0 + 8 .. n0 + 15: columns are a tile's rows (kTrans: columns)
template <class T, int LD, bool kTrans>
__device__ __forceinline__ void load_words(uint32_t (&r)[4], const T* tile, int n0, int k0) {
  const int lane = threadIdx.x & 31, a = lane >> 4, b = lane >> 3 & 1, row = lane & 7;
  ldmatrix<kTrans>(r, kTrans ? tile + (k0 + b * 8 + row) * LD + n0 + a * 8 : tile + (n0 + a * 8 + row) * LD + k0 + b * 8);
}
template <int LD, bool kTrans>
__device__ __forceinline__ void load_floats(float (&x)[8], const float* tile, int n0, int k0) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + g + (i >> 1) * 8, k = k0 + 2 * c + (i & 1) * 8;
    if (kTrans) {
      x[2 * i] = tile[k * LD + n], x[2 * i + 1] = tile[(k + 1) * LD + n];
    } else {
      const float2 f = *reinterpret_cast<const float2*>(tile + n * LD + k);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
template <class T, int LD, bool kTrans>
__device__ __forceinline__ void load_b(InB<T> (&b)[2], const T* tile, int n0, int k0) {
  if constexpr (kHalfWord<T>) {
    uint32_t r[4];
    load_words<T, LD, kTrans>(r, tile, n0, k0);
    b[0].x[0] = r[0], b[0].x[1] = r[1], b[1].x[0] = r[2], b[1].x[1] = r[3];
  } else {
    float x[8];
    load_floats<LD, kTrans>(x, tile, n0, k0);
#pragma unroll
    for (int i = 0; i < 8; ++i) split_tf32(x[i], b[i >> 2].hi[i & 3], b[i >> 2].lo[i & 3]);
  }
}

// The state as an operand in shared memory: beside bfloat16 planes of its terms, two forward and three backward, whose products
// with it go into the decays' gradients (of two, those are 1e-6 to 3e-6 off, of three 3e-7, in 4 % more time of a backward of 64 x 64); else,
// and where three planes of two states have no room (128 x 128), 32 bits, which every warp splits that reads them (459 us with two planes,
// 607 with 32 bits, 802 with tf32 terms, of 192 rows of 1000 steps)
template <class T, bool kFlat>
using Stored = std::conditional_t<std::is_same<T, __nv_bfloat16>::value && !kFlat, __nv_bfloat16, float>;
template <class S>
constexpr bool kInPlanes = sizeof(S) == 2;

// kTerms: of bfloat16, two or three
template <class T, int LD, int PLANE, bool kTrans, int kTerms, class S>
__device__ __forceinline__ void load_state(MadeB<T> (&b)[2], const S* s, int n0, int k0) {
  if constexpr (kInPlanes<S>) {
    uint32_t r[4];
    load_words<__nv_bfloat16, LD, kTrans>(r, s, n0, k0);
    b[0].hi[0] = r[0], b[0].hi[1] = r[1], b[1].hi[0] = r[2], b[1].hi[1] = r[3];
    load_words<__nv_bfloat16, LD, kTrans>(r, s + PLANE, n0, k0);
    b[0].lo[0] = r[0], b[0].lo[1] = r[1], b[1].lo[0] = r[2], b[1].lo[1] = r[3];
    if constexpr (kTerms == 3) {
      load_words<__nv_bfloat16, LD, kTrans>(r, s + 2 * PLANE, n0, k0);
      b[0].least[0] = r[0], b[0].least[1] = r[1], b[1].least[0] = r[2], b[1].least[1] = r[3];
    }
  } else {
    float x[8];
    load_floats<LD, kTrans>(x, s, n0, k0);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        split_bf16(x[2 * i], x[2 * i + 1], b[i >> 1].hi[i & 1], b[i >> 1].lo[i & 1]);
        if constexpr (kTerms == 3) b[i >> 1].least[i & 1] = least_bf16(x[2 * i], x[2 * i + 1], b[i >> 1].hi[i & 1], b[i >> 1].lo[i & 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) split_tf32(x[i], b[i >> 2].hi[i & 3], b[i >> 2].lo[i & 3]);
    }
  }
}
// Two or four adjacent values to planes of their terms, or as they are
template <int LD, int PLANE, int kPlanes, class S>
__device__ __forceinline__ void store_state(S* s, int row, int col, float x, float y) {
  if constexpr (kInPlanes<S>) {
    uint32_t hi, lo;
    split_bf16(x, y, hi, lo);
    *reinterpret_cast<uint32_t*>(s + row * LD + col) = hi;
    *reinterpret_cast<uint32_t*>(s + PLANE + row * LD + col) = lo;
    if constexpr (kPlanes == 3) *reinterpret_cast<uint32_t*>(s + 2 * PLANE + row * LD + col) = least_bf16(x, y, hi, lo);
  } else {
    *reinterpret_cast<float2*>(s + row * LD + col) = make_float2(x, y);
  }
}
template <int PLANE>
__device__ __forceinline__ void store_state(__nv_bfloat16* at, float4 v) {
  uint2 hi, lo;
  split_bf16(v.x, v.y, hi.x, lo.x);
  split_bf16(v.z, v.w, hi.y, lo.y);
  *reinterpret_cast<uint2*>(at) = hi;
  *reinterpret_cast<uint2*>(at + PLANE) = lo;
  *reinterpret_cast<uint2*>(at + 2 * PLANE) = make_uint2(least_bf16(v.x, v.y, hi.x, lo.x), least_bf16(v.z, v.w, hi.y, lo.y));
}
// (all bits of them: of three planes)
template <int LD, int PLANE, class S>
__device__ __forceinline__ float2 read_state(const S* s, int row, int col) {
  if constexpr (kInPlanes<S>) {
    const float2 a = floats_of(*reinterpret_cast<const uint32_t*>(s + row * LD + col), S{});
    const float2 b = floats_of(*reinterpret_cast<const uint32_t*>(s + PLANE + row * LD + col), S{});
    const float2 c = floats_of(*reinterpret_cast<const uint32_t*>(s + 2 * PLANE + row * LD + col), S{});
    return make_float2(a.x + (b.x + c.x), a.y + (b.y + c.y));
  } else {
    return *reinterpret_cast<const float2*>(s + row * LD + col);
  }
}

// ------------------------------------------------------------------------------------------- products

template <class T>
__device__ __forceinline__ void widen_a(uint32_t (&w)[8], const InA<T>& a) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = floats_of(a.x[i], T{});
    w[2 * i] = __float_as_uint(f.x), w[2 * i + 1] = __float_as_uint(f.y);
  }
}
// input times input
template <class T>
__device__ __forceinline__ void mma(float (&c)[4], const InA<T>& a, const InB<T>& b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    mma_bf16(c, a.x, b.x);
  } else if constexpr (std::is_same<T, __half>::value) {
    mma_f16(c, a.x, b.x);
  } else {
    mma_tf32(c, a.hi, a.lo, b.hi, b.lo);
  }
}
// computed times input
template <class T>
__device__ __forceinline__ void mma(float (&c)[4], const Made<T>& a, const InB<T>& b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    mma_bf16(c, a.lo, b.x);
    mma_bf16(c, a.hi, b.x);
  } else if constexpr (std::is_same<T, __half>::value) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = floats_of(b.x[i], T{});
      w[2 * i] = __float_as_uint(f.x), w[2 * i + 1] = __float_as_uint(f.y);
    }
    mma_tf32(c, a.lo, w);
    mma_tf32(c, a.hi, w);
  } else {
    mma_tf32(c, a.hi, a.lo, b.hi, b.lo);
  }
}
template <class T>
__device__ __forceinline__ void mma(float (&c)[4], const Finest<T>& a, const InB<T>& b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) mma_bf16(c, a.least, b.x);
  mma(c, static_cast<const Made<T>&>(a), b);
}
// input times state
template <int kTerms, class T>
__device__ __forceinline__ void mma(float (&c)[4], const InA<T>& a, const MadeB<T>& b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    if constexpr (kTerms == 3) mma_bf16(c, a.x, b.least);
    mma_bf16(c, a.x, b.lo);
    mma_bf16(c, a.x, b.hi);
  } else if constexpr (std::is_same<T, __half>::value) {
    uint32_t w[8];
    widen_a(w, a);
    mma_tf32(c, w, b.lo);
    mma_tf32(c, w, b.hi);
  } else {
    mma_tf32(c, a.hi, a.lo, b.hi, b.lo);
  }
}

// ------------------------------------------------------------------------------------------ geometry

template <class T, int D>
constexpr int kLd = D + (sizeof(T) == 2 ? 8 : 4);  // 16 bytes of padding: eight rows' pieces lie in different banks

// One row's steps: of the n that count, scan order s is time t; those past them follow in both orders
struct Row {
  int64_t b, steps, n;
  int h, reverse;
  __device__ __forceinline__ Row(const Args& p, int64_t row) {
    b = row / p.heads;
    h = (int)(row - b * p.heads);
    steps = p.steps;
    n = steps;
    if (p.lengths) n = max((int64_t)0, min(steps, p.lengths[b]));
    reverse = p.reverse;
  }
  __device__ __forceinline__ int64_t time(int64_t s) const { return reverse && s < n ? n - 1 - s : s; }
};

// What a CTA works on: a whole row, or a part of one of those after
struct Span {
  int64_t index;
  int part, c0, c1;
  __device__ __forceinline__ Span(const Args& p, int64_t unit) {
    const bool cut = unit >= p.whole;
    index = cut ? p.whole + (unit - p.whole) / p.parts : unit;
    part = cut ? (int)((unit - p.whole) % p.parts) : 0;
    c0 = part * p.part_chunks;
    c1 = cut ? min(p.chunks, c0 + p.part_chunks) : p.chunks;
  }
};

// Rows s0 .. s0 + C - 1 of an operand to a tile, zeros for steps past the row's length.  The columns past `cols` are
// zeros from before.
template <class T, int D, int C, int THREADS>
__device__ __forceinline__ void load_tile(T* tile, const Operand& o, int first, int cols, const Row& row, int64_t s0) {
  constexpr int LD = kLd<T, D>, kPer = D * (int)sizeof(T) / 16;  // 16-byte pieces of a row
  constexpr int kRows = THREADS / kPer < C ? THREADS / kPer : C;
  static_assert(THREADS % kPer == 0 && C % kRows == 0, "");
  const int piece = threadIdx.x % kPer, r0 = threadIdx.x / kPer, bytes = cols * (int)sizeof(T) - piece * 16;
  if (bytes <= 0 || r0 >= kRows) return;
  const char* base = static_cast<const char*>(o.p) + (row.b * o.sb + row.h * o.sh + first) * (int64_t)sizeof(T) + piece * 16;
  const uint32_t to0 = smem_of(tile) + r0 * LD * (int)sizeof(T) + piece * 16;
  const int64_t step = row.reverse ? -o.st * (int64_t)sizeof(T) : o.st * (int64_t)sizeof(T);
  const char* from = base + row.time(s0 + r0) * o.st * (int64_t)sizeof(T);
  if (o.unit == 16 && s0 + C <= row.n) {
#pragma unroll
    for (int k = 0; k < C / kRows; ++k) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to0 + k * kRows * LD * (int)sizeof(T)), "l"(from) : "memory");
      from += kRows * step;
    }
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (o.unit == 2) {
      // the aligned words that hold some of the piece, shifted into place; those of several rows on their way together
      constexpr int kTogether = C / kRows < 4 ? C / kRows : 4;
      const int count = min(16, bytes) / 2;  // elements
#pragma unroll 1
      for (int k0 = 0; k0 < C / kRows; k0 += kTogether) {
        uint32_t w[kTogether][5];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
          const bool live = s0 + r0 + (k0 + k) * kRows < row.n;
          const uintptr_t at = reinterpret_cast<uintptr_t>(from) + (k0 + k) * kRows * step;
          const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
          const int last = (int)((at & 3) + 2 * count + 3) / 4;  // words
#pragma unroll
          for (int i = 0; i < 5; ++i) w[k][i] = live && i < last ? words[i] : 0u;
        }
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
          const uint32_t shift = ((reinterpret_cast<uintptr_t>(from) + (k0 + k) * kRows * step) & 2) * 8;
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] = __funnelshift_r(w[k][i], w[k][i + 1], shift);
            v[i] = 2 * i + 1 < count ? v[i] : 2 * i < count ? v[i] & 0xffffu : 0u;
          }
          *reinterpret_cast<uint4*>(reinterpret_cast<char*>(tile + (r0 + (k0 + k) * kRows) * LD) + piece * 16) =
              make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      return;
    }
  }
#pragma unroll 1
  for (int k = 0; k < C / kRows; ++k) {
    const bool live = s0 + r0 + k * kRows < row.n;
    const uint32_t to = to0 + k * kRows * LD * (int)sizeof(T);
    // (a piece that is not live is zeros, of any address)
    const char* at = live ? from : static_cast<const char*>(o.p);
    if (o.unit == 16) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(at), "r"(live ? 16 : 0) : "memory");
    } else if (o.unit == 8) {
#pragma unroll
      for (int x = 0; x < 16; x += 8)
        if (x < bytes)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to + x), "l"(live ? at + x : at), "r"(live ? 8 : 0) : "memory");
    } else {
#pragma unroll
      for (int x = 0; x < 16; x += 4)
        if (x < bytes)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + x), "l"(live ? at + x : at), "r"(live ? 4 : 0) : "memory");
    }
    from += kRows * step;
  }
}
__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Decays of a chunk's steps, by one warp.  Between load (early) and store lies the latency of the loads.
template <int C>
struct Decays {
  static constexpr int E = C / 32;
  float g[E];
  __device__ __forceinline__ void load(const Args& p, const Row& row, int64_t s0) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t s = s0 + lane * E + e;
      g[e] = 0.0f;
      if (s < row.n) {
        const int64_t t = row.time(s);
        g[e] = p.decay[row.b * p.decay_sb + t * p.decay_st + row.h * p.decay_sh];
        if (p.reset && p.reset[row.b * p.reset_sb + t * p.reset_st]) g[e] = -INFINITY;
      }
    }
  }
  __device__ __forceinline__ static double log2_of(float g) {
    return g * kLog2e < kCut ? (double)kCut : (double)g * 1.4426950408889634;  // (a NaN stays one)
  }
  // sums as two floats, e^{G_i}, e^{G_C - G_j}, and e^{G_e - G_j} to the last step e of j's sixteen
  __device__ __forceinline__ void store(float2* sums) const {
    float *before = reinterpret_cast<float*>(sums + C), *after = before + C, *tail = after + C;
    const int lane = threadIdx.x & 31;
    double own[E], total = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) own[e] = total += log2_of(g[e]);
    double up = total;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, up, off);
      if (lane >= off) up += v;
    }
    const double all = __shfl_sync(0xffffffffu, up, 31), ends = __shfl_sync(0xffffffffu, up, lane | (16 / E - 1));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double at = up - total + own[e];
      const float hi = (float)at;
      sums[lane * E + e] = make_float2(hi, (float)(at - hi));
      before[lane * E + e] = exp2_approx(hi);
      after[lane * E + e] = exp2_approx((float)(all - at));
      tail[lane * E + e] = exp2_approx((float)(ends - at));
    }
  }
};
template <int C>
constexpr int kDecayBytes = 2 * C * 20;  // of two chunks
__device__ __forceinline__ float between(float2 i, float2 j) { return exp2_approx((i.x - j.x) + (i.y - j.y)); }
// Weights scale L of a thread's eighths of a 16 x 16 block, as `make` takes them: rows i0, i1 = i0 + 8 of steps i, columns of
// steps j0 + 2c, + 1, + 8, + 9.  Where every i is past every j, L is e^{G_i - G_e} e^{G_e - G_j} with e the last of the
// sixteen j, both of them 1 at most: two exponentials a thread instead of eight.
__device__ __forceinline__ void weights_by_row(float (&w)[8], const float2* sums, const float* tail, int i0, int j0, bool diagonal,
                                               float scale) {
  const int j = j0 + 2 * (threadIdx.x & 3);
  const float2 sum0 = sums[i0], sum1 = sums[i0 + 8];
  if (!diagonal) {
    const float2 end = sums[j0 + 15];
    const float f0 = scale * between(sum0, end), f1 = scale * between(sum1, end);
    const float2 t0 = *reinterpret_cast<const float2*>(tail + j), t1 = *reinterpret_cast<const float2*>(tail + j + 8);
    w[0] = f0 * t0.x, w[1] = f0 * t0.y, w[2] = f1 * t0.x, w[3] = f1 * t0.y;
    w[4] = f0 * t1.x, w[5] = f0 * t1.y, w[6] = f1 * t1.x, w[7] = f1 * t1.y;
    return;
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int at = j + 8 * half;
    const float4 two = *reinterpret_cast<const float4*>(sums + at);
    const float2 a = make_float2(two.x, two.y), b = make_float2(two.z, two.w);
    w[4 * half] = at <= i0 ? scale * between(sum0, a) : 0.0f;
    w[4 * half + 1] = at + 1 <= i0 ? scale * between(sum0, b) : 0.0f;
    w[4 * half + 2] = at <= i0 + 8 ? scale * between(sum1, a) : 0.0f;
    w[4 * half + 3] = at + 1 <= i0 + 8 ? scale * between(sum1, b) : 0.0f;
  }
}
// The same of the transpose: rows of steps j = j0, j0 + 8, columns of steps i0 + 2c ..
__device__ __forceinline__ void weights_by_column(float (&w)[8], const float2* sums, const float* tail, int j0, int i0, int block,
                                                  bool diagonal, float scale) {
  const int i = i0 + 2 * (threadIdx.x & 3);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int at = i + 8 * half;
    const float4 two = *reinterpret_cast<const float4*>(sums + at);
    const float2 a = make_float2(two.x, two.y), b = make_float2(two.z, two.w);
    if (!diagonal) {
      const float2 end = sums[block + 15];  // (of j's sixteen)
      const float f0 = scale * between(a, end), f1 = scale * between(b, end), t0 = tail[j0], t1 = tail[j0 + 8];
      w[4 * half] = f0 * t0, w[4 * half + 1] = f1 * t0, w[4 * half + 2] = f0 * t1, w[4 * half + 3] = f1 * t1;
    } else {
      const float2 sum0 = sums[j0], sum1 = sums[j0 + 8];
      w[4 * half] = j0 <= at ? scale * between(a, sum0) : 0.0f;
      w[4 * half + 1] = j0 <= at + 1 ? scale * between(b, sum0) : 0.0f;
      w[4 * half + 2] = j0 + 8 <= at ? scale * between(a, sum1) : 0.0f;
      w[4 * half + 3] = j0 + 8 <= at + 1 ? scale * between(b, sum1) : 0.0f;
    }
  }
}
// a factor of zero cuts off whatever it multiplies
__device__ __forceinline__ float decayed(float factor, float x) { return factor == 0.0f ? 0.0f : factor * x; }

// 16 rows of N times 8 columns times their rows' factors
template <int N>
__device__ __forceinline__ void decay_rows(float (&x)[N][4], float f0, float f1) {
  if (__any_sync(0xffffffffu, f0 == 0.0f || f1 == 0.0f)) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (f0 == 0.0f) x[n][0] = x[n][1] = 0.0f;
      if (f1 == 0.0f) x[n][2] = x[n][3] = 0.0f;
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) x[n][0] *= f0, x[n][1] *= f0, x[n][2] *= f1, x[n][3] *= f1;
}

// A warp's part of a DK x DV state: kTiles tiles of 16 rows, kCols columns
template <int DK, int DV, int WARPS>
struct StateShape {
  static constexpr int kRowWarps = WARPS < DK / 16 ? WARPS : DK / 16;
  static constexpr int kColWarps = WARPS / kRowWarps;
  static constexpr int kTiles = DK / 16 / kRowWarps;
  static constexpr int kCols = DV / kColWarps;
  static_assert(kCols % 16 == 0, "");
};
template <int DK, int DV, int WARPS>
struct State {
  using Shape = StateShape<DK, DV, WARPS>;
  float x[Shape::kTiles][Shape::kCols / 8][4];

  // (warps past the first WARPS have no part in it)
  // its tiles of 16 rows and blocks of 16 columns lie in turn with the other warps', so that a state narrower than DK x DV
  // is shared out evenly too
  static __device__ __forceinline__ int row_of(int tile) {
    return (tile * Shape::kRowWarps + (int)(threadIdx.x >> 5) % Shape::kRowWarps) * 16;
  }
  static __device__ __forceinline__ int col_of(int block) {
    return (block * Shape::kColWarps + (int)(threadIdx.x >> 5) / Shape::kRowWarps) * 16;
  }
  // f(row, column, value of it, of the next column), rows and columns of the state, of tiles within `rows` and `cols`
  template <class F>
  __device__ __forceinline__ void each(F f, int rows = DK, int cols = DV) {
    const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
#pragma unroll
    for (int m = 0; m < Shape::kTiles; ++m) {
      if (row_of(m) >= rows) continue;
#pragma unroll
      for (int n = 0; n < Shape::kCols / 8; ++n) {
        if (col_of(n / 2) >= cols) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half)
          f(row_of(m) + g + half * 8, col_of(n / 2) + n % 2 * 8 + 2 * c, x[m][n][2 * half], x[m][n][2 * half + 1]);
      }
    }
  }
  // from a dense [key, value] matrix's columns from `first`, or zeros
  __device__ __forceinline__ void read(const float* from, int key, int value, int first) {
    each([&](int r, int c, float& a, float& b) {
      const bool in = from && r < key;
      a = in && first + c < value ? from[(int64_t)r * value + first + c] : 0.0f;
      b = in && first + c + 1 < value ? from[(int64_t)r * value + first + c + 1] : 0.0f;
    });
  }
  __device__ __forceinline__ void write(float* to, int key, int value, int first) {
    each([&](int r, int c, float& a, float& b) {
      if (r < key && first + c < value) to[(int64_t)r * value + first + c] = a;
      if (r < key && first + c + 1 < value) to[(int64_t)r * value + first + c + 1] = b;
    });
  }
  // What a part begins from: the row's state `from`, and what the parts before it in scan order (after it, kBackward) add
  template <bool kBackward>
  __device__ __forceinline__ void begin(const Args& p, int64_t index, int part, const float* from, int padded, int first) {
    if (index < p.whole) {
      read(from, p.key, p.value, first);
      return;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // for the sweep, or the join, which this kernel is launched close to
    const int64_t cut = (index - p.whole) * p.parts;
    const float* starts = p.starts + cut * DK * padded;
    if (p.joined) {
      read(starts + (int64_t)part * DK * padded, DK, padded, first);
      return;
    }
    read(from, p.key, p.value, first);
#pragma unroll 1
    for (int i = kBackward ? p.parts - 1 : 0; i != part; i += kBackward ? -1 : 1) {
      const float factor = p.factors[cut + i];
      const float* add = starts + (int64_t)i * DK * padded + first;
      each([&](int r, int c, float& a, float& b) {
        const float2 more = *reinterpret_cast<const float2*>(add + (int64_t)r * padded + c);
        a = decayed(factor, a) + more.x, b = decayed(factor, b) + more.y;
      });
    }
  }
  // S = factor S + sum over the chunk's steps of weight a b^T.  The chunk's sum is made by itself and added, rounded: the
  // instruction cuts off what its accumulator does not hold, which over the chunks that a slow head remembers is 1e-5.
  template <class T, int C>
  __device__ __forceinline__ void update(const T* a, const T* b, const float* weights, float factor, float scale, int rows, int cols) {
    const int c = threadIdx.x & 3;
    if (factor == 0.0f) {  // (cuts off whatever the state holds)
#pragma unroll
      for (int m = 0; m < Shape::kTiles; ++m)
#pragma unroll
        for (int n = 0; n < Shape::kCols / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[m][n][e] = 0.0f;
    }
    constexpr int kBlocks = C / 16, kTogether = 2;  // of registers' worth
#pragma unroll
    for (int m = 0; m < Shape::kTiles; ++m) {
      if (row_of(m) >= rows) continue;
#pragma unroll
      for (int k0 = 0; k0 < kBlocks; k0 += kTogether) {
        Finest<T> left[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
          const int at = (k0 + k) * 16;
          const float2 w0 = *reinterpret_cast<const float2*>(weights + at + 2 * c);
          const float2 w1 = *reinterpret_cast<const float2*>(weights + at + 8 + 2 * c);
          float f[8];
          load_a<T, kLd<T, DK>, true>(f, a, row_of(m), at);
          f[0] *= w0.x * scale, f[1] *= w0.y * scale, f[2] *= w0.x * scale, f[3] *= w0.y * scale;
          f[4] *= w1.x * scale, f[5] *= w1.y * scale, f[6] *= w1.x * scale, f[7] *= w1.y * scale;
          make(left[k], f);
        }
#pragma unroll
        for (int n = 0; n < Shape::kCols / 16; ++n) {
          if (col_of(n) >= cols) continue;
          float sum[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
          for (int k = 0; k < kTogether; ++k) {
            InB<T> right[2];
            load_b<T, kLd<T, DV>, true>(right, b, col_of(n), (k0 + k) * 16);
            mma(sum[0], left[k], right[0]);
            mma(sum[1], left[k], right[1]);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& s = x[m][2 * n + half][e];
              s = k0 == 0 ? fmaf(factor, s, sum[half][e]) : s + sum[half][e];
            }
        }
      }
    }
  }
  // to shared memory, as an operand
  template <int kPlanes, class S>
  __device__ __forceinline__ void publish(S* s, int rows, int cols) {
    constexpr int LD = kLd<S, DV>;
    each([&](int r, int c, float& a, float& b) { store_state<LD, DK * LD, kPlanes>(s, r, c, a, b); }, rows, cols);
  }
};

// Bytes of the state before a chunk: 32 bits of [DK][DV]
__host__ __device__ constexpr int64_t kept_bytes(int DK, int DV) { return (int64_t)4 * DK * DV; }

__device__ __forceinline__ float2 narrow_pair(float x, float y, float) { return make_float2(x, y); }
// A warp's 16 rows of N times 8 columns to rows of `width`: those of steps s and s + 8, where they are within the row; zeros
// past its length.  The columns are blocks of 16, WC blocks apart, the thread's first at col
template <class T, int WC, int N>
__device__ __forceinline__ void store_rows(void* base, const Args& p, const Row& row, int64_t s, int width, int col, const float (&x)[N][4]) {
  constexpr auto column = [](int n) { return n / 2 * WC * 16 + n % 2 * 8; };
  constexpr int kLast = (N - 1) / 2 * WC * 16 + (N - 1) % 2 * 8;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int64_t at = s + 8 * half;
    if (at >= row.steps) continue;
    const bool live = at < row.n;
    T* to = static_cast<T*>(base) + ((row.b * row.steps + row.time(at)) * p.heads + row.h) * width + col;
    const int left = width - col;
    if (width % 2 == 0) {
      using Pair = decltype(narrow_pair(0.0f, 0.0f, T{}));
      Pair* pairs = reinterpret_cast<Pair*>(to);
      if (live && kLast < left) {
#pragma unroll
        for (int n = 0; n < N; ++n) pairs[column(n) / 2] = narrow_pair(x[n][2 * half], x[n][2 * half + 1], T{});
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (column(n) < left) pairs[column(n) / 2] = narrow_pair(live ? x[n][2 * half] : 0.0f, live ? x[n][2 * half + 1] : 0.0f, T{});
      }
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (column(n) < left) to[column(n)] = narrow<T>(live ? x[n][2 * half] : 0.0f);
        if (column(n) + 1 < left) to[column(n) + 1] = narrow<T>(live ? x[n][2 * half + 1] : 0.0f);
      }
    }
  }
}
// two adjacent values of a tile
template <class T>
__device__ __forceinline__ float2 two_of(const T* at) {
  if constexpr (kHalfWord<T>) return floats_of(*reinterpret_cast<const uint32_t*>(at), T{});
  else return *reinterpret_cast<const float2*>(at);
}

template <int THREADS>
__device__ __forceinline__ void clear(void* p, int bytes) {
  uint4* q = static_cast<uint4*>(p);
  for (int i = threadIdx.x; i < bytes / 16; i += THREADS) q[i] = make_uint4(0u, 0u, 0u, 0u);
}

// Loops over the channels of a contraction.  Where a product is many instructions, code that repeats them outgrows the
// instruction cache (two thirds of the stalls of a float32 forward)
template <class T, class S = T>
constexpr int kUnroll = std::is_same<T, __nv_bfloat16>::value && kHalfWord<S> ? 4 : 1;

// 16 rows of a from m0 times 16 rows of b from n0, over their channels, `width` of at most D
template <class T, int D>
__device__ __forceinline__ void products(float (&sum)[2][4], const T* a, int m0, const T* b, int n0, int width) {
#pragma unroll kUnroll<T>
  for (int kk = 0; kk < D; kk += 16) {
    if (kk >= width) break;
    InA<T> left;
    InB<T> right[2];
    load_a<T, kLd<T, D>>(left, a, m0, kk);
    load_b<T, kLd<T, D>, false>(right, b, n0, kk);
    mma(sum[0], left, right[0]);
    mma(sum[1], left, right[1]);
  }
}

// 16 rows of a from m0, over their channels, `width` of at most D, times a state's columns (kTrans; else its rows), those of the
// blocks of 16 in turn from wc that lie within `cols`
template <class T, int D, int LDS, int PLANE, bool kTrans, int WC, int kTerms, class S, int N>
__device__ __forceinline__ void times_state(float (&out)[N][4], const T* a, int m0, const S* state, int wc, int width, int cols) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) out[n][e] = 0.0f;
#pragma unroll (kUnroll<T, S>)
  for (int kk = 0; kk < D; kk += 16) {
    if (kk >= width) break;
    InA<T> left;
    load_a<T, kLd<T, D>>(left, a, m0, kk);
#pragma unroll
    for (int n = 0; n < N / 2; ++n) {
      if ((n * WC + wc) * 16 >= cols) continue;
      MadeB<T> right[2];
      load_state<T, LDS, PLANE, kTrans, kTerms>(right, state, (n * WC + wc) * 16, kk);
      mma<kTerms>(out[2 * n], left, right[0]);
      mma<kTerms>(out[2 * n + 1], left, right[1]);
    }
  }
}
// A computed 16 x 16 block times 16 rows of b from k0, the same columns of it
template <class T, int LD, int WC, int N>
__device__ __forceinline__ void add_product(float (&out)[N][4], const Made<T>& left, const T* b, int k0, int wc, int cols) {
#pragma unroll
  for (int n = 0; n < N / 2; ++n) {
    if ((n * WC + wc) * 16 >= cols) continue;
    InB<T> right[2];
    load_b<T, LD, true>(right, b, (n * WC + wc) * 16, k0);
    mma(out[2 * n], left, right[0]);
    mma(out[2 * n + 1], left, right[1]);
  }
}
// sums over the same columns of x times a tile's rows i0 and i0 + 8; in every lane of a row
template <class T, int LD, int WC, int N>
__device__ __forceinline__ float2 row_sums(const float (&x)[N][4], const T* tile, int i0, int wc) {
  float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const T* at = tile + i0 * LD + (n / 2 * WC + wc) * 16 + n % 2 * 8 + 2 * (threadIdx.x & 3);
    const float2 a = two_of(at), b = two_of(at + 8 * LD);
    s0 = fmaf(x[n][0], a.x, fmaf(x[n][1], a.y, s0));
    s1 = fmaf(x[n][2], b.x, fmaf(x[n][3], b.y, s1));
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    s0 += __shfl_xor_sync(0xffffffffu, s0, off);
    s1 += __shfl_xor_sync(0xffffffffu, s1, off);
  }
  return make_float2(s0, s1);
}
__device__ __forceinline__ int sixteens(int n) { return (n + 15) & ~15; }

// ------------------------------------------------------------------------------------------- forward

template <class T, int DK, int DV, int C>
struct ForwardShared {
  static constexpr int kTiles = (2 * C * kLd<T, DK> + C * kLd<T, DV>) * (int)sizeof(T);
  using S = Stored<T, false>;
  static constexpr int kPlanes = kInPlanes<S> ? 2 : 1;
  static constexpr int kState = kPlanes * DK * kLd<S, DV> * (int)sizeof(S);
  static constexpr int kDecays = kDecayBytes<C>;
  // the next chunk's tiles come in while one is worked on, where three CTAs an SM have the room (of 896 rows of 500 steps
  // four CTAs with one set of tiles are 6 % slower, of 448 rows 12 % faster)
  static constexpr int kStages = 2 * kTiles + kState + kDecays <= (75 << 10) ? 2 : 1;
  static constexpr int kBytes = kStages * kTiles + kState + kDecays;
};

// kWhole: keys and values fill DK and DV (the loops over less would keep the compiler from mixing their rounds: 20 % of a
// forward and 35 % of a backward)
template <class T, int DK, int DV, int C, bool kWhole>
__global__ void __launch_bounds__(128, DK > 64 ? 2 : 3) forward_kernel(const __grid_constant__ Args p) {
  constexpr int THREADS = 128, WARPS = 4, RG = C / 16, WC = WARPS / RG, NY = DV / WC / 8;
  using Sh = ForwardShared<T, DK, DV, C>;
  constexpr int LDK = kLd<T, DK>, LDV = kLd<T, DV>, LDS = kLd<typename Sh::S, DV>, PLANE = DK * LDS;
  extern __shared__ __align__(16) char shared[];
  char* tiles = shared;
  auto* s_state = reinterpret_cast<typename Sh::S*>(shared + Sh::kStages * Sh::kTiles);
  char* decays = shared + Sh::kStages * Sh::kTiles + Sh::kState;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int rg = warp % RG, wc = warp / RG;

  const int slice = blockIdx.x % p.slices;
  const Span span(p, blockIdx.x / p.slices);
  const int64_t index = span.index;
  const int part = span.part, c0 = span.c0, c1 = span.c1;
  const Row row(p, index);
  const int first = slice * DV, cols = min(DV, p.value - first);
  const int padded = DV * p.slices;  // columns of the states in memory
  const int key = kWhole ? DK : sixteens(p.key), value = kWhole ? DV : sixteens(cols);

  clear<THREADS>(shared, Sh::kStages * Sh::kTiles);
  State<DK, DV, WARPS> S;
  S.template begin<false>(p, index, part, p.state ? p.state + index * p.key * p.value : nullptr, padded, first);
  S.template publish<Sh::kPlanes>(s_state, key, value);
  __syncthreads();

  const auto q_of = [&](int stage) { return reinterpret_cast<T*>(tiles + stage * Sh::kTiles); };
  const auto load = [&](int chunk, int stage) {
    T* q = q_of(stage);
    const int64_t s0 = (int64_t)chunk * C;
    if (s0 < row.n) {
      load_tile<T, DK, C, THREADS>(q, p.q, 0, p.key, row, s0);
      load_tile<T, DK, C, THREADS>(q + C * LDK, p.k, 0, p.key, row, s0);
      load_tile<T, DV, C, THREADS>(q + 2 * C * LDK, p.v, first, cols, row, s0);
    }
    copies_issued();
  };
  const auto sums_of = [&](int chunk) { return reinterpret_cast<float2*>(decays + (chunk & 1) * C * 20); };
  Decays<C> next;
  load(c0, 0);
  if (warp == WARPS - 1) {
    next.load(p, row, (int64_t)c0 * C);
    next.store(sums_of(c0));
  }
#pragma unroll 1
  for (int chunk = c0; chunk < c1; ++chunk) {
    const int stage = Sh::kStages == 2 ? (chunk - c0) & 1 : 0;
    const int64_t s0 = (int64_t)chunk * C;
    copies_done();
    __syncthreads();  // the chunk's tiles, decays and state are there
    if (Sh::kStages == 2 && chunk + 1 < c1) load(chunk + 1, stage ^ 1);
    if (warp == WARPS - 1 && chunk + 1 < c1) next.load(p, row, s0 + C);
    const T *q = q_of(stage), *k = q + C * LDK, *v = q + 2 * C * LDK;
    const float2* sums = sums_of(chunk);
    const float *before = reinterpret_cast<const float*>(sums + C), *after = before + C, *tail = after + C;
    const bool live = s0 < row.n;
    if (live && p.kept) {  // the state before the chunk, for the backward
      float* to = reinterpret_cast<float*>(static_cast<char*>(p.kept) + (index * p.chunks + chunk) * kept_bytes(DK, padded)) + first;
      if constexpr (kInPlanes<typename Sh::S>) {
        S.each([&](int r, int col, float& a, float& b) { *reinterpret_cast<float2*>(to + (int64_t)r * padded + col) = make_float2(a, b); },
               key, value);
      } else {
        constexpr int kPieces = DV / 4;
        const int piece = threadIdx.x % kPieces * 4;
        if (piece < value) {
#pragma unroll 4
          for (int r = threadIdx.x / kPieces; r < key; r += THREADS / kPieces)
            *reinterpret_cast<float4*>(to + (int64_t)r * padded + piece) = *reinterpret_cast<const float4*>(s_state + r * LDS + piece);
        }
      }
    }
    float y[NY][4];
    if (live) {
      const int i0 = rg * 16 + g;
      times_state<T, DK, LDS, PLANE, true, WC, 2>(y, q, rg * 16, s_state, wc, key, value);
      decay_rows(y, before[i0] * p.scale, before[i0 + 8] * p.scale);
      // sixteen steps j at a time, up to the warp's own
#pragma unroll 1
      for (int n = 0; n <= rg; ++n) {
        float a[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        products<T, DK>(a, q, rg * 16, k, n * 16, key);
        float w[8], x[8];
        weights_by_row(w, sums, tail, i0, n * 16, n == rg, p.scale);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = a[e >> 2][e & 3] * w[e];
        Made<T> left;
        make(left, x);
        add_product<T, LDV, WC>(y, left, v, n * 16, wc, value);
      }
      S.template update<T, C>(k, v, after, before[C - 1], 1.0f, key, value);
    } else {
#pragma unroll
      for (int n = 0; n < NY; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[n][e] = 0.0f;
    }
    store_rows<T, WC>(p.y, p, row, s0 + rg * 16 + g, p.value, first + wc * 16 + 2 * c, y);
    if (warp == WARPS - 1 && chunk + 1 < c1) {
      next.store(sums_of(chunk + 1));
    }
    __syncthreads();  // the chunk's tiles and state are read
    if (live) S.template publish<Sh::kPlanes>(s_state, key, value);
    if (Sh::kStages == 1 && chunk + 1 < c1) load(chunk + 1, 0);
  }
  if (p.last && c1 == p.chunks) S.write(p.last + index * p.key * p.value, p.key, p.value, first);
}

// ------------------------------------------------------------------------------------- states of parts

// What a part's steps add to the state, and its decay: from keys and values in scan order (kBackward: from queries and
// the upstream gradient, from the end)
template <class T, int DK, int DV, int C>
struct SweepShared {
  static constexpr int kTiles = C * (kLd<T, DK> + kLd<T, DV>) * (int)sizeof(T);
  static constexpr int kDecays = kDecayBytes<C>;
  static constexpr int kBytes = 2 * kTiles + kDecays;
};
template <class T, int DK, int DV, int C, bool kWhole, bool kBackward>
__global__ void __launch_bounds__(128) sweep_kernel(const __grid_constant__ Args p) {
  constexpr int THREADS = 128, WARPS = 4;
  using Sh = SweepShared<T, DK, DV, C>;
  constexpr int LDK = kLd<T, DK>;
  extern __shared__ __align__(16) char shared[];
  char* decays = shared + 2 * Sh::kTiles;
  const int warp = threadIdx.x >> 5;
  const int slice = blockIdx.x % p.slices;
  const int64_t unit = blockIdx.x / p.slices;  // of the rows that are cut
  const Span span(p, p.whole + unit);
  const int part = span.part, c0 = span.c0, c1 = span.c1;
  const Row row(p, span.index);
  const int first = slice * DV, cols = min(DV, p.value - first), padded = DV * p.slices;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (part == (kBackward ? 0 : p.parts - 1)) return;  // (nothing begins from it)
  clear<THREADS>(shared, 2 * Sh::kTiles);
  State<DK, DV, WARPS> S;
  S.read(nullptr, 0, 0, 0);
  float factor = 1.0f;
  __syncthreads();
  const auto load = [&](int chunk, int stage) {
    T* a = reinterpret_cast<T*>(shared + stage * Sh::kTiles);
    const int64_t s0 = (int64_t)chunk * C;
    if (s0 < row.n) {
      load_tile<T, DK, C, THREADS>(a, kBackward ? p.q : p.k, 0, p.key, row, s0);
      load_tile<T, DV, C, THREADS>(a + C * LDK, kBackward ? p.dy : p.v, first, cols, row, s0);
    }
    copies_issued();
  };
  const int count = c1 - c0;
  const auto chunk_of = [&](int i) { return kBackward ? c1 - 1 - i : c0 + i; };
  const auto sums_of = [&](int i) { return reinterpret_cast<float2*>(decays + (i & 1) * C * 20); };
  Decays<C> next;
  const auto store = [&](int i) {
    next.store(sums_of(i));
  };
  load(chunk_of(0), 0);
  if (warp == WARPS - 1) {
    next.load(p, row, (int64_t)chunk_of(0) * C);
    store(0);
  }
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    copies_done();
    __syncthreads();
    if (i + 1 < count) {
      load(chunk_of(i + 1), (i + 1) & 1);
      if (warp == WARPS - 1) next.load(p, row, (int64_t)chunk_of(i + 1) * C);
    }
    if ((int64_t)chunk_of(i) * C < row.n) {
      const T* a = reinterpret_cast<const T*>(shared + (i & 1) * Sh::kTiles);
      const float *before = reinterpret_cast<const float*>(sums_of(i) + C), *after = before + C;
      S.template update<T, C>(a, a + C * LDK, kBackward ? before : after, before[C - 1], kBackward ? p.scale : 1.0f,
                              kWhole ? DK : sixteens(p.key), kWhole ? DV : sixteens(cols));
      factor *= before[C - 1];
    }
    if (warp == WARPS - 1 && i + 1 < count) store(i + 1);
    __syncthreads();
  }
  S.write(p.starts + unit * DK * padded, DK, padded, first);
  if (threadIdx.x == 0 && slice == 0) p.factors[unit] = factor;
}

// What the parts add, to the states that they begin from; a thread takes an element of a row's state
template <int kThreads>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ Args p, int DK, int DV, int backward) {
  asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
  const int64_t size = (int64_t)DK * DV, per = (size + kThreads - 1) / kThreads;
  const int64_t cut = blockIdx.x / per, index = p.whole + cut, at = (blockIdx.x - cut * per) * kThreads + threadIdx.x;
  if (at >= size) return;
  const int r = (int)(at / DV), c = (int)(at - (int64_t)r * DV);
  const float* from = backward ? p.dlast : p.state;
  float s = from && r < p.key && c < p.value ? from[(index * p.key + r) * p.value + c] : 0.0f;
  float* starts = p.starts + cut * p.parts * size + at;
  const float* factors = p.factors + cut * p.parts;
  constexpr int kAhead = 8;  // parts whose loads are on their way together
  for (int i0 = 0; i0 < p.parts; i0 += kAhead) {
    float add[kAhead], factor[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k, part = backward ? p.parts - 1 - i : i;
      const bool in = i + 1 < p.parts;
      add[k] = in ? starts[part * size] : 0.0f;
      factor[k] = in ? factors[part] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k, part = backward ? p.parts - 1 - i : i;
      if (i >= p.parts) break;
      starts[part * size] = s;
      s = decayed(factor[k], s) + add[k];
    }
  }
}

// ------------------------------------------------------------------------------------------ backward

// Half the warps work by rows i (dQ, and the state's gradient, which takes about as long as the rest of the other half),
// half by rows j (dK and dV).
template <class T, int DK, int DV>
constexpr int kSide = DK > 64 || DV > 64 ? 8 : 4;

template <class T, int DK, int DV, int C>
struct BackwardShared {
  static constexpr int SIDE = kSide<T, DK, DV>, WC = SIDE / (C / 16);
  static constexpr int kTiles = 2 * C * (kLd<T, DK> + kLd<T, DV>) * (int)sizeof(T);
  // (beside bfloat16 two states of three planes, 209 KB of 128 x 128)
  using S = Stored<T, DK * DV == 128 * 128>;
  static constexpr int kState = (kInPlanes<S> ? 3 : 1) * DK * kLd<S, DV> * (int)sizeof(S);
  static constexpr int kDecays = kDecayBytes<C>;
  static constexpr int kSums = ((2 * WC + C / 16 + 1) * C + SIDE) * 4;
  static constexpr int kBytes = kTiles + 2 * kState + kDecays + kSums;
};

template <class T, int DK, int DV, int C, bool kWhole>
__global__ void __launch_bounds__(64 * kSide<T, DK, DV>, kSide<T, DK, DV> == 4 ? 2 : 1)
    backward_kernel(const __grid_constant__ Args p) {
  using Sh = BackwardShared<T, DK, DV, C>;
  constexpr int SIDE = Sh::SIDE, WARPS = 2 * SIDE, THREADS = 32 * WARPS, RG = C / 16, WC = Sh::WC;
  constexpr int NK = DK / WC / 8, NV = DV / WC / 8;
  constexpr int LDK = kLd<T, DK>, LDV = kLd<T, DV>, LDS = kLd<typename Sh::S, DV>, PLANE = DK * LDS;
  constexpr bool kPlanes = kInPlanes<typename Sh::S>;
  extern __shared__ __align__(16) char shared[];
  T *q = reinterpret_cast<T*>(shared), *k = q + C * LDK, *v = k + C * LDK, *dy = v + C * LDV;
  auto* s_state = reinterpret_cast<typename Sh::S*>(shared + Sh::kTiles);  // before the chunk
  auto* s_grad = reinterpret_cast<typename Sh::S*>(shared + Sh::kTiles + Sh::kState);
  char* decays = shared + Sh::kTiles + 2 * Sh::kState;
  float* s_far = reinterpret_cast<float*>(decays + Sh::kDecays);  // [WC][C]: scale e^{G_i} q_i S dy_i
  float* s_end = s_far + WC * C;                                  // [WC][C]: e^{G_C - G_j} k_j dS v_j
  float* s_row = s_end + WC * C;                                  // [RG][C]: sums of W over sixteen j, of each i
  float* s_col = s_row + RG * C;                                  // [C]: over i, of each j
  float* s_all = s_col + C;                                       // [SIDE]: <S, dS>
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const bool by_rows = warp < SIDE;
  const int rg = warp % SIDE % RG, wc = warp % SIDE / RG;

  const Span span(p, blockIdx.x);
  const int64_t index = span.index;
  const int part = span.part, c0 = span.c0, c1 = span.c1;
  const Row row(p, index);

  const int key = kWhole ? DK : sixteens(p.key), value = kWhole ? DV : sixteens(p.value);

  clear<THREADS>(shared, Sh::kTiles);
  State<DK, DV, SIDE> S;  // the gradient of the state, of the warps by rows
  if (by_rows) {
    S.template begin<true>(p, index, part, p.dlast ? p.dlast + index * p.key * p.value : nullptr, DV, 0);
    S.template publish<3>(s_grad, key, value);
  } else if (index >= p.whole) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
  __syncthreads();

  const auto kept_of = [&](int chunk) {
    return reinterpret_cast<const float*>(static_cast<const char*>(p.kept) + (index * p.chunks + chunk) * kept_bytes(DK, DV));
  };
  const auto load = [&](int chunk) {
    const int64_t s0 = (int64_t)chunk * C;
    if (s0 < row.n) {
      load_tile<T, DK, C, THREADS>(q, p.q, 0, p.key, row, s0);
      load_tile<T, DK, C, THREADS>(k, p.k, 0, p.key, row, s0);
      load_tile<T, DV, C, THREADS>(v, p.v, 0, p.value, row, s0);
      load_tile<T, DV, C, THREADS>(dy, p.dy, 0, p.value, row, s0);
      if constexpr (!kPlanes) {
        constexpr int kPieces = DV / 4;
        const int piece = threadIdx.x % kPieces * 4;
        const float* at = kept_of(chunk) + piece;
        if (piece < value) {
#pragma unroll 4
          for (int r = threadIdx.x / kPieces; r < key; r += THREADS / kPieces)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_of(s_state + r * LDS + piece)), "l"(at + (int64_t)r * DV) : "memory");
        }
      }
    }
    copies_issued();
  };
  // The state before a chunk to its planes, by the warps that hold no state
  const auto split = [&](int chunk) {
    if constexpr (kPlanes) {
      constexpr int kPieces = DV / 4, kRows = 32 * SIDE / kPieces;
      static_assert(DK % kRows == 0, "");
      if (by_rows || (int64_t)chunk * C >= row.n) return;
      const int t = threadIdx.x - 32 * SIDE;
      const float4* at = reinterpret_cast<const float4*>(kept_of(chunk)) + t;
      float4 v[DK / kRows];
#pragma unroll
      for (int i = 0; i < DK / kRows; ++i) v[i] = at[i * 32 * SIDE];
#pragma unroll
      for (int i = 0; i < DK / kRows; ++i) store_state<PLANE>(s_state + (t / kPieces + i * kRows) * LDS + t % kPieces * 4, v[i]);
    }
  };
  // There is no room for a chunk's tiles while another's are worked on: they come as far as the L2 cache meanwhile (896 rows of 500
  // steps of 64 x 64: 2 % of bfloat16's time, 7 % of float16's)
  const auto fetch = [&](int chunk) {
    const int64_t s0 = (int64_t)chunk * C;
#pragma unroll 1
    for (int i = threadIdx.x; i < 4 * C; i += THREADS) {
      const Operand& o = i < C ? p.q : i < 2 * C ? p.k : i < 3 * C ? p.v : p.dy;
      const int64_t s = s0 + i % C;
      if (s >= row.n) continue;
      const char* at = static_cast<const char*>(o.p) + (row.b * o.sb + row.time(s) * o.st + row.h * o.sh) * (int64_t)sizeof(T);
      for (int x = 0; x < (i < 2 * C ? p.key : p.value) * (int)sizeof(T); x += 128) prefetch(at + x);
    }
    if (s0 < row.n) {
      const char* at = reinterpret_cast<const char*>(kept_of(chunk));
      for (int x = threadIdx.x * 128; x < DK * DV * 4; x += THREADS * 128) prefetch(at + x);
    }
  };
  const auto sums_of = [&](int chunk) { return reinterpret_cast<float2*>(decays + (chunk & 1) * C * 20); };
  Decays<C> now, next;
  const auto store = [&](int chunk) {
    next.store(sums_of(chunk));
    now = next;
  };
  load(c1 - 1);
  split(c1 - 1);
  if (warp == WARPS - 1) {
    next.load(p, row, (int64_t)(c1 - 1) * C);
    store(c1 - 1);
  }
#pragma unroll 1
  for (int chunk = c1 - 1; chunk >= c0; --chunk) {
    const int64_t s0 = (int64_t)chunk * C;
    copies_done();
    __syncthreads();
    if (chunk > c0) fetch(chunk - 1);
    if (warp == WARPS - 1 && chunk > c0) next.load(p, row, s0 - C);
    const float2* sums = sums_of(chunk);
    const float *before = reinterpret_cast<const float*>(sums + C), *after = before + C, *tail = after + C;
    const bool live = s0 < row.n;
    const int i0 = rg * 16 + g;  // the warp's rows are i0 and i0 + 8, i or j
    if (by_rows) {
      float dq[NK][4];
      if (live) {
        times_state<T, DV, LDS, PLANE, false, WC, 3>(dq, dy, rg * 16, s_state, wc, value, key);
        decay_rows(dq, before[i0] * p.scale, before[i0 + 8] * p.scale);
        const float2 far = row_sums<T, LDK, WC>(dq, q, i0, wc);
        if (c == 0) s_far[wc * C + i0] = far.x, s_far[wc * C + i0 + 8] = far.y;
#pragma unroll 1
        for (int n = 0; n <= rg; ++n) {
          float d[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
          products<T, DV>(d, dy, rg * 16, v, n * 16, value);
          float w[8], x[8];
          weights_by_row(w, sums, tail, i0, n * 16, n == rg, p.scale);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = d[e >> 2][e & 3] * w[e];
          Made<T> left;
          make(left, x);
          add_product<T, LDK, WC>(dq, left, k, n * 16, wc, key);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) dq[n][e] = 0.0f;
      }
      store_rows<T, WC>(p.dq, p, row, s0 + i0, p.key, wc * 16 + 2 * c, dq);
      if (live) {
        // what passes the chunk whole
        float all = 0.0f;
        S.each([&](int r, int col, float& x, float& y) {
          const float2 s = read_state<LDS, PLANE>(s_state, r, col);
          all = fmaf(x, s.x, fmaf(y, s.y, all));
        }, key, value);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
        if (lane == 0) s_all[warp] = decayed(before[C - 1], all);
        S.template update<T, C>(q, dy, before, before[C - 1], p.scale, key, value);
      }
    } else {
      float dv[NV][4], dk[NK][4];
      if (live) {
        times_state<T, DK, LDS, PLANE, true, WC, 2>(dv, k, rg * 16, s_grad, wc, key, value);
        times_state<T, DV, LDS, PLANE, false, WC, 3>(dk, v, rg * 16, s_grad, wc, value, key);
        decay_rows(dv, after[i0], after[i0 + 8]);
        decay_rows(dk, after[i0], after[i0 + 8]);
        const float2 end = row_sums<T, LDK, WC>(dk, k, i0, wc);
        if (c == 0) s_end[wc * C + i0] = end.x, s_end[wc * C + i0 + 8] = end.y;
        float col0 = 0.0f, col1 = 0.0f;  // sums of W over i, of j = i0 and i0 + 8
#pragma unroll 1
        for (int n = rg; n < RG; ++n) {
          float a[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
          float d[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
          products<T, DK>(a, k, rg * 16, q, n * 16, key);
          products<T, DV>(d, v, rg * 16, dy, n * 16, value);
          float w[8], x[8], z[8];
          weights_by_column(w, sums, tail, i0, n * 16, rg * 16, n == rg, p.scale);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = a[e >> 2][e & 3] * w[e];
            z[e] = d[e >> 2][e & 3] * w[e];
          }
          if (wc == 0) {
            const bool same = n == rg;  // (W has no diagonal)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int i = n * 16 + half * 8 + 2 * c;
              const float u0 = same && i == i0 ? 0.0f : x[4 * half] * d[half][0];
              const float u1 = same && i + 1 == i0 ? 0.0f : x[4 * half + 1] * d[half][1];
              const float u2 = same && i == i0 + 8 ? 0.0f : x[4 * half + 2] * d[half][2];
              const float u3 = same && i + 1 == i0 + 8 ? 0.0f : x[4 * half + 3] * d[half][3];
              col0 += u0 + u1, col1 += u2 + u3;
              float r0 = u0 + u2, r1 = u1 + u3;
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) {
                r0 += __shfl_xor_sync(0xffffffffu, r0, off);
                r1 += __shfl_xor_sync(0xffffffffu, r1, off);
              }
              if (g == 0) *reinterpret_cast<float2*>(s_row + rg * C + i) = make_float2(r0, r1);
            }
          }
          Made<T> left;
          make(left, x);
          add_product<T, LDV, WC>(dv, left, dy, n * 16, wc, value);
          make(left, z);
          add_product<T, LDK, WC>(dk, left, q, n * 16, wc, key);
        }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
          col0 += __shfl_xor_sync(0xffffffffu, col0, off);
          col1 += __shfl_xor_sync(0xffffffffu, col1, off);
        }
        if (c == 0 && wc == 0) s_col[i0] = col0, s_col[i0 + 8] = col1;
      } else {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) dv[n][e] = 0.0f;
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) dk[n][e] = 0.0f;
      }
      store_rows<T, WC>(p.dv, p, row, s0 + i0, p.value, wc * 16 + 2 * c, dv);
      store_rows<T, WC>(p.dk, p, row, s0 + i0, p.key, wc * 16 + 2 * c, dk);
    }
    __syncthreads();  // the chunk's tiles, states and sums are read or written
    if (chunk > c0) load(chunk - 1), split(chunk - 1);
    if (by_rows && live) S.template publish<3>(s_grad, key, value);
    if (warp == WARPS - 1) {
      // the decays' gradients: prefix sums over the chunk's steps in 64 bits
      constexpr int E = C / 32;
      double back = 0.0, ahead = 0.0, own_back[E], own_ahead[E], through = 0.0;
      if (live) {
#pragma unroll
        for (int w = 0; w < SIDE; ++w) through += s_all[w];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int t = lane * E + e;
        own_back[e] = back, own_ahead[e] = ahead;  // of the steps before this one
        if (live) {
          float rows = 0.0f;
#pragma unroll
          for (int r = 0; r < RG; ++r)
            if (r <= t / 16) rows += s_row[r * C + t];
          back += (double)s_col[t] - (double)rows;
#pragma unroll
          for (int w = 0; w < WC; ++w) back += s_end[w * C + t], ahead += s_far[w * C + t];
        }
      }
      double up_back = back, up_ahead = ahead;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, up_back, off), y = __shfl_up_sync(0xffffffffu, up_ahead, off);
        if (lane >= off) up_back += x, up_ahead += y;
      }
      const double all_ahead = __shfl_sync(0xffffffffu, up_ahead, 31);
      double sum = 0.0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t s = s0 + lane * E + e;
        const double x = (up_back - back + own_back[e]) + (all_ahead - (up_ahead - ahead + own_ahead[e])) + through;
        const bool cut = !(now.g[e] * kLog2e >= kCut) && now.g[e] == now.g[e];
        const double out = s < row.n && !cut ? x : 0.0;
        sum += out;
        if (p.ddecay && s < row.steps) p.ddecay[(row.b * row.steps + row.time(s)) * p.heads + row.h] = (float)out;
      }
      if (p.chunk_ddecay) {
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane == 0) p.chunk_ddecay[index * p.chunks + chunk] = sum;
      }
      if (chunk > c0) store(chunk - 1);
    }
  }
  if (by_rows && p.dstate && part == 0) S.write(p.dstate + index * p.key * p.value, p.key, p.value, 0);
}

// ---------------------------------------------------------------------------------------- single steps

// Few steps, one after the other, with the state in registers: a CTA takes a row's columns by 32, a thread four
// adjacent columns of every 16th row.
constexpr int kStepColumns = 32;
template <class T, int DK>
__global__ void __launch_bounds__(128) steps_kernel(const __grid_constant__ Args p) {
  constexpr int kGroups = 16, kEach = DK / kGroups;
  __shared__ float s_part[2][4][kStepColumns];
  const int blocks = (p.value + kStepColumns - 1) / kStepColumns;
  const int64_t index = blockIdx.x / blocks;
  const int first = (int)(blockIdx.x - index * blocks) * kStepColumns;
  const Row row(p, index);
  const int group = threadIdx.x / 8, col = first + threadIdx.x % 8 * 4, warp = threadIdx.x >> 5;
  const bool whole = p.value % 4 == 0;
  const int64_t state = index * p.key * p.value;
  float S[kEach][4];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int r = e * kGroups + group;
#pragma unroll
    for (int j = 0; j < 4; ++j) S[e][j] = 0.0f;
    if (p.state && r < p.key && col < p.value) {
      const float* at = p.state + state + (int64_t)r * p.value + col;
      if (whole && reinterpret_cast<uintptr_t>(p.state) % 16 == 0) {
        const float4 f = *reinterpret_cast<const float4*>(at);
        S[e][0] = f.x, S[e][1] = f.y, S[e][2] = f.z, S[e][3] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < p.value) S[e][j] = at[j];
      }
    }
  }
  const T *q = static_cast<const T*>(p.q.p), *k = static_cast<const T*>(p.k.p), *v = static_cast<const T*>(p.v.p);
  for (int64_t s = 0; s < row.steps; ++s) {
    const int64_t t = row.time(s);
    const bool live = s < row.n;
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
      float x[4], kk[kEach], qq[kEach];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = col + j < p.value ? widen(v[row.b * p.v.sb + t * p.v.st + row.h * p.v.sh + col + j]) : 0.0f;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int r = e * kGroups + group;
        kk[e] = r < p.key ? widen(k[row.b * p.k.sb + t * p.k.st + row.h * p.k.sh + r]) : 0.0f;
        qq[e] = r < p.key ? widen(q[row.b * p.q.sb + t * p.q.st + row.h * p.q.sh + r]) : 0.0f;
      }
      float g = p.decay[row.b * p.decay_sb + t * p.decay_st + row.h * p.decay_sh];
      if (p.reset && p.reset[row.b * p.reset_sb + t * p.reset_st]) g = -INFINITY;
      const float a = g * kLog2e < kCut ? 0.0f : expf(g);
#pragma unroll
      for (int e = 0; e < kEach; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          S[e][j] = fmaf(kk[e], x[j], decayed(a, S[e][j]));
          y[j] = fmaf(qq[e], S[e][j], y[j]);
        }
    }
    // over the groups: those of a warp by shuffles, the warps through shared memory (two buffers in turn)
#pragma unroll
    for (int off = 8; off < 32; off <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] += __shfl_xor_sync(0xffffffffu, y[j], off);
    float(*part)[kStepColumns] = s_part[s & 1];
    if ((threadIdx.x & 31) < 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) part[warp][threadIdx.x % 8 * 4 + j] = y[j];
    }
    __syncthreads();
    if (threadIdx.x < kStepColumns && first + threadIdx.x < p.value) {
      const float sum = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
      static_cast<T*>(p.y)[((row.b * row.steps + t) * p.heads + row.h) * p.value + first + threadIdx.x] =
          narrow<T>(live ? p.scale * sum : 0.0f);
    }
  }
  if (!p.last) return;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int r = e * kGroups + group;
    if (r >= p.key || col >= p.value) continue;
    float* at = p.last + state + (int64_t)r * p.value + col;
    if (whole && reinterpret_cast<uintptr_t>(p.last) % 16 == 0) {
      *reinterpret_cast<float4*>(at) = make_float4(S[e][0], S[e][1], S[e][2], S[e][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.value) at[j] = S[e][j];
    }
  }
}

// -------------------------------------------------------------------------------------------- launches

enum Kind { kForward, kSweep, kSweepBackward, kSteps };

struct Geometry {
  int dk, dv;  // padded; dv of a CTA
  int chunk;
  int64_t blocks;
};

template <class T>
cudaError_t forward_of(const Args& p, const Geometry& g, Kind kind, cudaStream_t s);
template <class T>
cudaError_t backward_of(const Args& p, const Geometry& g, cudaStream_t s);

// Steps of a chunk.  Two tiles of 32-bit queries and values of 128 columns beside two states fill an SM's shared memory
// at 32 steps; everything else has 64.
constexpr int chunk_of(int dtype, int dk, int dv) { return dtype == PESQ_F32 && dk == 128 && dv == 128 ? 32 : 64; }

}  // namespace lattn
}  // namespace pesq
