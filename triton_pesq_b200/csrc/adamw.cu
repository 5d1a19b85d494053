// AdamW over many tensors in one launch, moments in 32 or in 8 bits.
//
// With g the gradient (times grad_scale), t the step:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Every value is read and written once: the bound is memory (28 bytes a value
// with 32-bit moments and gradients, 18 with 8-bit moments, a 16-bit gradient and
// a 16-bit copy).  All tensors go in one launch: their addresses and sizes travel as
// kernel parameters, so nothing of them is kept or copied beforehand.  The moments
// of all tensors lie in one buffer each, a tensor's part beginning at a multiple of
// 256 values, so that the blocks of 256 of the buffer are the units of work, and one warp
// takes a unit: eight values a lane.  A warp finds its tensor by bisection.
// Measured (B200, share of the bytes at the measured copy rate): 35M values, 32-bit moments and
// gradients 157 us, 96 %; 106M values, 8-bit moments, 16-bit gradients and copies 329 us, 79 %, where
// the arithmetic of the 8 bits (70 % of the issue slots) is as long as the bytes; 275,000 values in 52 tensors 7 us.
//
// 8 bits.  A block of 256 has a 32-bit scale, its largest magnitude / 448, and its
// values are float8 (e4m3) in units of it.  Nearest rounding holds a value for good that
// moves by less than half a rounding step at a time; such a value is rounded stochastically,
// with bits that are a hash of position, step and seed, so that its mean is right and a
// run can be repeated.
// The first moment moves by (1 - b1) (g - m).  Without a gradient that is more than half a step (1/16
// of the value) where b1 <= 15/16 and the value is above 2^-6 units; there it is rounded to nearest,
// and a gradient that stays the same is met to half a step / (1 - b1), 5/8 of the value for b1 = 0.9.
// Below 2^-6 units the steps are 2^-9 throughout (codes of 1 to 4 steps times 0.9 round back
// to themselves, and the parameter would move on without a gradient), and with a larger b1 nothing
// need move that far: there a value that moves by less than half a step is rounded stochastically.
// The second moment is kept as its root, which halves the range that 8 bits have to
// span (2^-9 .. 448 of the root are 10 decades of the moment), and moves by less
// than 1 / 2000 of itself a step: it is always rounded stochastically.
// A root that is not zero is never rounded to zero: the update would divide by
// the gradient's own share alone and be too large by up to 1 / sqrt(1 - b2).  The hash
// is the multiply-xorshift finaliser "lowbias32" (C. Wellons, "Prospecting for Hash
// Functions", 2018).
//
// The step count lives on the device, so that a captured step counts on: [0]
// counts the steps, [1] the launch's blocks that are done; the last one adds to
// [0] and clears [1].  A grad_scale that is not finite skips the step whole.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "../../include/pesq_cuda.h"
#include "train.cuh"

namespace {

using namespace pesq::train;
using pesq::set_error;

constexpr int kBlock = 256;   // values of a unit, and of a scale
constexpr int kThreads = 256; // of a CTA
constexpr float kTop = 448.0f;

struct Entry {
  float* param;
  const void* grad;
  void* copy;
  int64_t n;      // values
  int64_t first;  // first unit
};

// Tensors of a launch.  Kernel parameters hold 32,764 bytes; a launch of few tensors
// takes the short table.
template <int N>
struct Table {
  Entry e[N];
};
constexpr int kShort = 96, kLong = 800;

struct Args {
  int count;
  int64_t units, first;  // of this launch, and before it
  void *moment1, *moment2;
  float *scale1, *scale2;  // of the units (8 bits)
  long long* step;
  const float* grad_scale;
  double log_beta1, log_beta2;
  float beta1, beta2, rest1, rest2;  // betas, and 1 less them
  float lr, eps, decay;
  float held1;           // units below which nearest rounding may hold the first moment
  unsigned seed;
  int last;              // of the call's launches
};

__device__ __forceinline__ unsigned hash(unsigned h) {
  h = (h ^ (h >> 16)) * 0x7feb352du;
  h = (h ^ (h >> 15)) * 0x846ca68bu;
  return h ^ (h >> 16);
}

__device__ __forceinline__ void from_e4m3(unsigned w, float* v) {  // four values
  unsigned lo, hi;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
__device__ __forceinline__ unsigned to_e4m3(const float* v) {  // nearest
  unsigned w;
  asm("{\n.reg .b16 l, h;\ncvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\nmov.b32 %0, {l, h};\n}"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
  return w;
}

// u to one of its two neighbours in e4m3, the upper with the probability of its
// nearness: 20 random bits are added below the 3 mantissa bits that stay.  From 2^-6 on
__device__ __forceinline__ float dither(float u, unsigned bits) {
  return __uint_as_float((__float_as_uint(u) + (bits & 0xfffffu)) & ~0xfffffu);
}
// below, where the steps are 2^-9 throughout
__device__ __forceinline__ float dither_small(float u, unsigned bits) {
  return floorf(fmaf((float)(bits & 0xfffffu), 0x1p-20f, u * 512.0f)) * 0x1p-9f;
}
// The first moment, in units, that was `was` in the same units: left to nearest rounding
// where it has moved by half a step or more.  The twelve upper bits of a hash; the root takes the others.
__device__ __forceinline__ float dither_held(float m, float was, unsigned bits) {
  const float u = fabsf(m), power = __uint_as_float(__float_as_uint(u) & 0x7f800000u);
  const unsigned mine = bits >> 20 << 8 | 0x80u;
  float to = dither(u, mine);
  if (u < 0x1p-6f) to = dither_small(u, mine);
  return fabsf(m - was) < 0x1p-4f * fmaxf(power, 0x1p-6f) ? copysignf(to, m) : m;
}

// Eight values of a tensor, as the words they were read as
template <class T>
struct Eight {
  unsigned w[2 * sizeof(T)];
  // from `at` on of n, as 16-byte accesses where `wide`
  __device__ __forceinline__ void read(const T* p, int64_t at, int64_t n, bool wide) {
    if (wide) {
      const uint4* q = reinterpret_cast<const uint4*>(p + at);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint4 v = q[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = at + j < n ? widen(p[at + j]) : 0.0f;
      set(v);
    }
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[j]);
    else if constexpr (std::is_same<T, __half>::value)
      return __half2float(__ushort_as_half((unsigned short)(j % 2 ? w[j / 2] >> 16 : w[j / 2])));
    else
      return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if constexpr (sizeof(T) == 4)
        w[j] = __float_as_uint(v[j]), w[j + 1] = __float_as_uint(v[j + 1]);
      else if constexpr (std::is_same<T, __half>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[j / 2]) : "f"(v[j + 1]), "f"(v[j]));
      else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j / 2]) : "f"(v[j + 1]), "f"(v[j]));
    }
  }
  __device__ __forceinline__ void write(T* p, int64_t at, int64_t n, bool wide) const {
    if (wide) {
      uint4* q = reinterpret_cast<uint4*>(p + at);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        q[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j < n) p[at + j] = narrow<T>(this->at(j));
    }
  }
};

__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));  // (small gradients' squares lie below the normal range)
  return r;
}

// The warp's largest of values >= 0, whose bits order as they do; a NaN is the largest
__device__ __forceinline__ float warp_max(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
}

// What a lane has read of a unit
template <class G, bool kEight>
struct Unit {
  int tensor;
  int64_t at;  // in the tensor
  bool wide, wide_g;
  Eight<float> p;
  Eight<G> g;
  Eight<float> m, v;  // 32 bits
  uint2 c1, c2;       // 8 bits
  float s1, s2;
};

// CTAs an SM holds, all of a launch: the registers of a thread, and how many rows of DRAM are open
template <bool kEight>
constexpr int kCtas = kEight ? 3 : 2;  // (32 bits, 35M values: 1 takes 190 us, 2 162, 3 178, 4 193)

// The CTAs take eight units at a time in turn, a warp one of them; the next unit's
// values are on their way while one is worked on.
template <class G, bool kEight, int N>
__global__ void __launch_bounds__(kThreads, kCtas<kEight>) adamw_kernel(const __grid_constant__ Args p,
                                                                        const __grid_constant__ Table<N> t) {
  __shared__ float s_c[3];  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), grad scale
  __shared__ unsigned s_step;
  const int lane = threadIdx.x & 31;
  constexpr int kWarps = kThreads / 32;
  const int64_t end = p.units, turn = (int64_t)gridDim.x * kWarps;
  int64_t unit = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;

  int lo = 0, hi = p.count;  // the last tensor that begins at or before the unit
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.e[mid].first <= unit) lo = mid;
    else hi = mid;
  }
  const auto read = [&](int64_t unit, Unit<G, kEight>& u) {
    while (lo + 1 < p.count && t.e[lo + 1].first <= unit) ++lo;
    const Entry& e = t.e[lo];
    u.tensor = lo;
    u.at = (unit - e.first) * kBlock + lane * 8;
    if (!e.grad) return;
    const bool whole = u.at + 8 <= e.n;
    u.wide = whole && reinterpret_cast<uintptr_t>(e.param) % 16 == 0;
    u.wide_g = whole && reinterpret_cast<uintptr_t>(e.grad) % 16 == 0;
    u.g.read(static_cast<const G*>(e.grad), u.at, e.n, u.wide_g);
    u.p.read(e.param, u.at, e.n, u.wide);
    const int64_t place = (p.first + unit) * kBlock + lane * 8;  // in the moments' buffers
    if (kEight) {
      u.c1 = *reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(p.moment1) + place);
      u.c2 = *reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(p.moment2) + place);
      u.s1 = p.scale1[p.first + unit], u.s2 = p.scale2[p.first + unit];
    } else {
      u.m.read(static_cast<const float*>(p.moment1), place, 0, true);
      u.v.read(static_cast<const float*>(p.moment2), place, 0, true);
    }
  };
  Unit<G, kEight> now;
  if (unit < end) read(unit, now);

  if (threadIdx.x < 32) {
    const long long step = *reinterpret_cast<volatile long long*>(p.step) + 1;
    // 1 - b^t = -expm1(t log b): the product in 64 bits, the rest is accurate in 32
    if (threadIdx.x == 0) s_c[0] = -p.lr / expm1f((float)((double)step * p.log_beta1)), s_step = (unsigned)step;
    if (threadIdx.x == 1) s_c[1] = 1.0f / sqrtf(-expm1f((float)((double)step * p.log_beta2)));
    if (threadIdx.x == 2) s_c[2] = p.grad_scale ? *p.grad_scale : 1.0f;
  }
  __syncthreads();
  const float scale = s_c[2];
  const bool skip = !isfinite(scale);
  const float rate = s_c[0], root = s_c[1], keep = 1.0f - p.lr * p.decay;
  const Vec<2> b1 = splat<2>(p.beta1), b2 = splat<2>(p.beta2), a1 = splat<2>(p.rest1);
  const Vec<2> a2 = splat<2>(p.rest2), sc = splat<2>(scale);
  const unsigned salt = s_step * 0x9e3779b9u + p.seed * 0x85ebca6bu;

  if (skip) unit = end;
  for (; unit < end; unit += turn) {
    Unit<G, kEight> next;
    if (unit + turn < end) read(unit + turn, next);
    const Entry& e = t.e[now.tensor];
    if (e.grad) {
      const int64_t place = (p.first + unit) * kBlock + lane * 8;
      float w[8], m[8], v[8], r[8];
      if (kEight) {
        from_e4m3(now.c1.x, m), from_e4m3(now.c1.y, m + 4), from_e4m3(now.c2.x, v), from_e4m3(now.c2.y, v + 4);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = now.m.at(j), v[j] = now.v.at(j);
      }
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const Vec<2> g{{now.g.at(j), now.g.at(j + 1)}}, gs = g * sc;
        Vec<2> m2{{m[j], m[j + 1]}}, v2{{v[j], v[j + 1]}}, p2{{now.p.at(j), now.p.at(j + 1)}};
        if (kEight) {
          m2 = m2 * splat<2>(now.s1);
          v2 = v2 * splat<2>(now.s2);
          v2 = v2 * v2;
        }
        Vec<2> r2;
        if (kEight) {
          // operation by operation: what is rounded to 8 bits has the bits of the definition in 32,
          // because a value that falls on the other side of a rounding is off by 1/8
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            m2.v[i] = __fadd_rn(__fmul_rn(p.beta1, m2.v[i]), __fmul_rn(p.rest1, gs.v[i]));
            v2.v[i] = __fadd_rn(__fmul_rn(p.beta2, v2.v[i]), __fmul_rn(__fmul_rn(p.rest2, gs.v[i]), gs.v[i]));
            r2.v[i] = __fsqrt_rn(v2.v[i]);
          }
        } else {
          m2 = fma(b1, m2, a1 * gs);
          v2 = fma(b2, v2, a2 * (gs * gs));
          r2 = {{root_of(v2.v[0]), root_of(v2.v[1])}};
        }
        const Vec<2> below = fma(r2, splat<2>(root), splat<2>(p.eps));
        const Vec<2> update = m2 * Vec<2>{{rcp_approx(below.v[0]), rcp_approx(below.v[1])}};
        p2 = fma(p2, splat<2>(keep), update * splat<2>(-rate));
        m[j] = m2.v[0], m[j + 1] = m2.v[1], v[j] = v2.v[0], v[j + 1] = v2.v[1];
        r[j] = r2.v[0], r[j + 1] = r2.v[1], w[j] = p2.v[0], w[j + 1] = p2.v[1];
      }
      Eight<float> out;
      out.set(w);
      out.write(e.param, now.at, e.n, now.wide);
      if (e.copy) {
        using C = typename std::conditional<std::is_same<G, __half>::value, __half, __nv_bfloat16>::type;
        Eight<C> c;
        c.set(w);
        c.write(static_cast<C*>(e.copy), now.at, e.n, now.at + 8 <= e.n && reinterpret_cast<uintptr_t>(e.copy) % 16 == 0);
      }
      if (kEight) {
        float top1 = 0.0f, top2 = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top1 = max_nan(top1, fabsf(m[j])), top2 = max_nan(top2, r[j]);
        const float s1 = warp_max(top1) * (1.0f / kTop), s2 = warp_max(top2) * (1.0f / kTop);
        const float i1 = s1 > 1e-36f ? __frcp_rn(s1) : 0.0f, i2 = s2 > 1e-36f ? __frcp_rn(s2) : 0.0f;
        float low1 = kTop, low2 = kTop;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          m[j] *= i1, r[j] *= i2;
          low1 = fminf(low1, fabsf(m[j])), low2 = min_nan(low2, r[j]);
        }
        bool held = low1 < p.held1;
        if (held && low1 == 0.0f) {  // (zeros stay)
          held = false;
#pragma unroll
          for (int j = 0; j < 8; ++j) held = held || (m[j] != 0.0f && fabsf(m[j]) < p.held1);
        }
        if (!held && low2 >= 0x1p-6f) {  // (rarely not with b1 <= 15/16; above, always: 106M values 385 us)
#pragma unroll
          for (int j = 0; j < 8; ++j) r[j] = dither(r[j], hash((unsigned)(place + j) + salt));
        } else {
          // (the codes are still in memory, which costs fewer registers than to keep them)
          const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(p.moment1) + place);
          const float then = now.s1 * i1;
          float was[8];
          from_e4m3(c.x, was), from_e4m3(c.y, was + 4);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const unsigned h = hash((unsigned)(place + j) + salt);
            const float to = dither_held(m[j], was[j] * then, h);
            m[j] = fabsf(m[j]) < p.held1 ? to : m[j];
            // (what is above zero does not become zero, and a NaN stays)
            if (r[j] >= 0x1p-6f)
              r[j] = dither(r[j], h);
            else if (r[j] > 0.0f)
              r[j] = fmaxf(dither_small(r[j], h), 0x1p-9f);
          }
        }
        uint2 c1, c2;
        c1.x = to_e4m3(m), c1.y = to_e4m3(m + 4), c2.x = to_e4m3(r), c2.y = to_e4m3(r + 4);
        *reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.moment1) + place) = c1;
        *reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.moment2) + place) = c2;
        if (lane == 0) p.scale1[p.first + unit] = s1, p.scale2[p.first + unit] = s2;
      } else {
        now.m.set(m), now.v.set(v);
        now.m.write(static_cast<float*>(p.moment1), place, 0, true);
        now.v.write(static_cast<float*>(p.moment2), place, 0, true);
      }
    }
    now = next;
  }

  // the call's last block counts the step: every block has read it by then
  if (p.last) {
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long* done = reinterpret_cast<unsigned long long*>(p.step) + 1;
      __threadfence();
      if (atomicAdd(done, 1ull) == gridDim.x - 1) {
        *done = 0ull;
        if (!skip) p.step[0] += 1;
      }
    }
  }
}

int sms() {
  static int count[64] = {0};  // by device; a property that does not change
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (count[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    count[dev] = n;
  }
  return count[dev];
}

template <class G, bool kEight, int N>
cudaError_t start(const Args& a, const Entry* e, cudaStream_t s) {
  Table<N> t;
  std::memcpy(t.e, e, sizeof(Entry) * a.count);
  // (one block at least: a step without values counts)
  const int64_t blocks = std::max<int64_t>(1, (a.units + kThreads / 32 - 1) / (kThreads / 32));
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, (int64_t)sms() * kCtas<kEight>);
  adamw_kernel<G, kEight, N><<<grid, kThreads, 0, s>>>(a, t);
  return cudaGetLastError();
}
template <class G>
cudaError_t launch(const Args& a, const Entry* e, bool eight, cudaStream_t s) {
  if (a.count <= kShort) return eight ? start<G, true, kShort>(a, e, s) : start<G, false, kShort>(a, e, s);
  return eight ? start<G, true, kLong>(a, e, s) : start<G, false, kLong>(a, e, s);
}

}  // namespace

extern "C" {

int pesq_adamw_step(const pesq_adamw_desc* d, const pesq_adamw_tensor* tensors, int64_t count, void* stream) {
  if (!d || (count > 0 && !tensors) || count < 0) return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL argument");
  if (d->grad_dtype < PESQ_F32 || d->grad_dtype > PESQ_F16)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "unknown gradient type");
  if (d->state_bits != 8 && d->state_bits != 32) return set_error(PESQ_ERR_INVALID_ARGUMENT, "states have 8 or 32 bits");
  if (!d->step ||
      (d->units > 0 && (!d->moment1 || !d->moment2 || (d->state_bits == 8 && (!d->scale1 || !d->scale2)))))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL state");
  if (reinterpret_cast<uintptr_t>(d->moment1) % 16 || reinterpret_cast<uintptr_t>(d->moment2) % 16 ||
      reinterpret_cast<uintptr_t>(d->step) % 8)
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "the moments are 16-byte, the step 8-byte aligned");
  if (!(d->beta1 >= 0.0 && d->beta1 < 1.0 && d->beta2 >= 0.0 && d->beta2 < 1.0))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "betas lie in [0, 1)");
  if (!(d->eps >= 0.0f) || !(d->lr >= 0.0f) || !(d->weight_decay >= 0.0f))
    return set_error(PESQ_ERR_INVALID_ARGUMENT, "lr, eps and weight decay must not be negative");
  int64_t units = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].n < 0 || (tensors[i].n > 0 && tensors[i].grad && !tensors[i].param))
      return set_error(PESQ_ERR_INVALID_ARGUMENT, "NULL tensor");
    if (tensors[i].copy && d->grad_dtype == PESQ_F32)
      return set_error(PESQ_ERR_INVALID_ARGUMENT, "copies are of the gradients' 16-bit type");
    units += (tensors[i].n + kBlock - 1) / kBlock;
  }
  if (units > d->units) return set_error(PESQ_ERR_WORKSPACE, "the moments are shorter than the tensors");
  Args a{};
  a.moment1 = d->moment1;
  a.moment2 = d->moment2;
  a.scale1 = d->scale1;
  a.scale2 = d->scale2;
  a.step = reinterpret_cast<long long*>(d->step);
  a.grad_scale = d->grad_scale;
  a.log_beta1 = std::log(d->beta1);  // (of 0: minus infinity, and 1 - 0^t = 1)
  a.log_beta2 = std::log(d->beta2);
  a.beta1 = (float)d->beta1;
  a.beta2 = (float)d->beta2;
  a.rest1 = (float)(1.0 - d->beta1);
  a.rest2 = (float)(1.0 - d->beta2);
  a.lr = d->lr;
  a.eps = d->eps;
  a.decay = d->weight_decay;
  a.held1 = d->beta1 <= 0.9375 ? 0x1p-6f : INFINITY;
  a.seed = d->seed;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  Entry table[kLong];
  int64_t i = 0, before = 0;
  do {  // (once at least)
    a.count = 0;
    a.units = 0;
    a.first = before;
    for (; i < count && a.count < kLong; ++i) {
      if (tensors[i].n == 0) continue;
      table[a.count++] = {tensors[i].param, tensors[i].grad, tensors[i].copy, tensors[i].n, a.units};
      a.units += (tensors[i].n + kBlock - 1) / kBlock;
    }
    before += a.units;
    a.last = before == units;
    if (a.units == 0) table[0] = {nullptr, nullptr, nullptr, 0, 0}, a.count = 1;
    const bool eight = d->state_bits == 8;
    const cudaError_t e = d->grad_dtype == PESQ_F32    ? launch<float>(a, table, eight, s)
                          : d->grad_dtype == PESQ_BF16 ? launch<__nv_bfloat16>(a, table, eight, s)
                                                       : launch<__half>(a, table, eight, s);
    if (e != cudaSuccess) return set_error(PESQ_ERR_CUDA, cudaGetErrorString(e));
  } while (!a.last);
  return PESQ_OK;
}

}  // extern "C"
