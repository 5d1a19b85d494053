// Element access and small device helpers of the training operators
// (gated_scan, norm_join, adamw): 16- and 32-bit streams read as they are and
// computed on in float.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace pesq {
namespace train {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half_rn(v);
}

// N consecutive elements, moved as one access of N * sizeof(T) bytes (at most 16)
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// and min
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// N floats worked on together; pairs go through the two-wide float instructions
// (half the issue slots of the scalar ones)
template <int N>
struct Vec {
  float v[N];
};
template <int N>
__device__ __forceinline__ Vec<N> splat(float x) {
  Vec<N> r;
#pragma unroll
  for (int j = 0; j < N; ++j) r.v[j] = x;
  return r;
}
__device__ __forceinline__ unsigned long long bits(Vec<2> a) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.v[0]), "f"(a.v[1]));
  return r;
}
__device__ __forceinline__ Vec<2> pair(unsigned long long a) {
  Vec<2> r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.v[0]), "=f"(r.v[1]) : "l"(a));
  return r;
}
__device__ __forceinline__ Vec<2> fma(Vec<2> a, Vec<2> b, Vec<2> c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return pair(r);
}
__device__ __forceinline__ Vec<2> operator*(Vec<2> a, Vec<2> b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ Vec<2> operator+(Vec<2> a, Vec<2> b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ Vec<1> fma(Vec<1> a, Vec<1> b, Vec<1> c) { return {{fmaf(a.v[0], b.v[0], c.v[0])}}; }
__device__ __forceinline__ Vec<1> operator*(Vec<1> a, Vec<1> b) { return {{a.v[0] * b.v[0]}}; }
__device__ __forceinline__ Vec<1> operator+(Vec<1> a, Vec<1> b) { return {{a.v[0] + b.v[0]}}; }

// elements N j .. N j + N - 1 of a pack, in float
template <int N, class T, int M>
__device__ __forceinline__ Vec<N> widen(const Pack<T, M>& p, int j) {
  Vec<N> r;
#pragma unroll
  for (int n = 0; n < N; ++n) r.v[n] = widen(p.v[N * j + n]);
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace train

int set_error(int code, const char* msg);
}  // namespace pesq
