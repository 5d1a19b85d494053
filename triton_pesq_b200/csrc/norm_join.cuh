// The join of a block's output with the residual stream, and the norm before
// the next block, row by row of [batch, step, channel]:
//
//   n = post * block / rms(block),        rms(v) = sqrt(mean(v^2) + eps)
//   stream' = stream + scale * act(gate) * n
//   normed = pre * stream' / rms(stream')
//
// A team of threads keeps a row in registers, eight channels a thread, so each
// operand is read once and each result written once: the bound is memory.  The
// next row's operands are on their way while a row is worked on.  The forward
// takes two sums over a row, one after the other.  The backward needs, with
// w = scale act n (so that stream' = stream + w) and h = stream' / rms(stream'),
//
//   q = dnormed pre,   dr = dstream' + (q - h mean(q h)) / rms(stream')
//   dblock = (dr scale act post - (block / rms(block)) mean(dr w)) / rms(block)
//   dgate = dr scale n act',   dstream = dr
//
// and mean(dr w) = mean(dstream' w) + (mean(q w) - mean(q h) mean(h w)) / rms(stream'),
// so its five sums are taken together: two rounds of sums again instead of four.
// The vectors' gradients are sums over rows of dnormed h (pre) and of
// u = dr act block / rms(block): dpost = scale sum u, dscale = post sum u.  They stay in
// registers over the rows of a CTA; the CTAs' sums are added up in a fixed order by a
// second kernel.  The gradient of a gate that the steps of a batch item share is summed
// the same way.
//
// A row's sums are two rounds of shuffles, and barriers where a team has several warps, that its
// loads and stores overlap only by the other teams of the SM and by the next row's loads.
// Measured (B200, cold caches, the call's kernels alone; bytes at the measured copy rate):
//                                    forward (bytes alone)     backward
//   64 x 500 x 896 bfloat16          55.3 us (43.9)            106.5 us (70.2)
//   64 x 500 x 385 float32           49.2 (37.7)               82.0 (60.3)
//   100000 x 64 bfloat16             20.5 (9.8)                34.7 (15.7)
//   6 x 1500 x 385, shared gate      18.5 (8.5)                32.8 (12.7)
//   16000 x 1024 bfloat16            34.8 (25.1)               63.5 (40.1)
//   16000 x 1040 bfloat16            53.3 (25.4)               129.1 (40.7)  teams of 256, 130 of them with channels
//   8000 x 2048 bfloat16             36.9 (25.1)               77.9 (40.1)   8 warps an SM
//   4000 x 8192 bfloat16             88.0 (50.1)               268.7 (80.2)  sums in shared memory, no next row
//   8 x 500 x 768, float32 stream    14.3 (6.6)                26.7 (10.3)   of which a launch is 6
//   the norm alone, 64 x 500 x 896   34.8 (17.5)               75.8 (26.3)
#pragma once

#include <type_traits>

#include "../../include/pesq_cuda.h"
#include "train.cuh"

namespace pesq {
namespace njoin {

using namespace train;

constexpr int kEach = 8;      // channels of a thread
constexpr int kThreads = 128; // of a CTA, unless a row takes more
// CTAs that an SM holds, which the registers of a thread follow from.  Teams up to 128: 72 in the forward (96
// where every channel is addressed by itself), 168 in the backward, where 16 warps of 128
// registers spill and take 25 % longer than 12 that do not.  Wider teams are a CTA each, as many as those registers
// allow and one at least: in the backward one of 256 threads (194 to 236 registers), of 512 (128) or of 1024 (64, which
// spills).  Nothing was tried to fill the SM better there.
constexpr int ctas(bool backward, bool wide, int team) {
  const int threads = team > kThreads ? team : kThreads, sm = backward ? 384 : wide ? 896 : 640;
  return sm / threads > 0 ? sm / threads : 1;
}

struct Rows {
  const void* p;
  int64_t sb, st;  // strides of batch and step, in elements
};

struct Args {
  Rows stream, block, gate, dstream, dnormed;  // block, gate and either upstream gradient may be null
  const float *post, *pre, *scale;             // scale may be null (ones)
  int64_t batch, steps;
  int width;
  int units, span;  // CTAs of a batch item, rows of a CTA
  int silu;
  float eps;
  void *out_stream, *out_normed;  // forward, dense; the stream may be null
  void *dx, *dblock, *dgate;      // backward, dense; dgate null where it is shared
  float *part_u, *part_pre, *part_gate;  // [batch * units, width]; part_gate null where the gate is not shared
};

// Backward rows of so many threads leave a thread too few registers (128, and 64 with 1024 threads) to hold
// the vectors, the sums and the next row: those come from cache, go to shared memory, and wait
template <int TEAM>
constexpr bool kLeanRow = TEAM >= 512;

// 1 / sqrt(mean), of means below the normal range too (rows of 1e-20, eps = 0)
__device__ __forceinline__ float inverse_root(float mean) {
  float y;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(mean));
  return y;
}

// Sums of K values over a team: by shuffles within a warp, through shared
// memory across warps (two buffers in turn, so that one barrier a round is enough).
template <int K, int TEAM>
__device__ __forceinline__ void team_sum(float (&v)[K], float (*s_sum)[32][8], int& turn) {
#pragma unroll
  for (int off = (TEAM < 32 ? TEAM : 32) / 2; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
  if constexpr (TEAM > 32) {
    constexpr int W = TEAM / 32;
    const int warp = threadIdx.x >> 5, first = warp / W * W;
    float(*s)[8] = s_sum[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) s[warp][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) t += s[first + w][k];
      v[k] = t;
    }
  }
}

// The same of five values.  Across a team of several warps the first four are added
// up by halves: half the lanes go on with two of them, a quarter with one, so that it takes 11
// shuffles instead of 25.
template <int TEAM>
__device__ __forceinline__ void team_sum5(float (&v)[5], float (*s_sum)[32][8], int& turn) {
  if constexpr (TEAM <= 32) {
    team_sum<5, TEAM>(v, s_sum, turn);
  } else {
    constexpr unsigned kAll = 0xffffffffu;
    constexpr int W = TEAM / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = warp / W * W;
    const bool high = lane & 16, odd = lane & 8;
    float k0 = high ? v[2] : v[0], k1 = high ? v[3] : v[1];
    k0 += __shfl_xor_sync(kAll, high ? v[0] : v[2], 16);
    k1 += __shfl_xor_sync(kAll, high ? v[1] : v[3], 16);
    float k = odd ? k1 : k0;
    k += __shfl_xor_sync(kAll, odd ? k0 : k1, 8);
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) k += __shfl_xor_sync(kAll, k, off);
    float last = v[4];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) last += __shfl_xor_sync(kAll, last, off);
    float(*s)[8] = s_sum[turn];
    turn ^= 1;
    if ((lane & 7) == 0) s[warp][lane >> 3] = k;
    if (lane == 0) s[warp][4] = last;
    __syncthreads();
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float t4 = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float4 q = *reinterpret_cast<const float4*>(s[first + w]);
      t.x += q.x, t.y += q.y, t.z += q.z, t.w += q.w;
      t4 += s[first + w][4];
    }
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w, v[4] = t4;
  }
}

// A thread's channels: eight in a row as 16-byte accesses (kWide), or one in
// every TEAM.  Those past the width are zero.  They stay as the words they were
// read as until they are used.
template <class T, int TEAM, bool kWide>
struct Eight {
  static constexpr int kWords = kWide ? kEach * (int)sizeof(T) / 4 : kEach;
  unsigned w[kWords];

  static __device__ __forceinline__ int column(int j) {
    const int t = threadIdx.x % TEAM;
    return kWide ? t * kEach + j : t + j * TEAM;
  }
  __device__ __forceinline__ void load(const void* row, int width, bool take) {
    const T* r = static_cast<const T*>(row);
    if (kWide) {
      take = take && column(0) < width;
      const uint4* q = reinterpret_cast<const uint4*>(r + column(0));
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (take) v = q[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        w[j] = 0u;
        if (take && column(j) < width) {
          if constexpr (sizeof(T) == 4)
            w[j] = reinterpret_cast<const unsigned*>(r)[column(j)];
          else
            w[j] = reinterpret_cast<const unsigned short*>(r)[column(j)];
        }
      }
    }
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else {
      const unsigned v = kWide ? w[j / 2] : w[j], half = kWide && j % 2 ? v >> 16 : v & 0xffffu;
      if constexpr (std::is_same<T, __half>::value) {
        return __half2float(__ushort_as_half((unsigned short)half));
      } else {
        return __uint_as_float(kWide && j % 2 ? v & 0xffff0000u : v << 16);
      }
    }
  }
  // channels j and j + 1 (j even)
  __device__ __forceinline__ Vec<2> two(int j) const { return {{at(j), at(j + 1)}}; }
  __device__ __forceinline__ void set(int j, Vec<2> v) { set(j, v.v[0], v.v[1]); }
  __device__ __forceinline__ void set(int j, float a, float b) {
    if constexpr (sizeof(T) == 4) {
      w[j] = __float_as_uint(a), w[j + 1] = __float_as_uint(b);
    } else {
      unsigned v;
      if constexpr (std::is_same<T, __half>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(b), "f"(a));
      else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(b), "f"(a));
      if (kWide)
        w[j / 2] = v;
      else
        w[j] = v & 0xffffu, w[j + 1] = v >> 16;
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t row, int width) const {
    T* r = static_cast<T*>(base) + row;
    if (kWide) {
      uint4* q = reinterpret_cast<uint4*>(r + column(0));
      if (column(0) < width) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) q[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (column(j) < width) {
          if constexpr (sizeof(T) == 4)
            reinterpret_cast<unsigned*>(r)[column(j)] = w[j];
          else
            reinterpret_cast<unsigned short*>(r)[column(j)] = (unsigned short)w[j];
        }
    }
  }
};

// The gate's activation of eight channels, and its slope
template <bool kSlope, class E>
__device__ __forceinline__ void activate(const E& g, int silu, Vec<2> (&value)[kEach / 2], Vec<2> (&slope)[kEach / 2]) {
  Vec<2> s[kEach / 2];
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i) s[i] = g.two(2 * i) * splat<2>(-kLog2e);
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i) s[i] = {{exp2_approx(s[i].v[0]), exp2_approx(s[i].v[1])}};
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i) s[i] = s[i] + splat<2>(1.0f);
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i) s[i] = {{rcp_approx(s[i].v[0]), rcp_approx(s[i].v[1])}};
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i) {
    value[i] = s[i];
    if (kSlope) slope[i] = fma(s[i], splat<2>(-1.0f), splat<2>(1.0f));  // 1 - s
  }
  if (silu) {  // g s, s (1 + g (1 - s))
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) {
      value[i] = g.two(2 * i) * s[i];
      if (kSlope) slope[i] = s[i] * fma(g.two(2 * i), slope[i], splat<2>(1.0f));
    }
  } else if (kSlope) {  // s, s (1 - s)
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) slope[i] = s[i] * slope[i];
  }
}

// The rows that a team works on in turn: every TEAMS-th of its CTA's
template <int TEAM, int THREADS>
struct Turns {
  static constexpr int kTeams = THREADS / TEAM;
  int64_t b, t;  // the team's first row
  int rows;      // of the CTA
  __device__ __forceinline__ Turns(const Args& p) {
    b = blockIdx.x / p.units;
    const int64_t first = (blockIdx.x - b * p.units) * p.span;
    rows = (int)min((int64_t)p.span, p.steps - first);
    t = first + threadIdx.x / TEAM;
  }
  __device__ __forceinline__ bool on(int k) const { return k * kTeams + (int)threadIdx.x / TEAM < rows; }
  // the first row of a dense result
  __device__ __forceinline__ int64_t dense(const Args& p) const { return (b * p.steps + t) * p.width; }
};
// An operand's rows.  With 16-bit blocks whose channels lie eight by eight the row's address is
// kept and moved on (64 x 500 x 896: forward 58.5 -> 56.4 us, backward 110 -> 105); the others have no registers left for it
// (64 x 500 x 385 float32: backward 81 -> 91 us) and work it out every time.
template <class TB, bool kWide>
constexpr bool kRunning = kWide && sizeof(TB) == 2;
template <class T, bool kRuns, int TEAM, int THREADS>
struct Cursor {
  const char* at;
  __device__ __forceinline__ Cursor(const Rows& r, const Turns<TEAM, THREADS>& of) : at(place(r, of, 0)) {}
  static __device__ __forceinline__ const char* place(const Rows& r, const Turns<TEAM, THREADS>& of, int k) {
    const int64_t row = of.b * r.sb + (of.t + (int64_t)k * of.kTeams) * r.st;
    return static_cast<const char*>(r.p) + row * (int64_t)sizeof(T);
  }
  // the row of turn k, turns one after the other
  __device__ __forceinline__ const char* row(const Rows& r, const Turns<TEAM, THREADS>& of, int k) {
    if (!kRuns) return place(r, of, k);
    const char* now = at;
    at += of.kTeams * r.st * (int64_t)sizeof(T);
    return now;
  }
};

// ------------------------------------------------------------------- forward

template <class TS, class TB, int TEAM, bool kWide>
__global__ void __launch_bounds__(TEAM > kThreads ? TEAM : kThreads, ctas(false, kWide, TEAM)) forward_kernel(const __grid_constant__ Args p) {
  constexpr int THREADS = TEAM > kThreads ? TEAM : kThreads, TEAMS = THREADS / TEAM;
  using S = Eight<TS, TEAM, kWide>;
  using B = Eight<TB, TEAM, kWide>;
  using F = Eight<float, TEAM, kWide>;
  __shared__ __align__(16) float s_sum[2][32][8];
  int turn = 0;
  F post, pre, scale;
  pre.load(p.pre, p.width, true);
  post.load(p.post, p.width, p.post != nullptr);
  scale.load(p.scale, p.width, p.scale != nullptr);
  if (p.scale) {
#pragma unroll
    for (int j = 0; j < kEach; j += 2) post.set(j, post.at(j) * scale.at(j), post.at(j + 1) * scale.at(j + 1));
  }
  const int turns = (p.span + TEAMS - 1) / TEAMS;
  const float inv = 1.0f / (float)p.width;
  S x;
  B z, g;
  const Turns<TEAM, THREADS> turn_of(p);
  Cursor<TS, kRunning<TB, kWide>, TEAM, THREADS> at_x(p.stream, turn_of);
  Cursor<TB, kRunning<TB, kWide>, TEAM, THREADS> at_z(p.block, turn_of), at_g(p.gate, turn_of);
  const auto load = [&](int k, bool on, S& x, B& z, B& g) {
    x.load(at_x.row(p.stream, turn_of, k), p.width, on);
    z.load(at_z.row(p.block, turn_of, k), p.width, on && p.block.p);
    g.load(at_g.row(p.gate, turn_of, k), p.width, on && p.gate.p);
  };
  int64_t to = turn_of.dense(p);
  bool on = turn_of.on(0);
  load(0, on, x, z, g);
#pragma unroll 1
  for (int k = 0; k < turns; ++k) {
    const bool on1 = turn_of.on(k + 1);
    S x1;
    B z1, g1;
    load(k + 1, on1, x1, z1, g1);

    constexpr int H = kEach / 2;
    Vec<2> r[H], total = splat<2>(0.0f);
    float sum[1];
    if (p.block.p) {
#pragma unroll
      for (int i = 0; i < H; ++i) total = fma(z.two(2 * i), z.two(2 * i), total);
      sum[0] = total.v[0] + total.v[1];
      team_sum<1, TEAM>(sum, s_sum, turn);
      const Vec<2> rz = splat<2>(inverse_root(fmaf(sum[0], inv, p.eps)));
      Vec<2> w[H];
#pragma unroll
      for (int i = 0; i < H; ++i) w[i] = z.two(2 * i) * (rz * post.two(2 * i));
      if (p.gate.p) {
        Vec<2> value[H], slope[H];
        activate<false>(g, p.silu, value, slope);
#pragma unroll
        for (int i = 0; i < H; ++i) w[i] = w[i] * value[i];
      }
#pragma unroll
      for (int i = 0; i < H; ++i) r[i] = x.two(2 * i) + w[i];
    } else {
#pragma unroll
      for (int i = 0; i < H; ++i) r[i] = x.two(2 * i);
    }
    total = splat<2>(0.0f);
#pragma unroll
    for (int i = 0; i < H; ++i) total = fma(r[i], r[i], total);
    sum[0] = total.v[0] + total.v[1];
    team_sum<1, TEAM>(sum, s_sum, turn);
    const Vec<2> rr = splat<2>(inverse_root(fmaf(sum[0], inv, p.eps)));
    if (on) {
      S out;
      B y;
#pragma unroll
      for (int i = 0; i < H; ++i) out.set(2 * i, r[i]), y.set(2 * i, r[i] * (rr * pre.two(2 * i)));
      if (p.out_stream) out.store(p.out_stream, to, p.width);
      y.store(p.out_normed, to, p.width);
    }
    x = x1, z = z1, g = g1, on = on1;
    to += (int64_t)TEAMS * p.width;
  }
}

// ------------------------------------------------------------------ backward

// The CTA's sum of what its teams hold, to a row of `part`
template <int TEAM, int TEAMS, bool kWide>
__device__ __forceinline__ void store_part(const Vec<2> (&v)[kEach / 2], float* part, int width, float* s_part) {
  using F = Eight<float, TEAM, kWide>;
  F f;
#pragma unroll
  for (int i = 0; i < kEach / 2; ++i) f.set(2 * i, v[i]);
  if (TEAMS == 1) {
    f.store(part, (int64_t)blockIdx.x * width, width);
    return;
  }
  const int team = threadIdx.x / TEAM;
  f.store(s_part, (int64_t)team * kEach * TEAM, kEach * TEAM);
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += TEAM * TEAMS) {
    float t = 0.0f;
#pragma unroll 8
    for (int w = 0; w < TEAMS; ++w) t += s_part[w * kEach * TEAM + c];
    part[(int64_t)blockIdx.x * width + c] = t;
  }
  __syncthreads();
}

template <class TS, class TB, int TEAM, bool kWide>
__global__ void __launch_bounds__(TEAM > kThreads ? TEAM : kThreads, ctas(true, kWide, TEAM)) backward_kernel(const __grid_constant__ Args p) {
  constexpr int THREADS = TEAM > kThreads ? TEAM : kThreads, TEAMS = THREADS / TEAM;
  constexpr bool kLean = kLeanRow<TEAM>;
  using S = Eight<TS, TEAM, kWide>;
  using B = Eight<TB, TEAM, kWide>;
  using F = Eight<float, TEAM, kWide>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ __align__(16) float s_sum[2][32][8];
  __shared__ __align__(16) float s_part[TEAMS > 1 ? THREADS * kEach : 4];
  int turn = 0;
  F post, pre;  // post times scale
  const auto vectors = [&] {
    pre.load(p.pre, p.width, true);
    post.load(p.post, p.width, p.post != nullptr);
    if (p.scale) {
      F scale;
      scale.load(p.scale, p.width, true);
#pragma unroll
      for (int j = 0; j < kEach; j += 2) post.set(j, post.at(j) * scale.at(j), post.at(j + 1) * scale.at(j + 1));
    }
  };
  if (!kLean) vectors();
  constexpr int H = kEach / 2;
  Vec<2> acc_u[H], acc_pre[H], acc_gate[H];
#pragma unroll
  for (int i = 0; i < H; ++i) acc_u[i] = acc_pre[i] = acc_gate[i] = splat<2>(0.0f);
  // (rows of 512 and more threads: sums in shared memory, [3][i][thread])
  extern __shared__ __align__(16) char dynamic[];
  Vec<2>* own = reinterpret_cast<Vec<2>*>(dynamic) + threadIdx.x;
  if (kLean) {
#pragma unroll
    for (int i = 0; i < 3 * H; ++i) own[i * THREADS] = splat<2>(0.0f);
  }
  const int turns = (p.span + TEAMS - 1) / TEAMS;
  const float inv = 1.0f / (float)p.width;
  S x, ds;
  B z, g, dy;
  const Turns<TEAM, THREADS> turn_of(p);
  Cursor<TS, kRunning<TB, kWide>, TEAM, THREADS> at_x(p.stream, turn_of), at_ds(p.dstream, turn_of);
  Cursor<TB, kRunning<TB, kWide>, TEAM, THREADS> at_z(p.block, turn_of), at_g(p.gate, turn_of),
      at_dy(p.dnormed, turn_of);
  const auto load = [&](int k, bool on, S& x, S& ds, B& z, B& g, B& dy) {
    z.load(at_z.row(p.block, turn_of, k), p.width, on && p.block.p);
    g.load(at_g.row(p.gate, turn_of, k), p.width, on && p.gate.p);
    x.load(at_x.row(p.stream, turn_of, k), p.width, on);
    dy.load(at_dy.row(p.dnormed, turn_of, k), p.width, on && p.dnormed.p);
    ds.load(at_ds.row(p.dstream, turn_of, k), p.width, on && p.dstream.p);
  };
  int64_t to = turn_of.dense(p);
  bool on = turn_of.on(0);
  if (!kLean) load(0, on, x, ds, z, g, dy);
#pragma unroll 1
  for (int k = 0; k < turns; ++k) {
    const bool on1 = turn_of.on(k + 1);
    S x1, ds1;
    B z1, g1, dy1;
    if (kLean) {
      load(k, on, x, ds, z, g, dy);
      vectors();
    } else {
      load(k + 1, on1, x1, ds1, z1, g1, dy1);
    }

    float rz = 0.0f;
    if (p.block.p) {
      Vec<2> total = splat<2>(0.0f);
#pragma unroll
      for (int i = 0; i < H; ++i) total = fma(z.two(2 * i), z.two(2 * i), total);
      float one[1] = {total.v[0] + total.v[1]};
      team_sum<1, TEAM>(one, s_sum, turn);
      rz = on ? inverse_root(fmaf(one[0], inv, p.eps)) : 0.0f;
    }
    // sums of r^2, q r, ds w, q w, r w
    Vec<2> value[H], slope[H], w[H], part[5];
#pragma unroll
    for (int k5 = 0; k5 < 5; ++k5) part[k5] = splat<2>(0.0f);
    if (p.gate.p) {
      activate<true>(g, p.silu, value, slope);
    } else {
#pragma unroll
      for (int i = 0; i < H; ++i) value[i] = splat<2>(1.0f), slope[i] = splat<2>(0.0f);
    }
#pragma unroll
    for (int i = 0; i < H; ++i) {
      w[i] = z.two(2 * i) * (splat<2>(rz) * (post.two(2 * i) * value[i]));
      const Vec<2> r = x.two(2 * i) + w[i], q = dy.two(2 * i) * pre.two(2 * i);
      part[0] = fma(r, r, part[0]);
      part[1] = fma(q, r, part[1]);
      part[2] = fma(ds.two(2 * i), w[i], part[2]);
      part[3] = fma(q, w[i], part[3]);
      part[4] = fma(r, w[i], part[4]);
    }
    float sum[5];
#pragma unroll
    for (int k5 = 0; k5 < 5; ++k5) sum[k5] = part[k5].v[0] + part[k5].v[1];
    team_sum5<TEAM>(sum, s_sum, turn);
    // (a row that is off is zeros, and adds zeros for any eps)
    const float rr = on ? inverse_root(fmaf(sum[0], inv, p.eps)) : 0.0f;
    const float mq = sum[1] * inv * rr * rr;                        // mean(q h) / rms
    const float mw = (sum[2] + rr * (sum[3] - mq * sum[4])) * inv;  // mean(dr w)
    Vec<2> dx[H], dz[H], dg[H];
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const Vec<2> r = x.two(2 * i) + w[i], zh = z.two(2 * i) * splat<2>(rz), ps = post.two(2 * i);
      const Vec<2> q = dy.two(2 * i) * pre.two(2 * i);
      dx[i] = fma(splat<2>(rr), fma(r, splat<2>(-mq), q), ds.two(2 * i));
      const Vec<2> u = dx[i] * zh;
      dg[i] = u * (ps * slope[i]);
      dz[i] = splat<2>(rz) * fma(dx[i], ps * value[i], zh * splat<2>(-mw));
      if (kLean) {
        own[i * THREADS] = fma(u, value[i], own[i * THREADS]);
        own[(H + i) * THREADS] = fma(dy.two(2 * i), r * splat<2>(rr), own[(H + i) * THREADS]);
        if (p.part_gate) own[(2 * H + i) * THREADS] = own[(2 * H + i) * THREADS] + dg[i];
      } else {
        acc_u[i] = fma(u, value[i], acc_u[i]);
        acc_pre[i] = fma(dy.two(2 * i), r * splat<2>(rr), acc_pre[i]);
        acc_gate[i] = acc_gate[i] + dg[i];
      }
    }
    if (on) {
      S a;
      B b;
#pragma unroll
      for (int i = 0; i < H; ++i) a.set(2 * i, dx[i]);
      a.store(p.dx, to, p.width);
      if (p.dblock) {
#pragma unroll
        for (int i = 0; i < H; ++i) b.set(2 * i, dz[i]);
        b.store(p.dblock, to, p.width);
      }
      if (p.dgate) {
#pragma unroll
        for (int i = 0; i < H; ++i) b.set(2 * i, dg[i]);
        b.store(p.dgate, to, p.width);
      }
    }
    if (!kLean) x = x1, ds = ds1, z = z1, g = g1, dy = dy1;
    on = on1;
    to += (int64_t)TEAMS * p.width;
  }
  if (kLean) {
#pragma unroll
    for (int i = 0; i < H; ++i)
      acc_u[i] = own[i * THREADS], acc_pre[i] = own[(H + i) * THREADS], acc_gate[i] = own[(2 * H + i) * THREADS];
  }
  if (p.part_u) store_part<TEAM, TEAMS, kWide>(acc_u, p.part_u, p.width, s_part);
  store_part<TEAM, TEAMS, kWide>(acc_pre, p.part_pre, p.width, s_part);
  if (p.part_gate) store_part<TEAM, TEAMS, kWide>(acc_gate, p.part_gate, p.width, s_part);
}

struct Geometry {
  int team;
  bool wide;
  int64_t blocks;
};

template <class TS, class TB>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, cudaStream_t s);

}  // namespace njoin
}  // namespace pesq
