// Layer norm over the last dimension of [batch, step, head, channel], with a weight (and bias) for each
// channel, or for each head and channel:
//
//   y = h weight + bias,   h = (x - mean(x)) / sqrt(mean((x - mean(x))^2) + eps)
//
// A team of threads keeps a row in registers, up to 32 channels a thread in groups of eight: x
// is read once, the mean subtracted before the squares are summed (two rounds of sums), and the next row is on its
// way while one is worked on.  A warp is a team for up to 1024 channels, so that its sums are shuffles without barriers.  The
// backward recomputes the statistics instead of reading them, and takes with q = dy weight the second round's three sums
// together:
//
//   dx = (q - mean(q) - h mean(q h)) / sqrt(..),   dweight = sum over rows of dy h,   dbias = of dy
//
// The vectors' sums stay in registers over the rows of a team, which all belong to one head; a CTA's teams of the
// same head are added up in shared memory, and the CTAs' sums in a fixed order by a second kernel, so that a
// result is the same every time.
//
// The bound is memory; what is in the way of it are rounds of sums and loads that 12 to 45 % of an SM's warps, whose registers hold
// the rows, have to hide, and instructions (16 bits to 32 and back, masks: issue slots 45 to 57 % full).
// Forward and backward on cold caches, with the bytes alone at the copy rate in brackets: 32000 x 896 bfloat16 26 (18) and 40 us
// (27), 32000 x 14 heads of 64 28 (18) and 46 (27), 24006 x 1155 float32 to float16 40 (26) and 60 (43).  More rows on their way
// (two to four) did not help, and took twice as long channel by channel (32000 x 895: 33 and 76 us), whose registers they leave no room for.
#pragma once

#include "norm_join.cuh"

namespace pesq {
namespace lnorm {

using namespace train;
using njoin::Eight;
using njoin::inverse_root;
using njoin::kEach;
using njoin::team_sum;

// Threads of a CTA: four warps, or a row's, where those are more or no divisor
__host__ __device__ constexpr int threads_of(int team) { return team <= 128 && 128 % team == 0 ? 128 : team; }

// An operand's rows: strides of batch, step and head in elements
struct Strided {
  const void* p;
  int64_t sb, st, sh;
};

struct Args {
  Strided x, dy;
  const float *weight, *bias;  // [heads, width]; bias may be null
  int64_t batch, steps;
  int heads, width;
  int block_heads;   // heads of a CTA
  int head_blocks;   // CTAs side by side over the heads
  int64_t units;     // CTAs over the rows, of each of which `span` rows
  int64_t span;
  float eps;
  void* y;           // forward, dense
  void* dx;          // backward, dense
  float *part_weight, *part_bias;  // [units, heads, width]; part_bias null without a bias
};

// CTAs that an SM holds, which the registers of a thread follow from.  (A forward of one group channel by channel needs 72 registers:
// with 64, 200000 x 130 bfloat16 takes 60 us instead of 50)
constexpr int ctas(bool backward, bool wide, int team, int groups) {
  const int threads = threads_of(team);
  const int sm = groups == 4 ? (backward ? 256 : 384) : groups == 2 ? (backward ? 384 : 640) : (backward ? 512 : wide ? 1024 : 896);
  return sm / threads > 0 ? sm / threads : 1;
}

// Eights of channels of a thread at most: channel by channel (kWide false) a backward of four spills
constexpr int most_groups(bool wide) { return wide ? 4 : 2; }

// Whether the next row of a backward comes in while one is worked on: not to 128 registers a thread, where it would be put off
// value by value (8000 x 8001 bfloat16: 433 us, and 203 without)
__host__ __device__ constexpr bool reads_ahead(int team) { return team < 512; }

// A thread's channels of a row: groups of eight, 8 TEAM channels apart
template <class T, int TEAM, int GROUPS, bool kWide>
struct Row {
  using E = Eight<T, TEAM, kWide>;
  static constexpr int kApart = kEach * TEAM, kBytes = sizeof(T);
  E e[GROUPS];
  __device__ __forceinline__ void load(const void* row, int width, bool take) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) e[g].load(static_cast<const T*>(row) + g * kApart, width - g * kApart, take);
  }
  __device__ __forceinline__ void store(void* base, int64_t row, int width) const {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) e[g].store(base, row + g * kApart, width - g * kApart);
  }
  // Channels j and j + 1 (j even) of group g less the mean; those past the width, which are zero, stay so.  Where a group is in the row
  // or out of it as a whole one selection takes the place of eight (a backward of 32000 x 896 bfloat16 42 us, then 40)
  __device__ __forceinline__ Vec<2> less(int g, int j, float mean, int width) const {
    const int left = width - g * kApart;
    if (kWide) return e[g].two(j) + splat<2>(E::column(0) < left ? -mean : 0.0f);
    Vec<2> d;
#pragma unroll
    for (int i = 0; i < 2; ++i) d.v[i] = E::column(j + i) < left ? e[g].at(j + i) - mean : 0.0f;
    return d;
  }
};

// The rows that a team works on in turn: those of one head, every kSlots-th of its CTA's
template <int TEAM, int THREADS>
struct Turns {
  static constexpr int kTeams = THREADS / TEAM;
  int head, slots;     // rows that the CTA's teams of one head take at once
  int64_t row, end;    // of [batch * steps]
  __device__ __forceinline__ Turns(const Args& p) {
    const int team = threadIdx.x / TEAM, block = blockIdx.x % p.head_blocks;
    const int64_t unit = blockIdx.x / p.head_blocks;
    slots = kTeams / p.block_heads;
    head = block * p.block_heads + team % p.block_heads;
    const bool on = team < slots * p.block_heads && head < p.heads;
    row = unit * p.span + team / p.block_heads;
    end = on ? min(p.batch * p.steps, (unit + 1) * p.span) : 0;
    if (!on) head = 0;
  }
};
// Where a team's rows of an operand lie.  Most calls' batch items lie as one run, whose rows are one stride apart: others divide
template <class T>
struct Walk {
  const char* at;
  int64_t step;
  __device__ __forceinline__ Walk(const Strided& r, const Args& p, int64_t row, int head, int slots) {
    step = slots * r.st * (int64_t)sizeof(T);
    at = static_cast<const char*>(r.p) + (row * r.st + head * r.sh) * (int64_t)sizeof(T);
    if (p.batch != 1) place(r, p, row, head);
  }
  __device__ __forceinline__ void place(const Strided& r, const Args& p, int64_t row, int head) {
    const int64_t b = row / p.steps, t = row - b * p.steps;
    at = static_cast<const char*>(r.p) + (b * r.sb + t * r.st + head * r.sh) * (int64_t)sizeof(T);
  }
  // to the team's next row, which is `row`
  __device__ __forceinline__ void next(const Strided& r, const Args& p, int64_t row, int head) {
    at += step;
    if (p.batch != 1) place(r, p, row, head);
  }
};

template <class TX, class TY, int TEAM, int GROUPS, bool kWide>
__global__ void __launch_bounds__(threads_of(TEAM), ctas(false, kWide, TEAM, GROUPS))
    forward_kernel(const __grid_constant__ Args p) {
  constexpr int THREADS = threads_of(TEAM), H = kEach / 2;
  using X = Row<TX, TEAM, GROUPS, kWide>;
  using Y = Row<TY, TEAM, GROUPS, kWide>;
  using F = Row<float, TEAM, GROUPS, kWide>;
  __shared__ __align__(16) float s_sum[2][32][8];
  int turn = 0;
  Turns<TEAM, THREADS> of(p);
  F weight, bias;
  weight.load(p.weight + (int64_t)of.head * p.width, p.width, true);
  bias.load(p.bias + (int64_t)of.head * p.width, p.width, p.bias != nullptr);
  const float inv = 1.0f / (float)p.width;
  const int64_t turns = (p.span + of.slots - 1) / of.slots;
  X x;
  bool on = of.row < of.end;
  Walk<TX> walk(p.x, p, of.row, of.head, of.slots);
  x.load(walk.at, p.width, on);
  char* to = static_cast<char*>(p.y) + (of.row * p.heads + of.head) * p.width * Y::kBytes;
  const int64_t apart = (int64_t)of.slots * p.heads * p.width * Y::kBytes;
#pragma unroll 1
  for (int64_t k = 0; k < turns; ++k) {
    const int64_t next = of.row + of.slots;
    const bool on1 = next < of.end;
    X x1;
    walk.next(p.x, p, next, of.head);
    x1.load(walk.at, p.width, on1);
    Vec<2> d[GROUPS][H], total = splat<2>(0.0f);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < H; ++i) total = total + x.e[g].two(2 * i);
    float sum[1] = {total.v[0] + total.v[1]};
    team_sum<1, TEAM>(sum, s_sum, turn);
    const float mean = sum[0] * inv;
    total = splat<2>(0.0f);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        d[g][i] = x.less(g, 2 * i, mean, p.width);
        total = fma(d[g][i], d[g][i], total);
      }
    sum[0] = total.v[0] + total.v[1];
    team_sum<1, TEAM>(sum, s_sum, turn);
    const Vec<2> r = splat<2>(inverse_root(fmaf(sum[0], inv, p.eps)));
    if (on) {
      Y y;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int i = 0; i < H; ++i) y.e[g].set(2 * i, fma(d[g][i] * r, weight.e[g].two(2 * i), bias.e[g].two(2 * i)));
      y.store(to, 0, p.width);
    }
    x = x1, on = on1, of.row = next, to += apart;
  }
}

// What the CTA's teams of each head hold, added up, to the CTA's row of `part`
template <int TEAM, int GROUPS, int TEAMS, bool kWide>
__device__ __forceinline__ void store_part(const Vec<2> (&v)[GROUPS][kEach / 2], float* part, const Args& p, float* s_part) {
  using F = Row<float, TEAM, GROUPS, kWide>;
  constexpr int kRow = kEach * TEAM * GROUPS;
  F f;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) f.e[g].set(2 * i, v[g][i]);
  const int64_t unit = blockIdx.x / p.head_blocks;
  const int first = blockIdx.x % p.head_blocks * p.block_heads, heads = min(p.block_heads, p.heads - first);
  float* to = part + (unit * p.heads + first) * p.width;
  if (TEAMS == 1) {
    f.store(to, 0, p.width);
    return;
  }
  f.store(s_part, (int64_t)(threadIdx.x / TEAM) * kRow, kRow);
  __syncthreads();
  const int slots = TEAMS / p.block_heads;
  for (int c = threadIdx.x; c < heads * p.width; c += TEAM * TEAMS) {
    const int head = c / p.width, at = c - head * p.width;
    float t = 0.0f;
    for (int w = 0; w < slots; ++w) t += s_part[(w * p.block_heads + head) * kRow + at];
    to[c] = t;
  }
  __syncthreads();
}

template <class TX, class TY, int TEAM, int GROUPS, bool kWide>
__global__ void __launch_bounds__(threads_of(TEAM), ctas(true, kWide, TEAM, GROUPS))
    backward_kernel(const __grid_constant__ Args p) {
  constexpr int THREADS = threads_of(TEAM), TEAMS = THREADS / TEAM, H = kEach / 2;
  constexpr bool kAhead = reads_ahead(TEAM);
  using X = Row<TX, TEAM, GROUPS, kWide>;
  using Y = Row<TY, TEAM, GROUPS, kWide>;
  using F = Row<float, TEAM, GROUPS, kWide>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ __align__(16) float s_sum[2][32][8];
  __shared__ __align__(16) float s_part[TEAMS > 1 ? THREADS * kEach * GROUPS : 4];
  int turn = 0;
  Turns<TEAM, THREADS> of(p);
  F weight;
  weight.load(p.weight + (int64_t)of.head * p.width, p.width, true);
  Vec<2> acc_weight[GROUPS][H], acc_bias[GROUPS][H];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
#pragma unroll
    for (int i = 0; i < H; ++i) acc_weight[g][i] = acc_bias[g][i] = splat<2>(0.0f);
  const float inv = 1.0f / (float)p.width;
  const int64_t turns = (p.span + of.slots - 1) / of.slots;
  X x;
  Y dy;
  bool on = of.row < of.end;
  Walk<TX> walk(p.x, p, of.row, of.head, of.slots);
  Walk<TY> walk_dy(p.dy, p, of.row, of.head, of.slots);
  x.load(walk.at, p.width, on);
  dy.load(walk_dy.at, p.width, on);
  char* to = static_cast<char*>(p.dx) + (of.row * p.heads + of.head) * p.width * X::kBytes;
  const int64_t apart = (int64_t)of.slots * p.heads * p.width * X::kBytes;
#pragma unroll 1
  for (int64_t k = 0; k < turns; ++k) {
    const int64_t next = of.row + of.slots;
    const bool on1 = next < of.end;
    X x1;
    Y dy1;
    walk.next(p.x, p, next, of.head);
    walk_dy.next(p.dy, p, next, of.head);
    if constexpr (kAhead) x1.load(walk.at, p.width, on1), dy1.load(walk_dy.at, p.width, on1);
    Vec<2> d[GROUPS][H], total = splat<2>(0.0f);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < H; ++i) total = total + x.e[g].two(2 * i);
    float sum[1] = {total.v[0] + total.v[1]};
    team_sum<1, TEAM>(sum, s_sum, turn);
    const float mean = sum[0] * inv;
    // sums of d^2, q, q d
    Vec<2> part[3];
#pragma unroll
    for (int k3 = 0; k3 < 3; ++k3) part[k3] = splat<2>(0.0f);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        d[g][i] = x.less(g, 2 * i, mean, p.width);
        const Vec<2> q = dy.e[g].two(2 * i) * weight.e[g].two(2 * i);
        part[0] = fma(d[g][i], d[g][i], part[0]);
        part[1] = part[1] + q;
        part[2] = fma(q, d[g][i], part[2]);
      }
    float three[3];
#pragma unroll
    for (int k3 = 0; k3 < 3; ++k3) three[k3] = part[k3].v[0] + part[k3].v[1];
    team_sum<3, TEAM>(three, s_sum, turn);
    // (a row that is off is zeros, and adds zeros for any eps)
    const float r = on ? inverse_root(fmaf(three[0], inv, p.eps)) : 0.0f;
    const Vec<2> rr = splat<2>(r), mq = splat<2>(-three[1] * inv), mh = splat<2>(-three[2] * inv * r);
    X dx;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const Vec<2> y = dy.e[g].two(2 * i), h = d[g][i] * rr, q = fma(y, weight.e[g].two(2 * i), mq);
        dx.e[g].set(2 * i, rr * fma(h, mh, q));
        acc_weight[g][i] = fma(y, h, acc_weight[g][i]);
        acc_bias[g][i] = acc_bias[g][i] + y;
      }
    if (on) dx.store(to, 0, p.width);
    if constexpr (kAhead) x = x1, dy = dy1;
    else x.load(walk.at, p.width, on1), dy.load(walk_dy.at, p.width, on1);
    on = on1, of.row = next, to += apart;
  }
  store_part<TEAM, GROUPS, TEAMS, kWide>(acc_weight, p.part_weight, p, s_part);
  if (p.part_bias) store_part<TEAM, GROUPS, TEAMS, kWide>(acc_bias, p.part_bias, p, s_part);
}

struct Geometry {
  int team, groups;  // threads of a row, eights of channels of a thread
  bool wide;
  int64_t blocks;
};

template <class TX, class TY>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, cudaStream_t s);

}  // namespace lnorm
}  // namespace pesq
