// Gated linear recurrence over [batch, step, channel] streams, forward and
// backward.  Per row b and channel d, in scan order t (time, or time reversed):
//
//   r = sigmoid(decay_gate), i = sigmoid(input_gate)
//   log a = -rate softplus(decay_d) r,  beta = sqrt(1 - a^2)
//   h_t = a_t h_{t-1} + beta_t i_t x_t,  y_t = h_t
//
// A `reset` step forgets the state (a = 0, hence beta = 1); a step at or past
// the row's length keeps it (a = 1, beta = 0) and its output is zero.
//
// A warp owns V neighbouring channels per lane and a strip of consecutive steps,
// and walks the strip in chunks of 8 or 16 steps with the state in registers:
// everything of a step but one multiply-add is independent of the steps before it,
// so a chunk's gates are worked out side by side, two steps (or channels) an instruction, while
// the elements of the chunks to come are on their way.  Warps wait for nobody but their own
// copies: no flag, no atomic, and the order of every operation is fixed.
//
// Elements come in two ways.  Where channels and strides allow (multiples of 16
// bytes) and the row has 16 steps, a warp's chunks are boxes of 64 channels x 8 steps, or 32 x 16,
// that tensor copies bring to a ring in shared memory: one instruction for a box, no registers held.
// Otherwise every lane loads its own elements a chunk ahead (64 x 500 x 896 bfloat16: 86 us so, 77 by
// boxes; copies of 4 bytes a lane to shared memory: 259 us where plain loads take 95).
//
// With rows and channels enough to fill the device a strip is the whole row,
// and the data pass once.  Otherwise rows are cut into strips: the recurrence is
// the composition of maps h -> A h + H, a first kernel (`maps`) works out every
// strip's (A, H), and the second, launched while the first still runs and waiting for its end, starts
// each strip from the state that the maps before it give.  The strips of a CTA meet in shared memory,
// so a strip composes the maps of the CTAs before its own and one more.  Rows of 33 to 512 steps that
// would be cut go through one CTA for every 32 channels in one launch instead, which holds its steps as (a, b) in
// registers: of up to 512 threads, one an SM.
//
// What bounds it.  The bytes, 4 elements a step forward and 7 backward, are the floor; an element
// also takes 40 instruction slots forward and 65 backward, 5 of them special functions of eight
// cycles a warp.  With n warps a scheduler of 32 chunks each the time is 28 + 11 n us
// forward and 36 + 18 n backward: a warp's work on every pipe in turn, of which n warps overlap the rest.
// Measured (B200, cold caches, the call's kernels alone with the 6 us of a launch, channels that stay
// below kNear; bytes at the measured copy rate):
//                                             forward (bytes alone)    backward
//   64 x 500 x 896 bfloat16, uncut            73.8 us (35.1)           110.6 us (61.4)
//   96 x 512 x 512 float32, uncut, pairs      77.8 (61.6)              139.3 (107.8)
//   16 x 1000 x 512 float32, cut, boxes       49.2 (20.0)              61.5 (35.1)
//   6 x 4001 x 385 float32, cut, plain loads  63.5 (22.6)              85 (39.6)
//   1 x 32768 x 1040 bfloat16, cut, boxes     129.1 (41.7)             142 (73.0)
//   1 x 65537 x 129 float32, cut, plain loads 61.5 (20.7)              79.9 (36.2)   the fifth warp across: one lane
//   1 x 65537 x 128 float32, cut, boxes       51.2 (20.5)              63.5 (35.9)
//   8 x 500 x 768 bfloat16, one CTA each      22.5 (3.8)               26.7 (6.6)    192 CTAs forward: two rounds
// Cut rows read x and both gates twice forward, the decay gate and dy twice backward, which the bytes alone
// do not count.  Channels above kNear take the exponential: 64 x 500 x 896 81.9 and 116.7 us.
//
// Backward.  With g_t = dL/dh_t: g_t = dy_t + a_{t+1} g_{t+1}, the same kind of
// scan from the end of the row, carried as e_t = a_t g_t.  Then
//   dx = g beta i,   dinput_gate = dx x (1 - i),
//   dlog a = g (a h_{t-1} - (a^2 / beta) i x),   ddecay_gate = dlog a log a (1 - r),
//   ddecay = -rate sigmoid(decay) sum over rows and steps of dlog a r.
// h is not read back from the rounded y: the forward keeps the state before every
// chunk in 32 bits (1 / 8 or 1 / 16 of the elements), and the backward recomputes the
// chunk from it, by the same operations.  Chunks follow from the streams' addresses and strides, which
// may be others by the time of the backward, while a tracer needs the buffer's size from shapes alone: it
// has room for a state before every eighth step, of which chunks of 16 fill every other one.
// beta -> 0 only together with log a, whose quotient goes to zero: the term is dropped there.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "../../include/pesq_cuda.h"
#include "common.cuh"
#include "train.cuh"

namespace pesq {
namespace gscan {

using namespace train;

// steps of a chunk, by the channels of a lane: in shared memory sixteen elements of each
// stream either way, in registers no more than 8 steps
constexpr int chunk_steps(int vec, bool bulk) { return bulk ? 16 / vec : 8; }
constexpr int kKept = 8;  // steps between the places for states that a forward keeps
constexpr int kStrips = 8;  // strips (warps) of a CTA at most, where rows are cut
// CTAs of so many strips (4 or 8) that an SM holds by registers and shared memory, of elements of `size` bytes
constexpr int forward_ctas(int strips, bool bulk, int size) {
  return bulk && size == 2 ? (strips == 8 ? 3 : 5) : 16 / strips;
}
// (backward: 8 strips of 128 registers in the one case, where spills of 36 bytes cost less than the
// warps that they make room for; 4 of 168 in the others)
constexpr int backward_strips(bool bulk, bool mask, int size) { return bulk && !mask && size == 2 ? 8 : 4; }
constexpr int backward_ctas(int strips, bool bulk, bool mask, int size) {
  return (backward_strips(bulk, mask, size) == 8 ? 16 : 12) / strips;
}
constexpr int kRowWarps = 16, kHeld = 32;  // a row of up to 512 steps in one CTA
// chunks of a warp in shared memory: what 8 warps' chunks of four 32-bit streams leave room for
template <class T>
constexpr int kRing = sizeof(T) == 2 ? 3 : 2;

struct Stream {
  const void* p;
  int64_t sb;  // strides of batch, in elements,
  int st;      // and step, in bytes
};

struct Args {
  Stream x, ig, rg, dy;
  const float* decay;
  const float* state;         // [batch, width] or null (zeros)
  const uint8_t* reset;
  int64_t reset_b, reset_t;
  const int64_t* lengths;
  int64_t batch, steps, width;
  int ctiles;                 // warps across the channels
  int strips, strip;          // strips of a row, steps of one (a multiple of the chunk)
  int reverse;
  float rate;
  // cut rows: (A, H) of the strips before a strip in its CTA, [batch][rank][width],
  // and of a CTA's strips, [batch][CTA][width]; ranks count in the order of the scan at hand
  float2* before;
  float2* total;
  float* kept;                // state before every chunk, [batch][its first step / 8][width]
  // forward
  void* y;
  float* last;
  // backward
  const float* dlast;
  void *dx, *dig, *drg;
  float* dstate;
  float* dpart;               // [batch * strips, width] sums of dlog a r
  uint32_t* error;            // set when a copy does not come
};

// Tensor maps of the streams: [batch][step][channel], boxes of a chunk.  `out` by the input whose box in
// shared memory it leaves from: ddecay_gate, dinput_gate, and y or dx.
struct Maps {
  CUtensorMap rg, ig, x, dy, out[3];
};

// softplus(v): log1p(e) = 2 artanh(e / (2 + e)) by its series, e = exp(-|v|)
// (s <= 1/3: eight terms leave 1e-9).  Its error is the same at every step, so
// the exponential is the accurate one.
__device__ __forceinline__ float softplus(float v) {
  const float e = expf(-fabsf(v));
  const float s = e / (2.0f + e), q = s * s;
  float p = fmaf(q, 1.0f / 15, 1.0f / 13);
  p = fmaf(q, p, 1.0f / 11);
  p = fmaf(q, p, 1.0f / 9);
  p = fmaf(q, p, 1.0f / 7);
  p = fmaf(q, p, 1.0f / 5);
  p = fmaf(q, p, 1.0f / 3);
  p = fmaf(q, p, 1.0f);
  return max_nan(v, 0.0f) + 2.0f * s * p;
}

// The place of the state before chunk k
template <int L>
__device__ __forceinline__ int64_t kept_at(const Args& p, int64_t b, int k) {
  return (b * ((p.steps + kKept - 1) / kKept) + (int64_t)k * (L > kKept ? L / kKept : 1)) * p.width;
}

// The decay gate that steps past the length and outside the row read as
constexpr float kShut = -INFINITY;
// 1 - a^2 is held above this where its root is divided by
constexpr float kTiny = 1e-36f;
// rate softplus(decay) is held at this, so that times a shut gate it is zero
constexpr float kFast = 1e30f;
// rates -log a up to here go by the series alone
constexpr float kNear = 0.25f;

template <int N, int G>
struct Gates {
  Vec<N> i[G], r[G], a[G], beta[G];
  Vec<N> s[G];  // 1 / beta; where beta is zero, 1 / sqrt(kTiny), which its uses multiply by beta
};

// The gates of G Vecs side by side: operation by operation rather than Vec by
// Vec, so that every instruction has G independent ones next to it.
//
// k = rate softplus(decay) >= 0.  With m = -log a = k r, 1 - a = m (1 - m/2 + m^2/6 - ...)
// by its Taylor series (m^6 / 5040 < 5e-8 at 1/4): a is then rounded once, without the bias
// that a long memory would sum up, and 1 - a^2 = (1 - a)(2 - (1 - a)) does not
// cancel.  kFar: m may be above kNear, where the exponential takes over.
template <bool kFar, int N, int G>
__device__ __forceinline__ void decays(const Vec<N> (&r)[G], Vec<N> k, Vec<N> (&a)[G], Vec<N> (&w)[G]) {
  Vec<N> m[G], p[G];
  constexpr float kSeries[5] = {1.0f / 120, -1.0f / 24, 1.0f / 6, -0.5f, 1.0f};
#pragma unroll
  for (int g = 0; g < G; ++g) m[g] = k * r[g];
#pragma unroll
  for (int g = 0; g < G; ++g) p[g] = splat<N>(-1.0f / 720);
#pragma unroll
  for (int i = 0; i < 5; ++i)
#pragma unroll
    for (int g = 0; g < G; ++g) p[g] = fma(m[g], p[g], splat<N>(kSeries[i]));
#pragma unroll
  for (int g = 0; g < G; ++g) p[g] = m[g] * p[g];
#pragma unroll
  for (int g = 0; g < G; ++g) a[g] = fma(p[g], splat<N>(-1.0f), splat<N>(1.0f));
#pragma unroll
  for (int g = 0; g < G; ++g) w[g] = fma(p[g], splat<N>(-1.0f), splat<N>(2.0f));
#pragma unroll
  for (int g = 0; g < G; ++g) w[g] = p[g] * w[g];
  if (kFar) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!(m[g].v[j] < kNear)) {
          a[g].v[j] = exp2_approx(m[g].v[j] * -kLog2e);
          w[g].v[j] = fmaf(-a[g].v[j], a[g].v[j], 1.0f);
        }
  }
}

// 1 / (1 + exp(-v)); a reciprocal for each: one for the product of two needs both
// exponentials held below overflow, five operations more (64 x 500 x 896: 77 us, and 73 so)
template <int N, int G>
__device__ __forceinline__ void sigmoids(const Vec<N> (&v)[G], Vec<N> (&out)[G]) {
#pragma unroll
  for (int g = 0; g < G; ++g) out[g] = v[g] * splat<N>(-kLog2e);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) out[g].v[j] = exp2_approx(out[g].v[j]);
#pragma unroll
  for (int g = 0; g < G; ++g) out[g] = out[g] + splat<N>(1.0f);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) out[g].v[j] = rcp_approx(out[g].v[j]);
}

template <bool kFar, int N, int G>
__device__ __forceinline__ void gates(const Vec<N> (&ig)[G], const Vec<N> (&rg)[G], Vec<N> k, Gates<N, G>& o) {
  Vec<N> w[G];
  sigmoids(rg, o.r);
  sigmoids(ig, o.i);
  decays<kFar>(o.r, k, o.a, w);
#pragma unroll
  for (int g = 0; g < G; ++g) o.s[g] = w[g] + splat<N>(kTiny);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) o.s[g].v[j] = rsqrt_approx(o.s[g].v[j]);
#pragma unroll
  for (int g = 0; g < G; ++g) o.beta[g] = w[g] * o.s[g];
}

// a h + b.  A state that a = 0 cuts off is not looked at (it may be infinite or NaN).
template <bool kMask, int N>
__device__ __forceinline__ Vec<N> apply(Vec<N> a, Vec<N> h, Vec<N> b) {
  if (kMask) {
#pragma unroll
    for (int j = 0; j < N; ++j) h.v[j] = a.v[j] == 0.0f ? 0.0f : h.v[j];
  }
  return fma(a, h, b);
}
// The factor of a map that `a` comes after, as apply() looks at it: a = 0 cuts off what was not finite too
template <bool kMask>
__device__ __forceinline__ Vec<1> chain(Vec<1> a, Vec<1> A) {
  return kMask && a.v[0] == 0.0f ? Vec<1>{{0.0f}} : A * a;
}

// What a lane works on, and where its strip lies.  Chunks are counted in the order of
// the steps' scan.
struct Lane {
  int64_t b, c;      // row, first channel
  int rank;          // of the strip, in the order of this scan
  int lo, hi;        // the row's chunks that have a step before its length: the strips share these
  int first, count;  // the strip's
  int whole;         // those of them that have all their steps
  int dir;           // memory direction of the steps' scan
  int len;           // the row's length
  bool on;           // channels in range
  int64_t from;      // first channel to read
};

template <int V, int L, bool kMask, bool kBack>
__device__ __forceinline__ Lane lane_of(const Args& p) {
  Lane o;
  o.b = blockIdx.y;
  const unsigned block = L == 1 ? 0 : blockIdx.x / p.ctiles;  // CTA along the row
  // (a CTA's warps are strips of the row, but for single steps, which have none: neighbours in the channels)
  const unsigned tile = L == 1 ? blockIdx.x * blockDim.y + threadIdx.y : blockIdx.x - block * p.ctiles;
  o.c = (int64_t)tile * (32 * V) + threadIdx.x * V;
  o.on = o.c < p.width;
  o.from = o.on ? o.c : 0;
  o.rank = L == 1 ? 0 : block * blockDim.y + threadIdx.y;
  const int strip = kBack ? p.strips - 1 - o.rank : o.rank, steps = (int)p.steps;
  const int all = (steps + L - 1) / L;
  int per = p.strip / L;
  o.lo = 0, o.hi = all;
  o.len = steps;
  o.dir = p.reverse ? -1 : 1;
  if (kMask && p.lengths) {
    o.len = (int)max(INT64_C(0), min(p.lengths[o.b], p.steps));
    // (from a multiple of 16 steps on with chunks of eight too, for the states that chunks of 16 ask for)
    o.lo = p.reverse ? (steps - o.len) / 16 * 16 / L : 0;
    o.hi = o.len == 0 ? o.lo : p.reverse ? all : (o.len + L - 1) / L;
    per = (o.hi - o.lo + p.strips - 1) / p.strips;
  }
  o.first = o.lo + strip * per;
  o.count = strip < 0 || strip >= p.strips ? 0 : max(0, min(per, o.hi - o.first));
  o.whole = min(o.count, max(0, steps / L - o.first));
  return o;
}

// Steps of one chunk, a bit each
struct Chunk {
  int64_t t0;       // first step, in memory
  unsigned inside;  // steps of the row
  unsigned live;    // before the row's length
  unsigned flag;    // reset, of the step with the lane's number
};
template <int L, bool kMask>
__device__ __forceinline__ Chunk chunk_of(const Args& p, const Lane& o, int k) {
  constexpr unsigned kAll = (1u << L) - 1;
  Chunk q;
  const int s0 = k * L, left = (int)p.steps - s0, t0 = p.reverse ? left - 1 : s0;
  q.t0 = t0;
  q.inside = left >= L ? kAll : (1u << left) - 1;
  q.live = q.inside;
  if (kMask) {
    if (p.reverse) {
      const int dead = t0 - o.len + 1;  // steps at the chunk's start
      if (dead > 0) q.live &= dead >= L ? 0u : ~0u << dead;
    } else if (o.len - t0 < L) {
      q.live &= o.len <= t0 ? 0u : (1u << (o.len - t0)) - 1;
    }
  }
  q.flag = 0u;
  return q;
}
// Starts the load of the chunk's resets, one lane a step; cuts() gathers them
template <int L, bool kMask>
__device__ __forceinline__ void flag_chunk(const Args& p, const Lane& o, Chunk& q) {
  if (!kMask || !p.reset) return;
  const unsigned mine = threadIdx.x < L ? (q.live >> threadIdx.x) & 1u : 0u;
  const uint8_t* at = p.reset + o.b * p.reset_b + (q.t0 + (int)threadIdx.x * o.dir) * p.reset_t;
  asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n@q ld.global.u8 %0, [%1];\n}" : "+r"(q.flag) : "l"(at), "r"(mine));
}
template <bool kMask>
__device__ __forceinline__ unsigned cuts(const Args& p, const Chunk& q) {
  return kMask && p.reset ? __ballot_sync(0xffffffffu, q.flag != 0u) : 0u;
}

// Launches of one call follow one another closely: the next one may start once
// all blocks of this one have
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// and waits here until this one is done
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Loads one pack where `take` is nonzero and leaves it as it is otherwise: a
// predicated load, with no branch whose join would wait for it
template <class P>
__device__ __forceinline__ void load_if(P& out, const char* p, unsigned take) {
  if constexpr (sizeof(P) == 2) {
    asm("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n@q ld.global.b16 %0, [%1];\n}"
        : "+h"(reinterpret_cast<unsigned short&>(out))
        : "l"(p), "r"(take));
  } else if constexpr (sizeof(P) == 4) {
    asm("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n@q ld.global.b32 %0, [%1];\n}"
        : "+r"(reinterpret_cast<unsigned&>(out))
        : "l"(p), "r"(take));
  } else {
    asm("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n@q ld.global.b64 %0, [%1];\n}"
        : "+l"(reinterpret_cast<unsigned long long&>(out))
        : "l"(p), "r"(take));
  }
}

// The steps of a chunk, in scan order; those that are not live read as `other`
// and are not touched.  A decay gate of kShut makes a step the identity to the
// last bit: a = 1, and b = 0 for x = 0.  kFull: all steps are live.
template <class T, int V, int L, bool kFull>
__device__ __forceinline__ void load(Pack<T, V> (&out)[L], const Stream& s, const Lane& o, const Chunk& q,
                                     float other = 0.0f) {
  // (lanes past the width read the row's first channels)
  const char* p = reinterpret_cast<const char*>(static_cast<const T*>(s.p) + o.b * s.sb + o.from) + q.t0 * s.st;
  const int step = o.dir * s.st;
  if (kFull) {
#pragma unroll
    for (int l = 0; l < L; ++l) out[l] = *reinterpret_cast<const Pack<T, V>*>(p + (int64_t)step * l);
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l) {
#pragma unroll
      for (int v = 0; v < V; ++v) out[l].v[v] = narrow<T>(other);
      load_if(out[l], p + (int64_t)step * l, (q.live >> l) & 1u);
    }
  }
}
template <class T, int V>
__device__ __forceinline__ void store(void* p, Vec<V> val) {
  Pack<T, V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.v[v] = narrow<T>(val.v[v]);
  *static_cast<Pack<T, V>*>(p) = o;
}

// The L x V elements of a chunk as G Vecs for the two-wide instructions: pairs of
// channels, or of steps where a lane has a single channel.
template <int V, int L>
struct Cells {
  static constexpr int N = V == 2 || L % 2 == 0 ? 2 : 1, G = L * V / N;
  using Array = Vec<N>[G];
  // those of a step
  static __device__ __forceinline__ Vec<V> at(const Array& c, int l) {
    if constexpr (V == N)
      return c[l];
    else
      return {{c[l / N].v[l % N]}};
  }
  static __device__ __forceinline__ void put(Array& c, int l, Vec<V> x) {
    if constexpr (V == N)
      c[l] = x;
    else
      c[l / N].v[l % N] = x.v[0];
  }
  template <class T>
  static __device__ __forceinline__ void widen(const Pack<T, V> (&p)[L], Array& out) {
#pragma unroll
    for (int l = 0; l < L; ++l) put(out, l, train::widen<V>(p[l], 0));
  }
};

// The gates of a chunk; a step that `cut` has a bit for forgets the state
template <class T, int V, int L, bool kMask, bool kFar>
__device__ __forceinline__ void gates_of(unsigned cut, const Pack<T, V> (&ig)[L], const Pack<T, V> (&rg)[L],
                                         Vec<V> rate, Gates<Cells<V, L>::N, Cells<V, L>::G>& out) {
  using C = Cells<V, L>;
  typename C::Array i, r;
  C::widen(ig, i), C::widen(rg, r);
  Vec<C::N> k;
#pragma unroll
  for (int j = 0; j < C::N; ++j) k.v[j] = rate.v[j % V];
  gates<kFar>(i, r, k, out);
  if (kMask) {
#pragma unroll
    for (int l = 0; l < L; ++l)
      if ((cut >> l) & 1u) C::put(out.a, l, splat<V>(0.0f)), C::put(out.beta, l, splat<V>(1.0f));
  }
}

// The rates of a lane's channels, and whether one of the warp's is above kNear
template <int V>
__device__ __forceinline__ bool rates(const Args& p, const Lane& o, Vec<V>& rate) {
  bool far = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float k = o.on ? p.rate * softplus(p.decay[o.c + v]) : 0.0f;
    if (k > kFast) k = kFast;
    rate.v[v] = k;
    far = far || !(k < kNear);
  }
  return __any_sync(0xffffffffu, far);
}

template <int V>
__device__ __forceinline__ Vec<V> read_row(const float* p) {
  Vec<V> out;
#pragma unroll
  for (int v = 0; v < V; ++v) out.v[v] = p[v];
  return out;
}

// Start value of a strip: the row's, through the maps of the CTAs before and of
// the strips before in the CTA
template <bool kMask>
__device__ __forceinline__ void start_of(const Args& p, const Lane& o, Vec<1>& h) {
  if (p.strips == 1 || !o.on || o.rank >= p.strips) return;
  const int w = blockDim.y, ctas = (p.strips + w - 1) / w, cta = o.rank / w;
  const float2* t = p.total + o.b * ctas * p.width + o.c;
#pragma unroll 8
  for (int k = 0; k < cta; ++k) {
    const float2 m = t[k * p.width];
    h = apply<kMask>(Vec<1>{{m.x}}, h, Vec<1>{{m.y}});
  }
  const float2 m = p.before[(o.b * p.strips + o.rank) * p.width + o.c];
  h = apply<kMask>(Vec<1>{{m.x}}, h, Vec<1>{{m.y}});
}

// The maps of a CTA's strips, warp by warp: leaves in `before` what the strips
// before each make of a state, and in `total` all of them.
template <bool kMask>
__device__ __forceinline__ void join_maps(const Args& p, const Lane& o, Vec<1> A, Vec<1> H) {
  __shared__ float2 s_map[kStrips][32];
  s_map[threadIdx.y][threadIdx.x] = make_float2(A.v[0], H.v[0]);
  __syncthreads();
  if (!o.on || o.rank >= p.strips) return;
  const int strips = blockDim.y;
  Vec<1> a{{1.0f}}, h{{0.0f}};
  for (int w = 0; w < (int)threadIdx.y; ++w) {
    const float2 m = s_map[w][threadIdx.x];
    h = apply<kMask>(Vec<1>{{m.x}}, h, Vec<1>{{m.y}});
    a = chain<kMask>(Vec<1>{{m.x}}, a);
  }
  p.before[(o.b * p.strips + o.rank) * p.width + o.c] = make_float2(a.v[0], h.v[0]);
  if ((int)threadIdx.y == strips - 1 || o.rank == p.strips - 1) {
    const float2 m = s_map[threadIdx.y][threadIdx.x];
    h = apply<kMask>(Vec<1>{{m.x}}, h, Vec<1>{{m.y}});
    const int ctas = (p.strips + strips - 1) / strips;
    p.total[(o.b * ctas + o.rank / strips) * p.width + o.c] =
        make_float2(chain<kMask>(Vec<1>{{m.x}}, a).v[0], h.v[0]);
  }
}

// What a chunk holds of the steps that are not live: the identity to the last bit
template <class T, int V, int L>
__device__ __forceinline__ void blank(Pack<T, V> (&out)[L], const Chunk& q, float other = 0.0f) {
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (!((q.live >> l) & 1u)) out[l].v[v] = narrow<T>(other);
}

// Zeros for the steps of the chunks that the row's length leaves out, the warps of
// the row sharing them
template <class T, int V, int L, int K>
__device__ __forceinline__ void zero_rest(const Args& p, const Lane& o, void* const (&out)[K]) {
  const int all = ((int)p.steps + L - 1) / L, dead = all - (o.hi - o.lo);
  if (dead == 0 || !o.on || o.rank >= p.strips) return;
  Pack<T, V> z;
#pragma unroll
  for (int v = 0; v < V; ++v) z.v[v] = narrow<T>(0.0f);
  // (they lie at one end of the row)
  const int base = o.lo > 0 ? 0 : o.hi, per = (dead + p.strips - 1) / p.strips;
  const int s0 = min((int)p.steps, min(base + dead, base + o.rank * per) * L);
  const int s1 = min((int)p.steps, min(base + dead, base + (o.rank + 1) * per) * L);
  const int64_t t = p.reverse ? p.steps - 1 - s0 : s0, step = o.dir * p.width;
  const int64_t at = (o.b * p.steps + t) * p.width + o.c;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    T* to = static_cast<T*>(out[k]) + at;
#pragma unroll 4
    for (int s = s0; s < s1; ++s, to += step) *reinterpret_cast<Pack<T, V>*>(to) = z;
  }
}

// Takes n chunks in turn, each read one before its use: read(k, in) and
// work(k, in) for k = 0 .. n - 1.  (The last reads are repeated rather than
// branched around: a join would wait for them.)
template <class In, class R, class W>
__device__ __forceinline__ void walk(int n, R read, W work) {
  if (n <= 0) return;
  In one, two;
  read(0, one);
#pragma unroll 1
  for (int k = 0; k < n; k += 2) {
    read(min(k + 1, n - 1), two);
    work(k, one);
    read(min(k + 2, n - 1), one);
    if (k + 1 < n) work(k + 1, two);
  }
}

// A warp's ring of chunks in shared memory: kRing stages of S streams' boxes
// [L][32 V] and, with kState, the states before the chunk.  With kOut, 16-bit results take the place
// of the inputs in their stage and leave by tensor copies as well, which saves a thread their
// addresses (64 x 500 x 896: backward 114 -> 109 us); the stage is filled again a chunk later.  32-bit
// rings have two stages only, and their results leave from the registers.
template <class T, int V, int L, int S, bool kState, bool kOut>
struct Ring {
  static constexpr bool kStaged = kOut && sizeof(T) == 2;
  static constexpr int kBox = L * 32 * V * (int)sizeof(T);
  static constexpr int kStage = S * kBox + (kState ? 128 * V : 0);
  static constexpr int kBytes = kRing<T> * kStage;  // of a warp
  char* base;
  uint64_t* bar;
  const CUtensorMap *map[S], *out;

  __device__ __forceinline__ Ring(char* smem, uint64_t* bars)
      : base(smem + threadIdx.y * kBytes), bar(bars + threadIdx.y * kRing<T>) {
    if (threadIdx.x == 0) {
#pragma unroll
      for (int i = 0; i < kRing<T>; ++i) mbar_init(bar + i);
    }
    __syncwarp();
  }
  // one lane
  __device__ __forceinline__ void send(const Args& p, const Lane& o, int k, int stage) {
    const int c0 = (int)o.c, t0 = p.reverse ? (int)p.steps - (k + 1) * L : k * L;
    char* to = base + stage * kStage;
    uint32_t bytes = S * kBox, state = 0;
    if (kState) state = (uint32_t)min((int64_t)(32 * V), p.width - o.c) * 4, bytes += state;
    mbar_arrive_expect_tx(bar + stage, bytes);
#pragma unroll
    for (int i = 0; i < S; ++i)
      asm volatile(
          "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
              smem_u32(to + i * kBox)),
          "l"(map[i]), "r"(smem_u32(bar + stage)), "r"(c0), "r"(t0), "r"((int)o.b)
          : "memory");
    if (kState)
      bulk_g2s(to + S * kBox, p.kept + kept_at<L>(p, o.b, k) + o.c, state, bar + stage);
  }
  // one stream of the stage, in scan order
  __device__ __forceinline__ void get(const Args& p, int stage, int i, Pack<T, V> (&out)[L]) const {
    const Pack<T, V>* s = reinterpret_cast<const Pack<T, V>*>(base + stage * kStage + i * kBox) + threadIdx.x;
    const int step = p.reverse ? -32 : 32;
    s += p.reverse ? (L - 1) * 32 : 0;
#pragma unroll
    for (int l = 0; l < L; ++l) out[l] = s[l * step];
  }
  // a result of step l in the place of stream i, and all of the chunk's from stream `from` on to memory
  __device__ __forceinline__ void put(const Args& p, int stage, int i, int l, Vec<V> val) const {
    Pack<T, V>* s = reinterpret_cast<Pack<T, V>*>(base + stage * kStage + i * kBox) + threadIdx.x;
    const int step = p.reverse ? -32 : 32;
    s += p.reverse ? (L - 1) * 32 : 0;
    store<T>(s + l * step, val);
  }
  template <int kFrom>
  __device__ __forceinline__ void leave(const Args& p, const Lane& o, int k, int stage) const {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (threadIdx.x == 0) {
      const int c0 = (int)o.c, t0 = p.reverse ? (int)p.steps - (k + 1) * L : k * L;  // (a whole chunk: not negative)
#pragma unroll
      for (int i = kFrom; i < 3; ++i)
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(out + i),
                     "r"(smem_u32(base + stage * kStage + i * kBox)), "r"(c0), "r"(t0), "r"((int)o.b)
                     : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  __device__ __forceinline__ Pack<float, V> state(int stage) const {
    return reinterpret_cast<const Pack<float, V>*>(base + stage * kStage + S * kBox)[threadIdx.x];
  }
  // The first copies of a walk
  __device__ __forceinline__ void start(const Args& p, const Lane& o, int first, int n, int way) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < kRing<T> && i < n; ++i) send(p, o, first + way * i, i);
    }
  }
  // Chunks first, first + way, ..., after start(): read(stage, q, in) takes a chunk out of its
  // stage, work(k, in) works on it while the stage fills again.  Returns false where a copy
  // does not come.
  template <bool kMask, class In, class R, class W>
  __device__ __forceinline__ bool walk(const Args& p, const Lane& o, int first, int n, int way, R read, W work) {
    int stage = 0, parity = 0;
    bool ok = true;
    Chunk q = chunk_of<L, kMask>(p, o, first);
    if (n > 0) flag_chunk<L, kMask>(p, o, q);
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      if (!__all_sync(0xffffffffu, mbar_wait(bar + stage, parity))) {
        ok = false;
        break;
      }
      In in;
      in.q = q;
      in.stage = stage;
      read(stage, in);
      __syncwarp();
      if (kStaged) {  // the stage before, once its results have left it
        if (threadIdx.x == 0 && k > 0 && k - 1 + kRing<T> < n) {
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          send(p, o, first + way * (k - 1 + kRing<T>), stage == 0 ? kRing<T> - 1 : stage - 1);
        }
      } else if (threadIdx.x == 0 && k + kRing<T> < n) {
        send(p, o, first + way * (k + kRing<T>), stage);
      }
      q = chunk_of<L, kMask>(p, o, first + way * min(k + 1, n - 1));
      flag_chunk<L, kMask>(p, o, q);
      work(first + way * k, in);
      if (++stage == kRing<T>) stage = 0, parity ^= 1;
    }
    if (!ok) {  // nothing may be in flight to shared memory that another block gets
      if (threadIdx.x == 0) atomicOr(p.error, 1u);
      for (int i = 0; i < kRing<T>; ++i) mbar_wait(bar + i, i < stage ? parity ^ 1 : parity);
    }
    if (kStaged && threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    return ok;
  }
};
// a warp without a ring, where every lane loads its own
struct NoRing {
  static constexpr bool kStaged = false;
};

// ------------------------------------------------------------------- forward

template <class T, int V, int L>
struct Loaded {
  Chunk q;
  int stage;  // of a ring
  Pack<T, V> x[L], ig[L], rg[L];
  template <class R>
  __device__ __forceinline__ void get(const Args& p, const R& ring, int stage) {
    ring.get(p, stage, 0, rg);
    ring.get(p, stage, 1, ig);
    ring.get(p, stage, 2, x);
  }
  template <bool kMask, bool kFull>
  __device__ __forceinline__ void read(const Args& p, const Lane& o, int k) {
    q = chunk_of<L, kMask>(p, o, k);
    flag_chunk<L, kMask>(p, o, q);
    load<T, V, L, kFull>(rg, p.rg, o, q, kShut);
    load<T, V, L, kFull>(ig, p.ig, o, q);
    load<T, V, L, kFull>(x, p.x, o, q);
  }
  // Every step as h -> a h + b
  template <bool kMask, bool kFar>
  __device__ __forceinline__ void steps(const Args& p, Vec<V> rate, Gates<Cells<V, L>::N, Cells<V, L>::G>& g,
                                        typename Cells<V, L>::Array& b) {
    if (q.live != (1u << L) - 1) blank(rg, q, kShut), blank(ig, q), blank(x, q);
    gates_of<T, V, L, kMask, kFar>(cuts<kMask>(p, q), ig, rg, rate, g);
    Cells<V, L>::widen(x, b);
#pragma unroll
    for (int i = 0; i < Cells<V, L>::G; ++i) b[i] = g.beta[i] * (g.i[i] * b[i]);
  }
};

// Takes the strip's chunks in scan order: work(k, in, whole).  The last one of a row may lack steps.
template <class T, int V, int L, bool kMask, class R, class W>
__device__ __forceinline__ bool forward_walk(const Args& p, const Lane& o, R& ring, W work) {
  using In = Loaded<T, V, L>;
  if constexpr (!std::is_same<R, NoRing>::value) {
    return ring.template walk<kMask, In>(
        p, o, o.first, o.count, 1, [&](int stage, In& in) { in.get(p, ring, stage); },
        [&](int k, In& in) {
          if (k - o.first < o.whole)
            work(k, in, std::true_type{});
          else
            work(k, in, std::false_type{});
        });
  } else {
    walk<In>(
        o.whole, [&](int k, In& in) { in.template read<kMask, true>(p, o, o.first + k); },
        [&](int k, In& in) { work(o.first + k, in, std::true_type{}); });
    if (o.whole < o.count) {
      In in;
      in.template read<kMask, false>(p, o, o.first + o.whole);
      work(o.first + o.whole, in, std::false_type{});
    }
    return true;
  }
}

template <class T, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void forward_maps(const Args& p, const Lane& o, R& ring, Vec<1> rate) {
  using C = Cells<1, L>;
  Vec<1> A = splat<1>(1.0f), H = splat<1>(0.0f);
  forward_walk<T, 1, L, kMask>(p, o, ring, [&](int, Loaded<T, 1, L>& in, auto) {
    Gates<C::N, C::G> g;
    typename C::Array b;
    in.template steps<kMask, kFar>(p, rate, g, b);
#pragma unroll
    for (int l = 0; l < L; ++l) {
      H = apply<kMask>(C::at(g.a, l), H, C::at(b, l));
      A = chain<kMask>(C::at(g.a, l), A);
    }
  });
  join_maps<kMask>(p, o, A, H);
}

// The ring of a forward warp, with its first copies on their way
template <class T, int V, int L, bool kBulk, bool kOut>
__device__ __forceinline__ auto forward_ring(const Args& p, const Maps& m, const Lane& o) {
  if constexpr (kBulk) {
    extern __shared__ __align__(128) char dynamic[];
    __shared__ uint64_t s_bar[kRowWarps * kRing<T>];
    Ring<T, V, L, 3, false, kOut> ring(dynamic, s_bar);
    ring.map[0] = &m.rg, ring.map[1] = &m.ig, ring.map[2] = &m.x, ring.out = m.out;
    ring.start(p, o, o.first, o.count, 1);
    return ring;
  } else {
    return NoRing{};
  }
}

template <class T, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kStrips, forward_ctas(8, kBulk, sizeof(T)))
    forward_maps_kernel(const __grid_constant__ Args p, const __grid_constant__ Maps m) {
  let_next_start();
  const Lane o = lane_of<1, L, kMask, false>(p);
  auto ring = forward_ring<T, 1, L, kBulk, false>(p, m, o);
  Vec<1> rate;
  // (the CTA's warps share their channels, so they agree, and meet in join_maps)
  if (rates<1>(p, o, rate))
    forward_maps<T, L, kMask, true>(p, o, ring, rate);
  else
    forward_maps<T, L, kMask, false>(p, o, ring, rate);
}

template <class T, int V, int L, bool kMask, bool kFar, bool kFull, class R>
__device__ __forceinline__ void forward_chunk(const Args& p, const Lane& o, const R& ring, int k, Loaded<T, V, L>& in,
                                              Vec<V> rate, Vec<V>& h) {
  using C = Cells<V, L>;
  if (p.kept && o.on) {
    float* keep = p.kept + kept_at<L>(p, o.b, k) + o.c;
#pragma unroll
    for (int v = 0; v < V; ++v) keep[v] = h.v[v];
  }
  Gates<C::N, C::G> g;
  typename C::Array b;
  in.template steps<kMask, kFar>(p, rate, g, b);
  char* y = reinterpret_cast<char*>(static_cast<T*>(p.y) + (o.b * p.steps + in.q.t0) * p.width + o.c);
  const int step = o.dir * (int)p.width * (int)sizeof(T);
#pragma unroll
  for (int l = 0; l < L; ++l) {
    h = apply<kMask>(C::at(g.a, l), h, C::at(b, l));
    const Vec<V> out = !kMask || ((in.q.live >> l) & 1u) ? h : splat<V>(0.0f);
    if constexpr (R::kStaged && kFull)
      ring.put(p, in.stage, 2, l, out);
    else if (o.on && (kFull || ((in.q.inside >> l) & 1u)))
      store<T>(y + (int64_t)step * l, out);
  }
  if constexpr (R::kStaged && kFull) ring.template leave<2>(p, o, k, in.stage);
}

template <class T, int V, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void forward_strip(const Args& p, const Lane& o, R& ring, Vec<V> rate) {
  Vec<V> h = splat<V>(0.0f);
  if (p.state) h = read_row<V>(p.state + o.b * p.width + o.from);
  if constexpr (V == 1) {
    if (p.strips > 1) wait_for_last();
    if (o.rank >= p.strips) return;
    start_of<kMask>(p, o, h);
  }
  if (!forward_walk<T, V, L, kMask>(p, o, ring, [&](int k, Loaded<T, V, L>& in, auto full) {
        forward_chunk<T, V, L, kMask, kFar, decltype(full)::value>(p, o, ring, k, in, rate, h);
      }))
    return;
  if (kMask) zero_rest<T, V, L, 1>(p, o, {p.y});
  if (o.rank == p.strips - 1 && o.on) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.last[o.b * p.width + o.c + v] = h.v[v];
  }
}

template <class T, int V, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(V == 2 && L > 1 ? 32 : 32 * kStrips,
                                  V == 2 && L > 1 ? (kBulk ? 16 : 11) : forward_ctas(8, kBulk, sizeof(T)))
    forward_kernel(const __grid_constant__ Args p, const __grid_constant__ Maps m) {
  const Lane o = lane_of<V, L, kMask, false>(p);
  auto ring = forward_ring<T, V, L, kBulk, true>(p, m, o);
  Vec<V> rate;
  if (rates<V>(p, o, rate))
    forward_strip<T, V, L, kMask, true>(p, o, ring, rate);
  else
    forward_strip<T, V, L, kMask, false>(p, o, ring, rate);
}

// A short row in one CTA: a warp holds its strip of kHeld steps as (a, b) in registers,
// the strips' maps meet in shared memory, and the recursion is run from the state that
// they give.  The data pass once, in one launch: 24 x 187 x 896 bfloat16 14.1 us, where strips in
// two launches take 18.2.  With more rows than fill the device whole rows a warp are as good:
// 32 x 500 x 896 47.6 us so, 45.7 as whole rows.
template <class T, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void forward_row(const Args& p, const Lane& o, R& ring, Vec<1> rate) {
  using C = Cells<1, L>;
  constexpr int NC = kHeld / L;
  __shared__ float2 s_map[kRowWarps][32];
  typename C::Array a[NC], b[NC];
  Vec<1> A{{1.0f}}, H{{0.0f}};
  unsigned live[NC];
  using In = Loaded<T, 1, L>;
  In in[2];
  if constexpr (std::is_same<R, NoRing>::value) {
    if (o.count > 0) in[0].template read<kMask, false>(p, o, o.first);
  }
  bool ok = true;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    live[c] = 0u;
#pragma unroll
    for (int g = 0; g < C::G; ++g) a[c][g] = splat<C::N>(1.0f), b[c][g] = splat<C::N>(0.0f);
    if (c >= o.count) continue;
    In& now = in[c % 2];
    if constexpr (std::is_same<R, NoRing>::value) {
      if (c + 1 < NC && c + 1 < o.count) in[(c + 1) % 2].template read<kMask, false>(p, o, o.first + c + 1);
    } else {
      now.q = chunk_of<L, kMask>(p, o, o.first + c);
      flag_chunk<L, kMask>(p, o, now.q);
      const bool came = __all_sync(0xffffffffu, mbar_wait(ring.bar + c, 0));
      ok = ok && came;
      now.get(p, ring, c);
    }
    Gates<C::N, C::G> g;
    now.template steps<kMask, kFar>(p, rate, g, b[c]);
    live[c] = now.q.live;
#pragma unroll
    for (int i = 0; i < C::G; ++i) a[c][i] = g.a[i];
#pragma unroll
    for (int l = 0; l < L; ++l) {
      H = apply<kMask>(C::at(a[c], l), H, C::at(b[c], l));
      A = chain<kMask>(C::at(a[c], l), A);
    }
  }
  if constexpr (!std::is_same<R, NoRing>::value) {
    if (!ok) {  // as in Ring::walk
      if (threadIdx.x == 0) atomicOr(p.error, 1u);
      for (int c = 0; c < o.count; ++c) mbar_wait(ring.bar + c, 0);
    }
  }
  s_map[threadIdx.y][threadIdx.x] = make_float2(A.v[0], H.v[0]);
  __syncthreads();
  Vec<1> h{{p.state ? p.state[o.b * p.width + o.from] : 0.0f}};
  for (int w = 0; w < (int)threadIdx.y; ++w) {
    const float2 m = s_map[w][threadIdx.x];
    h = apply<kMask>(Vec<1>{{m.x}}, h, Vec<1>{{m.y}});
  }
  if (!o.on) return;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c >= o.count) continue;
    const Chunk q = chunk_of<L, kMask>(p, o, o.first + c);
    if (p.kept) p.kept[kept_at<L>(p, o.b, o.first + c) + o.c] = h.v[0];
    char* y = reinterpret_cast<char*>(static_cast<T*>(p.y) + (o.b * p.steps + q.t0) * p.width + o.c);
    const int step = o.dir * (int)p.width * (int)sizeof(T);
#pragma unroll
    for (int l = 0; l < L; ++l) {
      h = apply<kMask>(C::at(a[c], l), h, C::at(b[c], l));
      const Vec<1> out = !kMask || ((live[c] >> l) & 1u) ? h : splat<1>(0.0f);
      if ((q.inside >> l) & 1u) store<T>(y + (int64_t)step * l, out);
    }
  }
  if (kMask) zero_rest<T, 1, L, 1>(p, o, {p.y});
  if (o.rank == p.strips - 1) p.last[o.b * p.width + o.c] = h.v[0];
}

template <class T, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kRowWarps) forward_row_kernel(const __grid_constant__ Args p,
                                                                     const __grid_constant__ Maps m) {
  const Lane o = lane_of<1, L, kMask, false>(p);
  auto ring = forward_ring<T, 1, L, kBulk, false>(p, m, o);
  Vec<1> rate;
  if (rates<1>(p, o, rate))
    forward_row<T, L, kMask, true>(p, o, ring, rate);
  else
    forward_row<T, L, kMask, false>(p, o, ring, rate);
}

// ------------------------------------------------------------------ backward

template <class T, int V, int L>
struct LoadedMap {
  Chunk q;
  int stage;  // of a ring
  Pack<T, V> rg[L], dy[L];
  template <class R>
  __device__ __forceinline__ void get(const Args& p, const R& ring, int stage) {
    ring.get(p, stage, 0, rg);
    ring.get(p, stage, 1, dy);
  }
  template <bool kMask, bool kFull>
  __device__ __forceinline__ void read(const Args& p, const Lane& o, int k) {
    q = chunk_of<L, kMask>(p, o, k);
    flag_chunk<L, kMask>(p, o, q);
    load<T, V, L, kFull>(rg, p.rg, o, q, kShut);
    load<T, V, L, kFull>(dy, p.dy, o, q);
  }
};

template <class T, int V, int L>
struct LoadedBack {
  Chunk q;
  int stage;  // of a ring
  Pack<T, V> x[L], ig[L], rg[L], dy[L];
  Vec<V> h;  // state before the chunk
  template <class R>
  __device__ __forceinline__ void get(const Args& p, const R& ring, int stage) {
    ring.get(p, stage, 0, rg);
    ring.get(p, stage, 1, ig);
    ring.get(p, stage, 2, x);
    ring.get(p, stage, 3, dy);
    h = widen<V>(ring.state(stage), 0);
  }
  template <bool kMask, bool kFull>
  __device__ __forceinline__ void read(const Args& p, const Lane& o, int k) {
    q = chunk_of<L, kMask>(p, o, k);
    flag_chunk<L, kMask>(p, o, q);
    load<T, V, L, kFull>(rg, p.rg, o, q, kShut);
    load<T, V, L, kFull>(ig, p.ig, o, q);
    load<T, V, L, kFull>(x, p.x, o, q);
    load<T, V, L, kFull>(dy, p.dy, o, q);
    h = read_row<V>(p.kept + kept_at<L>(p, o.b, k) + o.from);
  }
};

// Takes the strip's chunks against scan order
template <class T, int V, int L, bool kMask, class In, class R, class W>
__device__ __forceinline__ bool backward_walk(const Args& p, const Lane& o, R& ring, W work) {
  if constexpr (!std::is_same<R, NoRing>::value) {
    return ring.template walk<kMask, In>(
        p, o, o.first + o.count - 1, o.count, -1, [&](int stage, In& in) { in.get(p, ring, stage); },
        [&](int k, In& in) {
          if (k - o.first < o.whole)
            work(k, in, std::true_type{});
          else
            work(k, in, std::false_type{});
        });
  } else {
    if (o.whole < o.count) {
      In in;
      in.template read<kMask, false>(p, o, o.first + o.whole);
      work(o.first + o.whole, in, std::false_type{});
    }
    walk<In>(
        o.whole, [&](int k, In& in) { in.template read<kMask, true>(p, o, o.first + o.whole - 1 - k); },
        [&](int k, In& in) { work(o.first + o.whole - 1 - k, in, std::true_type{}); });
    return true;
  }
}

// e -> A e + E of a strip, from its last step to its first: the decay gate and
// dy are all it takes
template <class T, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void backward_maps(const Args& p, const Lane& o, R& ring, Vec<1> rate) {
  using C = Cells<1, L>;
  Vec<1> A = splat<1>(1.0f), E = splat<1>(0.0f);
  using In = LoadedMap<T, 1, L>;
  backward_walk<T, 1, L, kMask, In>(p, o, ring, [&](int, In& in, auto) {
    if (in.q.live != (1u << L) - 1) blank(in.rg, in.q, kShut), blank(in.dy, in.q);
    const unsigned cut = cuts<kMask>(p, in.q);
    typename C::Array r, a, w;
    C::widen(in.rg, a);
    sigmoids(a, r);
    Vec<C::N> k;
#pragma unroll
    for (int j = 0; j < C::N; ++j) k.v[j] = rate.v[0];
    decays<kFar>(r, k, a, w);
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      Vec<1> al = C::at(a, l);
      if (kMask && ((cut >> l) & 1u)) al = splat<1>(0.0f);
      E = apply<kMask>(al, E + widen<1>(in.dy[l], 0), splat<1>(0.0f));
      A = chain<kMask>(al, A);
    }
  });
  join_maps<kMask>(p, o, A, E);
}

template <class T, int V, int L, bool kBulk, bool kMaps>
__device__ __forceinline__ auto backward_ring(const Args& p, const Maps& m, const Lane& o) {
  if constexpr (kBulk) {
    extern __shared__ __align__(128) char dynamic[];
    __shared__ uint64_t s_bar[kStrips * kRing<T>];
    Ring<T, V, L, kMaps ? 2 : 4, !kMaps, !kMaps> ring(dynamic, s_bar);
    ring.map[0] = &m.rg, ring.out = m.out;
    if constexpr (kMaps)
      ring.map[1] = &m.dy;
    else
      ring.map[1] = &m.ig, ring.map[2] = &m.x, ring.map[3] = &m.dy;
    ring.start(p, o, o.first + o.count - 1, o.count, -1);
    return ring;
  } else {
    return NoRing{};
  }
}

template <class T, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kStrips) backward_maps_kernel(const __grid_constant__ Args p,
                                                                     const __grid_constant__ Maps m) {
  let_next_start();
  const Lane o = lane_of<1, L, kMask, true>(p);
  auto ring = backward_ring<T, 1, L, kBulk, true>(p, m, o);
  Vec<1> rate;
  if (rates<1>(p, o, rate))
    backward_maps<T, L, kMask, true>(p, o, ring, rate);
  else
    backward_maps<T, L, kMask, false>(p, o, ring, rate);
}

// With e = a g (see above) everything but g is known before the carry comes in:
//   dx = g P1, dinput_gate = dx P2, s = g R1, ddecay_gate = s R2,
//   P1 = beta i, P2 = x (1 - i), R1 = r (a h_{t-1} - (a / beta)^2 b), R2 = rate (r - 1),
// with b = beta i x, and s sums up to the decay gradient.
template <class T, int V, int L, bool kMask, bool kFar, bool kFull, class R>
__device__ __forceinline__ void backward_chunk(const Args& p, const Lane& o, const R& ring, int k,
                                               LoadedBack<T, V, L>& in, Vec<V> rate, Vec<V>& e, Vec<Cells<V, L>::N>& acc) {
  using C = Cells<V, L>;
  constexpr int N = C::N, G = C::G;
  const Vec<N> minus = splat<N>(-1.0f);
  if (in.q.live != (1u << L) - 1)
    blank(in.rg, in.q, kShut), blank(in.ig, in.q), blank(in.x, in.q), blank(in.dy, in.q);
  Gates<N, G> q;
  gates_of<T, V, L, kMask, kFar>(cuts<kMask>(p, in.q), in.ig, in.rg, rate, q);
  typename C::Array b, p1, p2, r1, r2, ah, g;
  C::widen(in.x, p2);
  Vec<N> fast;
#pragma unroll
  for (int j = 0; j < N; ++j) fast.v[j] = rate.v[j % V];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const Vec<N> ix = q.i[i] * p2[i], u = q.a[i] * q.s[i];
    b[i] = q.beta[i] * ix;
    p1[i] = q.beta[i] * q.i[i];
    p2[i] = fma(ix, minus, p2[i]);
    r1[i] = u * (u * b[i]);  // (where beta is zero, b is: the term is dropped)
    r2[i] = fast * (q.r[i] + minus);
  }
  Vec<V> h = in.h;
#pragma unroll
  for (int l = 0; l < L; ++l) {
    C::put(ah, l, apply<kMask>(C::at(q.a, l), h, splat<V>(0.0f)));
    h = apply<kMask>(C::at(q.a, l), h, C::at(b, l));
  }
#pragma unroll
  for (int i = 0; i < G; ++i) r1[i] = q.r[i] * fma(r1[i], minus, ah[i]);
  if (kMask) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      Vec<V> d = C::at(r1, l);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (C::at(q.a, l).v[v] == 0.0f || !((in.q.live >> l) & 1u)) d.v[v] = 0.0f;
      C::put(r1, l, d);
    }
  }
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
    const Vec<V> now = e + widen<V>(in.dy[l], 0);
    e = apply<kMask>(C::at(q.a, l), now, splat<V>(0.0f));
    C::put(g, l, now);
  }
  // dx, dinput_gate, ddecay_gate take the places of p1, p2, r2
#pragma unroll
  for (int i = 0; i < G; ++i) {
    p1[i] = g[i] * p1[i];
    Vec<N> s = g[i] * r1[i];
    if (kMask) {  // (a gradient, or a reset's decay gate, that is not finite is not spread to where nothing flows)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int l = V == N ? i : i * N + j;
        if (!((in.q.live >> l) & 1u)) p1[i].v[j] = 0.0f;
        if (r1[i].v[j] == 0.0f) s.v[j] = 0.0f, r2[i].v[j] = 0.0f;
      }
    }
    p2[i] = p1[i] * p2[i];
    acc = acc + s;
    r2[i] = s * r2[i];
  }
  if constexpr (R::kStaged && kFull) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      ring.put(p, in.stage, 2, l, C::at(p1, l));
      ring.put(p, in.stage, 1, l, C::at(p2, l));
      ring.put(p, in.stage, 0, l, C::at(r2, l));
    }
    ring.template leave<0>(p, o, k, in.stage);
    return;
  }
  if (!o.on) return;
  const int64_t first = (o.b * p.steps + in.q.t0) * p.width + o.c;
  const int step = o.dir * (int)p.width * (int)sizeof(T);
  char *px = reinterpret_cast<char*>(static_cast<T*>(p.dx) + first),
       *pi = reinterpret_cast<char*>(static_cast<T*>(p.dig) + first),
       *pr = reinterpret_cast<char*>(static_cast<T*>(p.drg) + first);
#pragma unroll
  for (int l = 0; l < L; ++l)
    if (kFull || ((in.q.inside >> l) & 1u)) {
      const int64_t at = (int64_t)step * l;
      store<T>(px + at, C::at(p1, l));
      store<T>(pi + at, C::at(p2, l));
      store<T>(pr + at, C::at(r2, l));
    }
}

template <class T, int V, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void backward_strip(const Args& p, const Lane& o, R& ring, Vec<V> rate) {
  using C = Cells<V, L>;
  Vec<V> e = splat<V>(0.0f);
  Vec<C::N> acc = splat<C::N>(0.0f);
  if (p.dlast) e = read_row<V>(p.dlast + o.b * p.width + o.from);
  if constexpr (V == 1) {
    if (p.strips > 1) wait_for_last();
    if (o.rank >= p.strips) return;
    start_of<kMask>(p, o, e);
  }
  using In = LoadedBack<T, V, L>;
  if (!backward_walk<T, V, L, kMask, In>(p, o, ring, [&](int k, In& in, auto full) {
        backward_chunk<T, V, L, kMask, kFar, decltype(full)::value>(p, o, ring, k, in, rate, e, acc);
      }))
    return;
  if (kMask) zero_rest<T, V, L, 3>(p, o, {p.dx, p.dig, p.drg});
  if (!o.on) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (o.rank == p.strips - 1 && p.dstate) p.dstate[o.b * p.width + o.c + v] = e.v[v];
    p.dpart[(o.b * p.strips + o.rank) * p.width + o.c + v] = V == C::N ? acc.v[v] : acc.v[0] + acc.v[C::N - 1];
  }
}

template <class T, int V, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(L == 1   ? 32 * kStrips
                                  : V == 2 ? 32
                                           : 32 * backward_strips(kBulk, kMask, sizeof(T)),
                                  L == 1   ? 2
                                  : V == 2 ? (kBulk ? 12 : 8)
                                           : backward_ctas(backward_strips(kBulk, kMask, sizeof(T)), kBulk, kMask, sizeof(T)))
    backward_kernel(const __grid_constant__ Args p, const __grid_constant__ Maps m) {
  let_next_start();
  const Lane o = lane_of<V, L, kMask, true>(p);
  auto ring = backward_ring<T, V, L, kBulk, false>(p, m, o);
  Vec<V> rate;
  if (rates<V>(p, o, rate))
    backward_strip<T, V, L, kMask, true>(p, o, ring, rate);
  else
    backward_strip<T, V, L, kMask, false>(p, o, ring, rate);
}

struct Geometry {
  int vec, chunk, ctiles, strips, strip, warps;
  bool bulk;
  bool row;  // the strips of a row are one CTA's, and are held by it (forward)
};

template <class T>
cudaError_t launch(const Args& p, const Maps& m, const Geometry& g, bool backward, bool mask, cudaStream_t s);

}  // namespace gscan
}  // namespace pesq
