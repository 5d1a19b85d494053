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
// so a chunk's gates are worked out side by side, while the elements of the chunks
// to come are on their way.  Warps wait for nobody but their own copies: no flag, no
// atomic, and the order of every operation is fixed.
//
// Elements come in two ways.  Where channels and strides allow (multiples of 16
// bytes), a warp's chunks are boxes of 64 channels x 8 steps, or 32 x 16, that tensor copies bring to
// a ring in shared memory: one instruction for a box, no registers held.  Otherwise every lane loads its own elements a chunk ahead.
//
// With rows and channels enough to fill the device a strip is the whole row,
// and the data pass once.  Otherwise rows are cut into strips: the recurrence is
// the composition of maps h -> A h + H, a first kernel (`maps`) works out every
// strip's (A, H), and the second starts each strip from the state that the maps
// before it give.  The strips of a CTA meet in shared memory, so a strip composes
// the maps of the CTAs before its own and one more.
//
// Backward.  With g_t = dL/dh_t: g_t = dy_t + a_{t+1} g_{t+1}, the same kind of
// scan from the end of the row, carried as e_t = a_t g_t.  Then
//   dx = g beta i,   dinput_gate = dx x (1 - i),
//   dlog a = g (a h_{t-1} - (a^2 / beta) i x),   ddecay_gate = dlog a log a (1 - r),
//   ddecay = -rate sigmoid(decay) sum over rows and steps of dlog a r.
// h is not read back from the rounded y: the forward keeps the state before every
// chunk in 32 bits (1 / 8 or 1 / 16 of the elements), and the backward recomputes the
// chunk from it.  beta -> 0 only together with log a, whose quotient goes to
// zero: the term is dropped there.
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
constexpr int kStrips = 8;  // strips (warps) of a CTA at most, where rows are cut
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
  float* kept;                // state before every chunk, [batch][chunk][width]
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

// Tensor maps of the streams: [batch][step][channel], boxes of a chunk
struct Maps {
  CUtensorMap rg, ig, x, dy;
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

// logits are held at kShut so that the product below stays finite
// (sigmoid(-43) = 2e-19)
constexpr float kShut = -43.0f;
// 1 - a^2 is held above this where its root is divided by
constexpr float kTiny = 1e-36f;
// rates -log a up to here go by the series alone
constexpr float kNear = 0.25f;

template <int N>
struct Gates {
  Vec<N> i, r, a;
};

// The gates of G Vecs side by side: operation by operation rather than Vec by
// Vec, so that every instruction has G independent ones next to it.
//
// k = rate softplus(decay) >= 0.  The two sigmoids share one reciprocal.
// With m = -log a = k r, 1 - a = m (1 - m/2 + m^2/6 - ...) by its Taylor
// series (m^6 / 5040 < 5e-8 at 1/4): a is then rounded once, without the bias
// that a long memory would sum up, and 1 - a^2 = (1 - a)(2 - (1 - a)) does not
// cancel.  kFar: m may be above kNear, where the exponential takes over.
template <bool kFar, int N, int G>
__device__ __forceinline__ void decays(const Vec<N> (&r)[G], const Vec<N> (&k)[G], Vec<N> (&a)[G], Vec<N> (&w)[G]) {
  Vec<N> m[G], p[G];
  constexpr float kSeries[5] = {1.0f / 120, -1.0f / 24, 1.0f / 6, -0.5f, 1.0f};
#pragma unroll
  for (int g = 0; g < G; ++g) m[g] = k[g] * r[g];
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

template <bool kFar, int N, int G>
__device__ __forceinline__ void gates(const Vec<N> (&ig)[G], const Vec<N> (&rg)[G], const Vec<N> (&k)[G],
                                      Gates<N> (&out)[G], Vec<N> (&beta)[G]) {
  Vec<N> di[G], dr[G], q[G], r[G], a[G], w[G];
#pragma unroll
  for (int g = 0; g < G; ++g) di[g] = ig[g] * splat<N>(-kLog2e), dr[g] = rg[g] * splat<N>(-kLog2e);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) di[g].v[j] = exp2_approx(di[g].v[j]), dr[g].v[j] = exp2_approx(dr[g].v[j]);
#pragma unroll
  for (int g = 0; g < G; ++g) di[g] = di[g] + splat<N>(1.0f), dr[g] = dr[g] + splat<N>(1.0f);
#pragma unroll
  for (int g = 0; g < G; ++g) q[g] = di[g] * dr[g];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) q[g].v[j] = rcp_approx(q[g].v[j]);
#pragma unroll
  for (int g = 0; g < G; ++g) r[g] = q[g] * di[g];
#pragma unroll
  for (int g = 0; g < G; ++g) di[g] = q[g] * dr[g];
  decays<kFar>(r, k, a, w);
  Vec<N> s[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) s[g].v[j] = rsqrt_approx(fmaxf(w[g].v[j], kTiny));
#pragma unroll
  for (int g = 0; g < G; ++g) {
    beta[g] = w[g] * s[g];
    out[g].i = di[g], out[g].r = r[g], out[g].a = a[g];
  }
}

// The decays alone
template <bool kFar, int N, int G>
__device__ __forceinline__ void decays_of(const Vec<N> (&rg)[G], const Vec<N> (&k)[G], Vec<N> (&a)[G]) {
  Vec<N> r[G], w[G];
#pragma unroll
  for (int g = 0; g < G; ++g) r[g] = rg[g] * splat<N>(-kLog2e);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) r[g].v[j] = exp2_approx(r[g].v[j]);
#pragma unroll
  for (int g = 0; g < G; ++g) r[g] = r[g] + splat<N>(1.0f);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < N; ++j) r[g].v[j] = rcp_approx(r[g].v[j]);
  decays<kFar>(r, k, a, w);
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

// logits at least kShut (a NaN stays)
__device__ __forceinline__ void hold(Pack<float, 1>& p) { p.v[0] = max_nan(p.v[0], kShut); }
__device__ __forceinline__ void hold(Pack<__nv_bfloat16, 1>& p) {
  p.v[0] = __hmax_nan(p.v[0], __float2bfloat16_rn(kShut));
}
__device__ __forceinline__ void hold(Pack<__half, 1>& p) { p.v[0] = __hmax_nan(p.v[0], __float2half_rn(kShut)); }
template <int V>
__device__ __forceinline__ void hold(Pack<float, V>& p) {
#pragma unroll
  for (int v = 0; v < V; ++v) p.v[v] = max_nan(p.v[v], kShut);
}
template <int V>
__device__ __forceinline__ void hold(Pack<__nv_bfloat16, V>& p) {
  __nv_bfloat162* q = reinterpret_cast<__nv_bfloat162*>(&p);
#pragma unroll
  for (int v = 0; v < V / 2; ++v) q[v] = __hmax2_nan(q[v], __float2bfloat162_rn(kShut));
}
template <int V>
__device__ __forceinline__ void hold(Pack<__half, V>& p) {
  __half2* q = reinterpret_cast<__half2*>(&p);
#pragma unroll
  for (int v = 0; v < V / 2; ++v) q[v] = __hmax2_nan(q[v], __float2half2_rn(kShut));
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
  const unsigned block = blockIdx.x / p.ctiles;  // CTA along the row
  o.c = (int64_t)(blockIdx.x - block * p.ctiles) * (32 * V) + threadIdx.x * V;
  o.on = o.c < p.width;
  o.from = o.on ? o.c : 0;
  o.rank = block * blockDim.y + threadIdx.y;
  const int strip = kBack ? p.strips - 1 - o.rank : o.rank, steps = (int)p.steps;
  const int all = (steps + L - 1) / L;
  int per = p.strip / L;
  o.lo = 0, o.hi = all;
  o.len = steps;
  o.dir = p.reverse ? -1 : 1;
  if (kMask && p.lengths) {
    o.len = (int)max(INT64_C(0), min(p.lengths[o.b], p.steps));
    o.lo = p.reverse ? (steps - o.len) / L : 0;
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
template <class T, int V, int N>
__device__ __forceinline__ void store(void* p, const Vec<N> (&val)[V / N]) {
  Pack<T, V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.v[v] = narrow<T>(val[v / N].v[v % N]);
  *static_cast<Pack<T, V>*>(p) = o;
}

// How L x V elements are paired for the two-wide instructions: by channel, or by
// step where a lane has a single channel.
template <int V, int L>
struct Pairing {
  static constexpr int N = V > 1 ? 2 : 1;  // channels of a Vec
  static constexpr int P = V / N;          // Vecs of a step
  static constexpr bool kBySteps = V == 1 && L % 2 == 0;
};

// Calls emit(l, j, gates, beta) for every step and Vec of a chunk, steps in order
template <class T, int V, int L, bool kMask, bool kFar, class F>
__device__ __forceinline__ void each_gate(unsigned cut, const Pack<T, V> (&ig)[L], const Pack<T, V> (&rg)[L],
                                          const Vec<Pairing<V, L>::N> (&rate)[Pairing<V, L>::P], F emit) {
  using Q = Pairing<V, L>;
  constexpr int N = Q::N;
  if constexpr (Q::kBySteps) {
    constexpr int G = L / 2;
    Vec<2> i2[G], r2[G], k2[G], beta[G];
    Gates<2> out[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      Pack<T, 2> r{{rg[2 * g].v[0], rg[2 * g + 1].v[0]}}, i{{ig[2 * g].v[0], ig[2 * g + 1].v[0]}};
      hold(r), hold(i);
      i2[g] = widen<2>(i, 0), r2[g] = widen<2>(r, 0), k2[g] = splat<2>(rate[0].v[0]);
    }
    gates<kFar>(i2, r2, k2, out, beta);
#pragma unroll
    for (int l = 0; l < L; ++l) {
      Gates<1> one{{{out[l / 2].i.v[l % 2]}}, {{out[l / 2].r.v[l % 2]}}, {{out[l / 2].a.v[l % 2]}}};
      Vec<1> b1{{beta[l / 2].v[l % 2]}};
      if (kMask && ((cut >> l) & 1u)) one.a = splat<1>(0.0f), b1 = splat<1>(1.0f);
      emit(l, 0, one, b1);
    }
  } else {
    constexpr int G = L * Q::P;
    Vec<N> i2[G], r2[G], k2[G], beta[G];
    Gates<N> out[G];
#pragma unroll
    for (int l = 0; l < L; ++l) {
      Pack<T, V> r = rg[l], i = ig[l];
      hold(r), hold(i);
#pragma unroll
      for (int j = 0; j < Q::P; ++j)
        i2[l * Q::P + j] = widen<N>(i, j), r2[l * Q::P + j] = widen<N>(r, j), k2[l * Q::P + j] = rate[j];
    }
    gates<kFar>(i2, r2, k2, out, beta);
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int j = 0; j < Q::P; ++j) {
        Gates<N>& one = out[l * Q::P + j];
        if (kMask && ((cut >> l) & 1u)) one.a = splat<N>(0.0f), beta[l * Q::P + j] = splat<N>(1.0f);
        emit(l, j, one, beta[l * Q::P + j]);
      }
  }
}

// The rates of a lane's channels, and whether one of the warp's is above kNear
template <int V, int N>
__device__ __forceinline__ bool rates(const Args& p, const Lane& o, Vec<N> (&rate)[V / N]) {
  bool far = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float k = o.on ? p.rate * softplus(p.decay[o.c + v]) : 0.0f;
    rate[v / N].v[v % N] = k;
    far = far || !(k < kNear);
  }
  return __any_sync(0xffffffffu, far);
}

template <int V, int N>
__device__ __forceinline__ void read_row(const float* p, Vec<N> (&out)[V / N]) {
#pragma unroll
  for (int v = 0; v < V; ++v) out[v / N].v[v % N] = p[v];
}

// Start value of a strip: the row's, through the maps of the CTAs before and of
// the strips before in the CTA
template <int V, int N, bool kMask>
__device__ __forceinline__ void start_of(const Args& p, const Lane& o, Vec<N> (&h)[V / N]) {
  if (p.strips == 1 || !o.on || o.rank >= p.strips) return;
  const int w = blockDim.y, ctas = (p.strips + w - 1) / w, cta = o.rank / w;
  const float2* t = p.total + o.b * ctas * p.width + o.c;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Vec<1> s{{h[v / N].v[v % N]}};
#pragma unroll 8
    for (int k = 0; k < cta; ++k) {
      const float2 m = t[k * p.width + v];
      s = apply<kMask>(Vec<1>{{m.x}}, s, Vec<1>{{m.y}});
    }
    const float2 m = p.before[(o.b * p.strips + o.rank) * p.width + o.c + v];
    h[v / N].v[v % N] = apply<kMask>(Vec<1>{{m.x}}, s, Vec<1>{{m.y}}).v[0];
  }
}

// The maps of a CTA's strips, warp by warp: leaves in `before` what the strips
// before each make of a state, and in `total` all of them.
template <int V, int N, bool kMask>
__device__ __forceinline__ void join_maps(const Args& p, const Lane& o, const Vec<N> (&A)[V / N], const Vec<N> (&H)[V / N]) {
  __shared__ float2 s_map[kStrips][32 * V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    s_map[threadIdx.y][threadIdx.x * V + v] = make_float2(A[v / N].v[v % N], H[v / N].v[v % N]);
  __syncthreads();
  if (!o.on || o.rank >= p.strips) return;
  const int strips = blockDim.y;
  const bool end = threadIdx.y == strips - 1 || o.rank == p.strips - 1;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Vec<1> a{{1.0f}}, h{{0.0f}};
    for (int w = 0; w < (int)threadIdx.y; ++w) {
      const float2 m = s_map[w][threadIdx.x * V + v];
      h = apply<kMask>(Vec<1>{{m.x}}, h, Vec<1>{{m.y}});
      a.v[0] *= m.x;
    }
    p.before[(o.b * p.strips + o.rank) * p.width + o.c + v] = make_float2(a.v[0], h.v[0]);
    if (end) {
      const float2 m = s_map[threadIdx.y][threadIdx.x * V + v];
      h = apply<kMask>(Vec<1>{{m.x}}, h, Vec<1>{{m.y}});
      const int ctas = (p.strips + strips - 1) / strips;
      p.total[(o.b * ctas + o.rank / strips) * p.width + o.c + v] = make_float2(a.v[0] * m.x, h.v[0]);
    }
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
  const int s0 = (base + o.rank * per) * L, s1 = min((int)p.steps, min(base + dead, base + (o.rank + 1) * per) * L);
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
// [L][32 V] and, with kState, the states before the chunk.
template <class T, int V, int L, int S, bool kState>
struct Ring {
  static constexpr int kBox = L * 32 * V * (int)sizeof(T);
  static constexpr int kStage = S * kBox + (kState ? 128 * V : 0);
  static constexpr int kBytes = kRing<T> * kStage;  // of a warp
  char* base;
  uint64_t* bar;
  const CUtensorMap* map[S];

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
      bulk_g2s(to + S * kBox, p.kept + (o.b * ((p.steps + L - 1) / L) + k) * p.width + o.c, state, bar + stage);
  }
  // one stream of the stage, in scan order
  __device__ __forceinline__ void get(const Args& p, int stage, int i, Pack<T, V> (&out)[L]) const {
    const Pack<T, V>* s = reinterpret_cast<const Pack<T, V>*>(base + stage * kStage + i * kBox) + threadIdx.x;
    const int step = p.reverse ? -32 : 32;
    s += p.reverse ? (L - 1) * 32 : 0;
#pragma unroll
    for (int l = 0; l < L; ++l) out[l] = s[l * step];
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
      read(stage, in);
      __syncwarp();
      if (threadIdx.x == 0 && k + kRing<T> < n) send(p, o, first + way * (k + kRing<T>), stage);
      q = chunk_of<L, kMask>(p, o, first + way * min(k + 1, n - 1));
      flag_chunk<L, kMask>(p, o, q);
      work(first + way * k, in);
      if (++stage == kRing<T>) stage = 0, parity ^= 1;
    }
    if (!ok) {  // nothing may be in flight to shared memory that another block gets
      if (threadIdx.x == 0) atomicOr(p.error, 1u);
      for (int i = 0; i < kRing<T>; ++i) mbar_wait(bar + i, i < stage ? parity ^ 1 : parity);
    }
    return ok;
  }
};
// a warp without a ring, where every lane loads its own
struct NoRing {};

// ------------------------------------------------------------------- forward

template <class T, int V, int L>
struct Loaded {
  Chunk q;
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

template <class T, int V, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void forward_maps(const Args& p, const Lane& o, R& ring,
                                             const Vec<Pairing<V, L>::N> (&rate)[Pairing<V, L>::P]) {
  using Q = Pairing<V, L>;
  constexpr int N = Q::N, P = Q::P;
  Vec<N> A[P], H[P];
#pragma unroll
  for (int j = 0; j < P; ++j) A[j] = splat<N>(1.0f), H[j] = splat<N>(0.0f);
  forward_walk<T, V, L, kMask>(p, o, ring, [&](int, Loaded<T, V, L>& in, auto) {
    if (in.q.live != (1u << L) - 1) blank(in.rg, in.q, kShut), blank(in.ig, in.q), blank(in.x, in.q);
    each_gate<T, V, L, kMask, kFar>(
        cuts<kMask>(p, in.q), in.ig, in.rg, rate, [&](int l, int j, const Gates<N>& g, Vec<N> beta) {
          H[j] = apply<kMask>(g.a, H[j], beta * (g.i * widen<N>(in.x[l], j)));
          A[j] = A[j] * g.a;
        });
  });
  join_maps<V, N, kMask>(p, o, A, H);
}

// The ring of a forward warp, with its first copies on their way
template <class T, int V, int L, bool kBulk>
__device__ __forceinline__ auto forward_ring(const Args& p, const Maps& m, const Lane& o) {
  if constexpr (kBulk) {
    extern __shared__ __align__(128) char dynamic[];
    __shared__ uint64_t s_bar[kRowWarps * kRing<T>];
    Ring<T, V, L, 3, false> ring(dynamic, s_bar);
    ring.map[0] = &m.rg, ring.map[1] = &m.ig, ring.map[2] = &m.x;
    ring.start(p, o, o.first, o.count, 1);
    return ring;
  } else {
    return NoRing{};
  }
}

template <class T, int V, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kStrips) forward_maps_kernel(const __grid_constant__ Args p,
                                                                    const __grid_constant__ Maps m) {
  using Q = Pairing<V, L>;
  let_next_start();
  const Lane o = lane_of<V, L, kMask, false>(p);
  auto ring = forward_ring<T, V, L, kBulk>(p, m, o);
  Vec<Q::N> rate[Q::P];
  // (the CTA's warps share their channels, so they agree, and meet in join_maps)
  if (rates<V, Q::N>(p, o, rate))
    forward_maps<T, V, L, kMask, true>(p, o, ring, rate);
  else
    forward_maps<T, V, L, kMask, false>(p, o, ring, rate);
}

template <class T, int V, int L, bool kMask, bool kFar, bool kFull>
__device__ __forceinline__ void forward_chunk(const Args& p, const Lane& o, int k, Loaded<T, V, L>& in,
                                              const Vec<Pairing<V, L>::N> (&rate)[Pairing<V, L>::P],
                                              Vec<Pairing<V, L>::N> (&h)[Pairing<V, L>::P]) {
  using Q = Pairing<V, L>;
  constexpr int N = Q::N, P = Q::P;
  if (p.kept && o.on) {
    float* keep = p.kept + (o.b * ((p.steps + L - 1) / L) + k) * p.width + o.c;
#pragma unroll
    for (int v = 0; v < V; ++v) keep[v] = h[v / N].v[v % N];
  }
  if (in.q.live != (1u << L) - 1) blank(in.rg, in.q, kShut), blank(in.ig, in.q), blank(in.x, in.q);
  char* y = reinterpret_cast<char*>(static_cast<T*>(p.y) + (o.b * p.steps + in.q.t0) * p.width + o.c);
  const int step = o.dir * (int)p.width * (int)sizeof(T);
  Vec<N> out[P];
  each_gate<T, V, L, kMask, kFar>(
      cuts<kMask>(p, in.q), in.ig, in.rg, rate, [&](int l, int j, const Gates<N>& g, Vec<N> beta) {
        h[j] = apply<kMask>(g.a, h[j], beta * (g.i * widen<N>(in.x[l], j)));
        out[j] = !kMask || ((in.q.live >> l) & 1u) ? h[j] : splat<N>(0.0f);
        if (j == P - 1 && o.on && (kFull || ((in.q.inside >> l) & 1u))) store<T, V, N>(y + (int64_t)step * l, out);
      });
}

template <class T, int V, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void forward_strip(const Args& p, const Lane& o, R& ring,
                                              const Vec<Pairing<V, L>::N> (&rate)[Pairing<V, L>::P]) {
  using Q = Pairing<V, L>;
  constexpr int N = Q::N, P = Q::P;
  Vec<N> h[P];
#pragma unroll
  for (int j = 0; j < P; ++j) h[j] = splat<N>(0.0f);
  if (p.state) read_row<V, N>(p.state + o.b * p.width + o.from, h);
  if (p.strips > 1) wait_for_last();
  if (o.rank >= p.strips) return;
  start_of<V, N, kMask>(p, o, h);
  if (!forward_walk<T, V, L, kMask>(p, o, ring, [&](int k, Loaded<T, V, L>& in, auto full) {
        forward_chunk<T, V, L, kMask, kFar, decltype(full)::value>(p, o, k, in, rate, h);
      }))
    return;
  if (kMask) zero_rest<T, V, L, 1>(p, o, {p.y});
  if (o.rank == p.strips - 1 && o.on) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.last[o.b * p.width + o.c + v] = h[v / N].v[v % N];
  }
}

template <class T, int V, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kStrips) forward_kernel(const __grid_constant__ Args p,
                                                               const __grid_constant__ Maps m) {
  using Q = Pairing<V, L>;
  const Lane o = lane_of<V, L, kMask, false>(p);
  auto ring = forward_ring<T, V, L, kBulk>(p, m, o);
  Vec<Q::N> rate[Q::P];
  if (rates<V, Q::N>(p, o, rate))
    forward_strip<T, V, L, kMask, true>(p, o, ring, rate);
  else
    forward_strip<T, V, L, kMask, false>(p, o, ring, rate);
}

// A short row in one CTA: a warp holds its strip of kHeld steps as (a, b) in registers,
// the strips' maps meet in shared memory, and the recursion is run from the state that
// they give.  The data pass once, in one launch.
template <class T, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void forward_row(const Args& p, const Lane& o, R& ring, const Vec<1> (&rate)[1]) {
  constexpr int NC = kHeld / L;
  __shared__ float2 s_map[kRowWarps][32];
  Vec<1> a[NC][L], b[NC][L], A{{1.0f}}, H{{0.0f}};
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
    for (int l = 0; l < L; ++l) a[c][l] = splat<1>(1.0f), b[c][l] = splat<1>(0.0f);
    if (c >= o.count) continue;
    In& now = in[c % 2];
    if constexpr (std::is_same<R, NoRing>::value) {
      if (c + 1 < NC && c + 1 < o.count) in[(c + 1) % 2].template read<kMask, false>(p, o, o.first + c + 1);
    } else {
      now.q = chunk_of<L, kMask>(p, o, o.first + c);
      flag_chunk<L, kMask>(p, o, now.q);
      ok = ok && __all_sync(0xffffffffu, mbar_wait(ring.bar + c, 0));
      now.get(p, ring, c);
    }
    if (now.q.live != (1u << L) - 1) blank(now.rg, now.q, kShut), blank(now.ig, now.q), blank(now.x, now.q);
    live[c] = now.q.live;
    each_gate<T, 1, L, kMask, kFar>(
        cuts<kMask>(p, now.q), now.ig, now.rg, rate, [&](int l, int, const Gates<1>& g, Vec<1> beta) {
          a[c][l] = g.a;
          b[c][l] = beta * (g.i * widen<1>(now.x[l], 0));
          H = apply<kMask>(g.a, H, b[c][l]);
          A = A * g.a;
        });
  }
  if (!ok && threadIdx.x == 0) atomicOr(p.error, 1u);
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
    if (p.kept) p.kept[(o.b * ((p.steps + L - 1) / L) + o.first + c) * p.width + o.c] = h.v[0];
    char* y = reinterpret_cast<char*>(static_cast<T*>(p.y) + (o.b * p.steps + q.t0) * p.width + o.c);
    const int step = o.dir * (int)p.width * (int)sizeof(T);
#pragma unroll
    for (int l = 0; l < L; ++l) {
      h = apply<kMask>(a[c][l], h, b[c][l]);
      const Vec<1> out[1] = {!kMask || ((live[c] >> l) & 1u) ? h : splat<1>(0.0f)};
      if ((q.inside >> l) & 1u) store<T, 1, 1>(y + (int64_t)step * l, out);
    }
  }
  if (kMask) zero_rest<T, 1, L, 1>(p, o, {p.y});
  if (o.rank == p.strips - 1) p.last[o.b * p.width + o.c] = h.v[0];
}

template <class T, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kRowWarps) forward_row_kernel(const __grid_constant__ Args p,
                                                                     const __grid_constant__ Maps m) {
  const Lane o = lane_of<1, L, kMask, false>(p);
  auto ring = forward_ring<T, 1, L, kBulk>(p, m, o);
  Vec<1> rate[1];
  if (rates<1, 1>(p, o, rate))
    forward_row<T, L, kMask, true>(p, o, ring, rate);
  else
    forward_row<T, L, kMask, false>(p, o, ring, rate);
}

// ------------------------------------------------------------------ backward

template <class T, int V, int L>
struct LoadedMap {
  Chunk q;
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
  Pack<T, V> x[L], ig[L], rg[L], dy[L];
  Vec<Pairing<V, L>::N> h[Pairing<V, L>::P];  // state before the chunk
  template <class R>
  __device__ __forceinline__ void get(const Args& p, const R& ring, int stage) {
    ring.get(p, stage, 0, rg);
    ring.get(p, stage, 1, ig);
    ring.get(p, stage, 2, x);
    ring.get(p, stage, 3, dy);
    const Pack<float, V> s = ring.state(stage);
#pragma unroll
    for (int j = 0; j < Pairing<V, L>::P; ++j) h[j] = widen<Pairing<V, L>::N>(s, j);
  }
  template <bool kMask, bool kFull>
  __device__ __forceinline__ void read(const Args& p, const Lane& o, int k) {
    q = chunk_of<L, kMask>(p, o, k);
    flag_chunk<L, kMask>(p, o, q);
    load<T, V, L, kFull>(rg, p.rg, o, q, kShut);
    load<T, V, L, kFull>(ig, p.ig, o, q);
    load<T, V, L, kFull>(x, p.x, o, q);
    load<T, V, L, kFull>(dy, p.dy, o, q);
    read_row<V, Pairing<V, L>::N>(p.kept + (o.b * ((p.steps + L - 1) / L) + k) * p.width + o.from, h);
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
            work(in, std::true_type{});
          else
            work(in, std::false_type{});
        });
  } else {
    if (o.whole < o.count) {
      In in;
      in.template read<kMask, false>(p, o, o.first + o.whole);
      work(in, std::false_type{});
    }
    walk<In>(
        o.whole, [&](int k, In& in) { in.template read<kMask, true>(p, o, o.first + o.whole - 1 - k); },
        [&](int, In& in) { work(in, std::true_type{}); });
    return true;
  }
}

// e -> A e + E of a strip, from its last step to its first: the decay gate and
// dy are all it takes
template <class T, int V, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void backward_maps(const Args& p, const Lane& o, R& ring,
                                              const Vec<Pairing<V, L>::N> (&rate)[Pairing<V, L>::P]) {
  using Q = Pairing<V, L>;
  constexpr int N = Q::N, P = Q::P;
  Vec<N> A[P], E[P];
#pragma unroll
  for (int j = 0; j < P; ++j) A[j] = splat<N>(1.0f), E[j] = splat<N>(0.0f);
  using In = LoadedMap<T, V, L>;
  backward_walk<T, V, L, kMask, In>(p, o, ring, [&](In& in, auto) {
    if (in.q.live != (1u << L) - 1) blank(in.rg, in.q, kShut), blank(in.dy, in.q);
    const unsigned cut = cuts<kMask>(p, in.q);
    Vec<N> rg[L * P], k2[L * P], a[L * P];
#pragma unroll
    for (int l = 0; l < L; ++l) {
      hold(in.rg[l]);
#pragma unroll
      for (int j = 0; j < P; ++j) rg[l * P + j] = widen<N>(in.rg[l], j), k2[l * P + j] = rate[j];
    }
    decays_of<kFar>(rg, k2, a);
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        Vec<N> al = a[l * P + j];
        if (kMask && ((cut >> l) & 1u)) al = splat<N>(0.0f);
        E[j] = apply<kMask>(al, E[j] + widen<N>(in.dy[l], j), splat<N>(0.0f));
        A[j] = A[j] * al;
      }
    }
  });
  join_maps<V, N, kMask>(p, o, A, E);
}

template <class T, int V, int L, bool kBulk, bool kMaps>
__device__ __forceinline__ auto backward_ring(const Args& p, const Maps& m, const Lane& o) {
  if constexpr (kBulk) {
    extern __shared__ __align__(128) char dynamic[];
    __shared__ uint64_t s_bar[kStrips * kRing<T>];
    Ring<T, V, L, kMaps ? 2 : 4, !kMaps> ring(dynamic, s_bar);
    ring.map[0] = &m.rg;
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

template <class T, int V, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kStrips) backward_maps_kernel(const __grid_constant__ Args p,
                                                                     const __grid_constant__ Maps m) {
  using Q = Pairing<V, L>;
  let_next_start();
  const Lane o = lane_of<V, L, kMask, true>(p);
  auto ring = backward_ring<T, V, L, kBulk, true>(p, m, o);
  Vec<Q::N> rate[Q::P];
  if (rates<V, Q::N>(p, o, rate))
    backward_maps<T, V, L, kMask, true>(p, o, ring, rate);
  else
    backward_maps<T, V, L, kMask, false>(p, o, ring, rate);
}

// With e = a g (see above) everything but g is known before the carry comes in:
//   dx = g P1, dinput_gate = dx P2, s = g R1, ddecay_gate = s R2,
//   P1 = beta i, P2 = x (1 - i), R1 = r (a h_{t-1} - (a^2 / beta) i x), R2 = rate (r - 1),
// and s sums up to the decay gradient.
template <class T, int V, int L, bool kMask, bool kFar, bool kFull>
__device__ __forceinline__ void backward_chunk(const Args& p, const Lane& o, LoadedBack<T, V, L>& in,
                                               const Vec<Pairing<V, L>::N> (&rate)[Pairing<V, L>::P],
                                               Vec<Pairing<V, L>::N> (&e)[Pairing<V, L>::P],
                                               Vec<Pairing<V, L>::N> (&acc)[Pairing<V, L>::P]) {
  using Q = Pairing<V, L>;
  constexpr int N = Q::N, P = Q::P;
  if (in.q.live != (1u << L) - 1)
    blank(in.rg, in.q, kShut), blank(in.ig, in.q), blank(in.x, in.q), blank(in.dy, in.q);
  Vec<N> a[L][P], p1[L][P], p2[L][P], r1[L][P], r2[L][P], h[P];
#pragma unroll
  for (int j = 0; j < P; ++j) h[j] = in.h[j];
  each_gate<T, V, L, kMask, kFar>(cuts<kMask>(p, in.q), in.ig, in.rg, rate, [&](int l, int j, const Gates<N>& g, Vec<N> beta) {
    const Vec<N> x = widen<N>(in.x[l], j);
    Vec<N> inverse;  // dropped with beta
#pragma unroll
    for (int i = 0; i < N; ++i) inverse.v[i] = beta.v[i] > kTiny ? -rcp_approx(beta.v[i]) : 0.0f;
    const Vec<N> ah = apply<kMask>(g.a, h[j], splat<N>(0.0f)), ix = g.i * x;
    Vec<N> d = fma(g.a * (g.a * inverse), ix, ah);
    if (kMask) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (g.a.v[i] == 0.0f || !((in.q.live >> l) & 1u)) d.v[i] = 0.0f;
    }
    a[l][j] = g.a;
    p1[l][j] = beta * g.i;
    p2[l][j] = fma(ix, splat<N>(-1.0f), x);
    r1[l][j] = g.r * d;
    r2[l][j] = rate[j] * (g.r + splat<N>(-1.0f));
    h[j] = fma(beta, ix, ah);
  });
  const int64_t first = (o.b * p.steps + in.q.t0) * p.width + o.c;
  const int step = o.dir * (int)p.width * (int)sizeof(T);
  char *px = reinterpret_cast<char*>(static_cast<T*>(p.dx) + first),
       *pi = reinterpret_cast<char*>(static_cast<T*>(p.dig) + first),
       *pr = reinterpret_cast<char*>(static_cast<T*>(p.drg) + first);
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
    Vec<N> dx[P], di[P], dr[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const Vec<N> g = e[j] + widen<N>(in.dy[l], j);
      e[j] = apply<kMask>(a[l][j], g, splat<N>(0.0f));
      dx[j] = g * p1[l][j];
      Vec<N> s = g * r1[l][j];
      if (kMask) {  // (a gradient that is not finite is not spread to where nothing flows)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (!((in.q.live >> l) & 1u)) dx[j].v[i] = 0.0f;
          if (r1[l][j].v[i] == 0.0f) s.v[i] = 0.0f;
        }
      }
      di[j] = dx[j] * p2[l][j];
      acc[j] = acc[j] + s;
      dr[j] = s * r2[l][j];
    }
    if (o.on && (kFull || ((in.q.inside >> l) & 1u))) {
      const int64_t at = (int64_t)step * l;
      store<T, V, N>(px + at, dx);
      store<T, V, N>(pi + at, di);
      store<T, V, N>(pr + at, dr);
    }
  }
}

template <class T, int V, int L, bool kMask, bool kFar, class R>
__device__ __forceinline__ void backward_strip(const Args& p, const Lane& o, R& ring,
                                               const Vec<Pairing<V, L>::N> (&rate)[Pairing<V, L>::P]) {
  using Q = Pairing<V, L>;
  constexpr int N = Q::N, P = Q::P;
  Vec<N> e[P], acc[P];
#pragma unroll
  for (int j = 0; j < P; ++j) e[j] = acc[j] = splat<N>(0.0f);
  if (p.dlast) read_row<V, N>(p.dlast + o.b * p.width + o.from, e);
  if (p.strips > 1) wait_for_last();
  if (o.rank >= p.strips) return;
  start_of<V, N, kMask>(p, o, e);
  using In = LoadedBack<T, V, L>;
  if (!backward_walk<T, V, L, kMask, In>(p, o, ring, [&](In& in, auto full) {
        backward_chunk<T, V, L, kMask, kFar, decltype(full)::value>(p, o, in, rate, e, acc);
      }))
    return;
  if (kMask) zero_rest<T, V, L, 3>(p, o, {p.dx, p.dig, p.drg});
  if (!o.on) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (o.rank == p.strips - 1 && p.dstate) p.dstate[o.b * p.width + o.c + v] = e[v / N].v[v % N];
    p.dpart[(o.b * p.strips + o.rank) * p.width + o.c + v] = acc[v / N].v[v % N];
  }
}

template <class T, int V, int L, bool kMask, bool kBulk>
__global__ void __launch_bounds__(32 * kStrips) backward_kernel(const __grid_constant__ Args p,
                                                                const __grid_constant__ Maps m) {
  using Q = Pairing<V, L>;
  let_next_start();
  const Lane o = lane_of<V, L, kMask, true>(p);
  auto ring = backward_ring<T, V, L, kBulk, false>(p, m, o);
  Vec<Q::N> rate[Q::P];
  if (rates<V, Q::N>(p, o, rate))
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
