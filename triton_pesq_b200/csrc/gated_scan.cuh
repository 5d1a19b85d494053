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
// The recurrence is the composition of maps h -> A h + H, so it splits over
// time: a tile is kTile = kWarps * L steps by 32 V channels.  Warp w of a CTA
// owns L consecutive steps of the tile, a lane V neighbouring channels of all
// of them, so a warp's access is one contiguous piece of a step.  Each
// thread reads its L x V elements of every stream once, forms (a, b) in
// registers and folds them to its (A, H); the warps' pairs meet in shared
// memory; the tiles of a row are chained by a look-back (below); the
// recursion is then run from the exact start state.  One pass over the data.
//
// Backward.  With g_t = dL/dh_t: g_t = dy_t + a_{t+1} g_{t+1}, the same kind of
// scan from the end of the row, carried as e_t = a_t g_t.  Then
//   dx = g beta i,   dinput_gate = dx x (1 - i),
//   dlog a = g (a h_{t-1} - (a^2 / beta) i x),   ddecay_gate = dlog a log a (1 - r),
//   ddecay = -rate sigmoid(decay) sum over rows and steps of dlog a r.
// h is not read back from the rounded y: each tile recomputes it from its
// start state, which the forward keeps in 32 bits (one value per channel and
// tile).  beta -> 0 only together with log a, whose quotient goes to zero: the
// term is dropped there.
//
// Look-back.  A tile publishes its (A, H) as soon as it has it and its end
// state once it knows its start state.  A tile walks back to the nearest
// predecessor whose end state is there and applies the pairs in between in
// time order, h <- A h + H -- the very operations the predecessors perform for
// their own end states, so the result does not depend, to the last bit, on how
// far it had to walk.  Tiles are claimed by a ticket, earliest steps first, so
// a predecessor is always running or done; the wait is bounded all the same
// (it sets the error word and goes on from zero).
#pragma once

#include "../../include/pesq_cuda.h"
#include "train.cuh"

namespace pesq {
namespace gscan {

using namespace train;

constexpr int kWarps = 8;
constexpr int kSteps = 8;                 // steps per thread (L) of a tiled row
constexpr int kTile = kWarps * kSteps;    // steps per tile
constexpr int kForwardCtas = 4;           // CTAs an SM holds: the registers a thread may use
constexpr int kBackwardCtas = 2;
constexpr uint32_t kSpinLimit = 1u << 21; // polls with a 64 ns pause: about 0.1 s

struct Stream {
  const void* p;
  int64_t sb, st;  // strides of batch and step, in elements
};

struct Args {
  Stream x, ig, rg, dy;
  const float* decay;
  const float* state;         // [batch, width] or null (zeros)
  const uint8_t* reset;
  int64_t reset_b, reset_t;
  const int64_t* lengths;
  int64_t batch, steps, width;
  int tiles;                  // per row
  int ctiles;                 // channel tiles
  int reverse;
  float rate;
  // look-back words, [batch][tile][width]
  unsigned long long* pair;   // (-A, H): the set sign bit is the tag
  unsigned long long* end;    // (1, end state)
  const unsigned long long* start;  // backward: the forward's `end` words
  unsigned* ticket;
  uint32_t* error;
  uint32_t spin_limit;
  // forward
  void* y;
  float* last;
  // backward
  const float* dlast;
  void *dx, *dig, *drg;
  float* dstate;
  float* dpart;               // [batch * tiles, width] sums of dlog a r
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

struct Gates {
  float i, r, a, w;  // w = 1 - a^2
};

// logits are held at kShut so that the product below stays finite
// (sigmoid(-43) = 2e-19)
constexpr float kShut = -43.0f;

// k = -rate softplus(decay).  The two sigmoids share one reciprocal.
__device__ __forceinline__ Gates gates(float ig, float rg, float k) {
  const float di = 1.0f + exp2_approx(max_nan(ig, kShut) * -kLog2e);
  const float dr = 1.0f + exp2_approx(max_nan(rg, kShut) * -kLog2e);
  const float q = rcp_approx(di * dr);
  Gates o;
  o.i = q * dr;
  o.r = q * di;
  const float la = k * o.r;
  // near zero u = a - 1 by its Taylor series (la^6 / 5040 < 5e-8 at 1/4): then
  // a = 1 + u is rounded once, without the bias that a long memory would sum
  // up, and 1 - a^2 = -u (2 + u) does not cancel
  float p = fmaf(la, 1.0f / 720, 1.0f / 120);
  p = fmaf(la, p, 1.0f / 24);
  p = fmaf(la, p, 1.0f / 6);
  p = fmaf(la, p, 0.5f);
  p = fmaf(la, p, 1.0f);
  const float u = la * p;
  o.a = 1.0f + u;
  o.w = -u * (2.0f + u);
  if (!(la > -0.25f)) {
    o.a = exp2_approx(la * kLog2e);
    o.w = fmaf(-o.a, o.a, 1.0f);
  }
  return o;
}

// A state that a = 0 cuts off is not looked at (it may be infinite or NaN)
template <bool kMask>
__device__ __forceinline__ float apply(float a, float h, float b) {
  if (kMask) h = a == 0.0f ? 0.0f : h;
  return fmaf(a, h, b);
}

// Start value of tile `tile` (>= 1 predecessors, nearest at `tile - dir`) of
// one channel: words at `pair`/`end` + k * pitch for the k-th tile back.
// `count` predecessors exist; the farthest always publishes its end value
// without waiting.
template <bool kMask>
__device__ float look_back(const Args& p, const unsigned long long* pair, const unsigned long long* end, int64_t pitch,
                           int count) {
  constexpr int kWin = 8;
  int done = 0;  // pairs nearer than this are all there
  unsigned polls = 0;
  float h = 0.0f;
  for (;;) {
    unsigned long long e[kWin], q[kWin];
#pragma unroll
    for (int j = 0; j < kWin; ++j) {
      const bool in = done + j < count;
      e[j] = in ? get_word(end + (done + j) * pitch) : 0ull;
      q[j] = in ? get_word(pair + (done + j) * pitch) : 0ull;
    }
    int at = -1;  // nearest end value with every pair before it there
    bool open = true;
#pragma unroll
    for (int j = 0; j < kWin; ++j) {
      if (open && at < 0 && e[j] != 0ull) at = j;
      if (q[j] == 0ull) open = false;
    }
    if (at >= 0) {
#pragma unroll
      for (int j = kWin - 1; j >= 0; --j) {
        if (j == at) h = __uint_as_float((unsigned)e[j]);
        if (j < at) h = apply<kMask>(-__uint_as_float((unsigned)(q[j] >> 32)), h, __uint_as_float((unsigned)q[j]));
      }
      break;
    }
    if (open) {
      done += kWin;
      continue;
    }
    if (++polls > p.spin_limit) {
      atomicOr(p.error, 1u);
      break;
    }
    __nanosleep(64);
  }
  // the windows passed on the way, farthest first
  for (int k = done; k > 0; k -= kWin) {
    unsigned long long q[kWin];
#pragma unroll
    for (int j = 0; j < kWin; ++j) q[j] = get_word(pair + (k - 1 - j) * pitch);
#pragma unroll
    for (int j = 0; j < kWin; ++j)
      h = apply<kMask>(-__uint_as_float((unsigned)(q[j] >> 32)), h, __uint_as_float((unsigned)q[j]));
  }
  return h;
}

__device__ __forceinline__ unsigned long long pair_word(float a, float h) {
  return ((unsigned long long)(__float_as_uint(a) | 0x80000000u) << 32) | __float_as_uint(h);
}
__device__ __forceinline__ unsigned long long end_word(float h) { return (1ull << 32) | __float_as_uint(h); }

// L steps of V channels of one stream, steps s0, s0 + 1, ... in scan order;
// those outside `live` (a bit per step) read as `other` and are not touched.
// A decay gate of kShut makes a step the identity to the last bit: a = 1, and
// b = 0 for x = 0.
template <class T, int V, int L>
__device__ __forceinline__ void load(Pack<T, V> (&out)[L], const Stream& s, int64_t b, int64_t t0, int dir, int64_t c,
                                     unsigned live, float other = 0.0f) {
  const T* p = static_cast<const T*>(s.p) + b * s.sb + t0 * s.st + c;
  const int64_t step = dir * s.st;
#pragma unroll
  for (int l = 0; l < L; ++l) {
    if ((live >> l) & 1u) {
      out[l] = *reinterpret_cast<const Pack<T, V>*>(p + l * step);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) out[l].v[v] = narrow<T>(other);
    }
  }
}

template <class T, int V, int L>
__device__ __forceinline__ void store(void* base, const Args& p, int64_t b, int64_t t, int64_t c, const float (&val)[V]) {
  Pack<T, V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.v[v] = narrow<T>(val[v]);
  *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(base) + (b * p.steps + t) * p.width + c) = o;
}

// What a thread works on
struct Place {
  int64_t b, c;      // row, first channel
  int tile;          // in scan order
  int64_t s0;        // first step of the thread, in scan order
  int64_t t0;        // and in memory
  int dir;
  bool on;           // channel in range
  unsigned inside;   // steps of the row
  unsigned live;     // before the row's length
  unsigned cut;      // reset
};

template <int V, int L, bool kMask>
__device__ __forceinline__ Place place(const Args& p, unsigned id, bool from_end) {
  Place o;
  const unsigned per = (unsigned)(p.batch * p.ctiles);
  o.tile = id / per;
  const unsigned rest = id - o.tile * per;
  if (from_end) o.tile = p.tiles - 1 - o.tile;
  o.b = rest / p.ctiles;
  o.c = (int64_t)(rest - (unsigned)o.b * p.ctiles) * (32 * V) + threadIdx.x * V;
  o.on = o.c < p.width;
  o.s0 = (int64_t)o.tile * (blockDim.y * L) + threadIdx.y * L;
  o.dir = p.reverse ? -1 : 1;
  o.t0 = p.reverse ? p.steps - 1 - o.s0 : o.s0;
  const int64_t left = p.steps - o.s0;
  o.inside = left >= L ? (1u << L) - 1 : left <= 0 ? 0u : (1u << left) - 1;
  o.live = o.inside;
  o.cut = 0u;
  if (kMask) {
    if (p.lengths) {
      const int64_t len = p.lengths[o.b];
#pragma unroll
      for (int l = 0; l < L; ++l)
        if (o.t0 + l * o.dir >= len) o.live &= ~(1u << l);
    }
    if (p.reset) {
#pragma unroll
      for (int l = 0; l < L; ++l)
        if ((o.live >> l) & 1u)
          if (p.reset[o.b * p.reset_b + (o.t0 + l * o.dir) * p.reset_t]) o.cut |= 1u << l;
    }
  }
  return o;
}

__device__ __forceinline__ unsigned claim(const Args& p) {
  __shared__ unsigned s_id;
  if (p.tiles == 1) return blockIdx.x;
  if (threadIdx.x == 0 && threadIdx.y == 0) s_id = atomicAdd(p.ticket, 1u);
  __syncthreads();
  return s_id;
}

template <class T, int V, int L, bool kMask>
__global__ void __launch_bounds__(32 * kWarps, kForwardCtas) forward_kernel(const __grid_constant__ Args p) {
  constexpr int C = 32 * V;
  __shared__ float sA[kWarps][C], sH[kWarps][C], sS[C];
  const Place o = place<V, L, kMask>(p, claim(p), false);
  const int lane = threadIdx.x, warp = threadIdx.y, warps = blockDim.y;

  Pack<T, V> x[L], ig[L], rg[L];
  const unsigned touch = o.on ? o.live : 0u;
  load<T, V, L>(rg, p.rg, o.b, o.t0, o.dir, o.c, touch, kShut);
  load<T, V, L>(ig, p.ig, o.b, o.t0, o.dir, o.c, touch);
  load<T, V, L>(x, p.x, o.b, o.t0, o.dir, o.c, touch);
  float kd[V];
#pragma unroll
  for (int v = 0; v < V; ++v) kd[v] = o.on ? -p.rate * softplus(p.decay[o.c + v]) : 0.0f;

  float a[L][V], b[L][V], A[V], H[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, H[v] = 0.0f;
#pragma unroll
  for (int l = 0; l < L; ++l) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gates g = gates(widen(ig[l].v[v]), widen(rg[l].v[v]), kd[v]);
      float beta = g.w > 0.0f ? g.w * rsqrt_approx(g.w) : g.w;
      float ga = g.a;
      if (kMask && ((o.cut >> l) & 1u)) ga = 0.0f, beta = 1.0f;
      a[l][v] = ga;
      b[l][v] = beta * g.i * widen(x[l].v[v]);
      H[v] = apply<kMask>(ga, H[v], b[l][v]);
      A[v] *= ga;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sA[warp][lane * V + v] = A[v], sH[warp][lane * V + v] = H[v];
  __syncthreads();

  const int64_t c0 = o.c - lane * V;
  for (int k = warp * 32 + lane; k < C; k += warps * 32) {
    const int64_t c = c0 + k;
    if (c >= p.width) break;
    float tA = 1.0f, tH = 0.0f;
    for (int w = 0; w < warps; ++w) {
      tH = apply<kMask>(sA[w][k], tH, sH[w][k]);
      tA *= sA[w][k];
    }
    const int64_t at = (o.b * p.tiles + o.tile) * p.width + c;
    float h = o.tile == 0 && p.state ? p.state[o.b * p.width + c] : 0.0f;
    if (o.tile > 0) {
      put_word(p.pair + at, pair_word(tA, tH));
      h = look_back<kMask>(p, p.pair + at - p.width, p.end + at - p.width, -p.width, o.tile);
    }
    sS[k] = h;
    h = apply<kMask>(tA, h, tH);
    if (p.tiles > 1) put_word(p.end + at, end_word(h));
    if (o.tile == p.tiles - 1) p.last[o.b * p.width + c] = h;
  }
  __syncthreads();
  if (!o.on || o.inside == 0u) return;

  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = sS[lane * V + v];
  for (int w = 0; w < warp; ++w) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = apply<kMask>(sA[w][lane * V + v], h[v], sH[w][lane * V + v]);
  }
#pragma unroll
  for (int l = 0; l < L; ++l) {
    float out[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = apply<kMask>(a[l][v], h[v], b[l][v]);
      out[v] = !kMask || ((o.live >> l) & 1u) ? h[v] : 0.0f;
    }
    if ((o.inside >> l) & 1u) store<T, V, L>(p.y, p, o.b, o.t0 + l * o.dir, o.c, out);
  }
}

template <class T, int V, int L, bool kMask>
__global__ void __launch_bounds__(32 * kWarps, kBackwardCtas) backward_kernel(const __grid_constant__ Args p) {
  constexpr int C = 32 * V;
  // (A, H): the forward map of each warp's steps; E: what the carry e leaves them with from zero
  __shared__ float sA[kWarps][C], sH[kWarps][C], sE[kWarps][C], sC[C];
  const Place o = place<V, L, kMask>(p, claim(p), true);
  const int lane = threadIdx.x, warp = threadIdx.y, warps = blockDim.y;

  Pack<T, V> x[L], ig[L], rg[L], dy[L];
  const unsigned touch = o.on ? o.live : 0u;
  load<T, V, L>(rg, p.rg, o.b, o.t0, o.dir, o.c, touch, kShut);
  load<T, V, L>(ig, p.ig, o.b, o.t0, o.dir, o.c, touch);
  load<T, V, L>(x, p.x, o.b, o.t0, o.dir, o.c, touch);
  load<T, V, L>(dy, p.dy, o.b, o.t0, o.dir, o.c, p.dy.p ? touch : 0u);
  float kd[V];
#pragma unroll
  for (int v = 0; v < V; ++v) kd[v] = o.on ? -p.rate * softplus(p.decay[o.c + v]) : 0.0f;

  float gi[L][V], gr[L][V], a[L][V], be[L][V], hp[L][V], A[V], H[V], E[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, H[v] = 0.0f, E[v] = 0.0f;
#pragma unroll
  for (int l = 0; l < L; ++l) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gates g = gates(widen(ig[l].v[v]), widen(rg[l].v[v]), kd[v]);
      gi[l][v] = g.i, gr[l][v] = g.r, a[l][v] = g.a;
      be[l][v] = g.w > 0.0f ? g.w * rsqrt_approx(g.w) : g.w;
      if (kMask && ((o.cut >> l) & 1u)) a[l][v] = 0.0f, be[l][v] = 1.0f;
      H[v] = apply<kMask>(a[l][v], H[v], be[l][v] * g.i * widen(x[l].v[v]));
      A[v] *= a[l][v];
    }
  }
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      E[v] += widen(dy[l].v[v]);
      E[v] = kMask && a[l][v] == 0.0f ? 0.0f : a[l][v] * E[v];
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sA[warp][lane * V + v] = A[v], sH[warp][lane * V + v] = H[v], sE[warp][lane * V + v] = E[v];
  __syncthreads();

  const int64_t c0 = o.c - lane * V;
  for (int k = warp * 32 + lane; k < C; k += warps * 32) {
    const int64_t c = c0 + k;
    if (c >= p.width) break;
    float tA = 1.0f, tE = 0.0f;
    for (int w = warps - 1; w >= 0; --w) {
      tE = apply<kMask>(sA[w][k], tE, sE[w][k]);
      tA *= sA[w][k];
    }
    const int64_t at = (o.b * p.tiles + o.tile) * p.width + c;
    const int after = p.tiles - 1 - o.tile;
    float e = after == 0 && p.dlast ? p.dlast[o.b * p.width + c] : 0.0f;
    if (after > 0) {
      put_word(p.pair + at, pair_word(tA, tE));
      e = look_back<kMask>(p, p.pair + at + p.width, p.end + at + p.width, p.width, after);
    }
    sC[k] = e;
    e = apply<kMask>(tA, e, tE);
    if (p.tiles > 1) put_word(p.end + at, end_word(e));
    if (o.tile == 0 && p.dstate) p.dstate[o.b * p.width + c] = e;
  }

  // the states before each step, from the tile's start state
  float h[V], e[V], acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = 0.0f, acc[v] = 0.0f;
    if (o.on) {
      if (o.tile > 0)
        h[v] = __uint_as_float((unsigned)p.start[(o.b * p.tiles + o.tile - 1) * p.width + o.c + v]);
      else if (p.state)
        h[v] = p.state[o.b * p.width + o.c + v];
    }
  }
  for (int w = 0; w < warp; ++w) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = apply<kMask>(sA[w][lane * V + v], h[v], sH[w][lane * V + v]);
  }
#pragma unroll
  for (int l = 0; l < L; ++l) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      hp[l][v] = h[v];
      h[v] = apply<kMask>(a[l][v], h[v], be[l][v] * gi[l][v] * widen(x[l].v[v]));
    }
  }
  __syncthreads();

#pragma unroll
  for (int v = 0; v < V; ++v) e[v] = sC[lane * V + v];
  for (int w = warps - 1; w > warp; --w) {
#pragma unroll
    for (int v = 0; v < V; ++v) e[v] = apply<kMask>(sA[w][lane * V + v], e[v], sE[w][lane * V + v]);
  }
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
    float dx[V], di[V], dr[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float g = e[v] + widen(dy[l].v[v]), av = a[l][v], bv = be[l][v], xv = widen(x[l].v[v]);
      const bool zero = kMask && av == 0.0f;
      e[v] = zero ? 0.0f : av * g;
      const bool dead = kMask && !((o.live >> l) & 1u);
      dx[v] = dead ? 0.0f : g * bv * gi[l][v];
      di[v] = dx[v] * xv * (1.0f - gi[l][v]);
      const float slope = bv > 0.0f ? av * av * rcp_approx(bv) : 0.0f;
      float dla = fmaf(e[v], hp[l][v], -g * gi[l][v] * xv * slope);
      if (zero || dead) dla = 0.0f;
      const float s = dla * gr[l][v];
      acc[v] += s;
      dr[v] = s * kd[v] * (1.0f - gr[l][v]);
    }
    if (o.on && ((o.inside >> l) & 1u)) {
      const int64_t t = o.t0 + l * o.dir;
      store<T, V, L>(p.dx, p, o.b, t, o.c, dx);
      store<T, V, L>(p.dig, p, o.b, t, o.c, di);
      store<T, V, L>(p.drg, p, o.b, t, o.c, dr);
    }
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) sE[warp][lane * V + v] = acc[v];
  __syncthreads();
  for (int k = warp * 32 + lane; k < C; k += warps * 32) {
    const int64_t c = c0 + k;
    if (c >= p.width) break;
    float s = 0.0f;
    for (int w = 0; w < warps; ++w) s += sE[w][k];
    p.dpart[(o.b * p.tiles + o.tile) * p.width + c] = s;
  }
}

struct Geometry {
  int tiles, ctiles, warps, steps_per_thread, vec;
  int64_t blocks;
};

template <class T>
cudaError_t launch(const Args& p, const Geometry& g, bool backward, bool mask, cudaStream_t s);

}  // namespace gscan
}  // namespace pesq
