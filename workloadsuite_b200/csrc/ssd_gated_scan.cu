// Per-channel gated linear recurrence, its gradient, and one token of it:
//   log a[t] = -rate * softplus(decay[c]) * sigmoid(r[t]),   u[t] = sqrt(1 - a[t]^2) * sigmoid(i[t]) * x[t],
//   h[t] = a[t] * h[t-1] + u[t]   (h[t-1] is left out where reset[t] is set),   y = h
// with x, i, r, y [b,s,d] (channels contiguous) and h, decay fp32.  The gradient, g[t] being that of h[t]:
//   g[t] = dy[t] + a[t+1] g[t+1],   dx = g b si,   di = g b x si (1 - si),
//   dr = (g a h[t-1] - g si x a^2 / b) la (1 - sr),   ddecay = -rate sigmoid(decay) sum_t (...) sr,   dh[0] = a[1] g[1]
// with b = sqrt(1 - a^2), si = sigmoid(i), sr = sigmoid(r), la = log a.
//
// Tokens fall into runs (one thread: kRun tokens of two channels, its a and u in registers), runs into tiles (one CTA: 64
// channels, up to 16 runs).  A run, a tile: h_out = P h_in + q.  The runs' pairs meet in shared memory, the tiles' in scratch: a
// tile publishes its pair, finds the state entering it by a look back at the pairs and states before it, publishes the state
// leaving it, and goes through its tokens again, in registers.  So every input is read once and every output written once.
// Tiles take their numbers from a counter in the order they start in: what a tile waits for has started before it.
// A state is only ever folded through whole tiles' pairs, h <- P h + q, one tile after the other, wherever the look back begins:
// results do not depend on what was published when.
// Entering states of 64-token pieces are kept for the gradient, which makes every h again in fp32 instead of reading y.
#include <algorithm>
#include <cmath>

#include "vec_io.cuh"

namespace ssd {
namespace {

constexpr int kRun = 8, kRunGrad = 4, kRuns = 16, kStrip = 64, kPiece = 64;
constexpr int kTile = kRun * kRuns, kTileGrad = kRunGrad * kRuns;
static_assert(kTile % kPiece == 0 && kPiece % kRun == 0 && kTileGrad == kPiece, "pieces start at runs");

struct Scan {
  const void *x, *i, *r, *dy;
  void *y, *dx, *di, *dr;
  const float *decay, *init, *dfinal;
  const unsigned char* reset;
  float *fin, *pieces, *part, *dinit;
  unsigned* counter;             // scratch, all bits set at launch: counter, pairs [tile][64], states [tile][64]
  unsigned long long* pairs;
  unsigned* states;
  int32_t* status;
  long long wait_clocks;
  float rate;
  int batch, seqlen, channels, strips, tiles, npieces;
  int64_t xs[2], is[2], rs[2], ys[2], dys[2], dxs[2], dis[2], drs[2], ms[2];
};

// A published word that is not there yet.  (A number with these bits, a NaN, is published as another NaN.)
constexpr unsigned kNone = 0xffffffffu;
// P of what nothing of the entering state is left in: a reset, or a state itself
constexpr unsigned kFresh = 0x80000000u;

__device__ __forceinline__ unsigned word(float v) {
  const unsigned b = __float_as_uint(v);
  return b == kNone ? 0x7fffffffu : b;
}
__device__ __forceinline__ unsigned load_word(const unsigned* p) {
  unsigned v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long load_word(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_word(unsigned* p, unsigned v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ void store_word(unsigned long long* p, unsigned long long v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

// State behind a run or a tile (P, q) that `s` enters.  Where P has underflowed an infinite state stays one, as token by token.
__device__ __forceinline__ float pass(float P, float q, float s) {
  if (__float_as_uint(P) == kFresh) return q;
  if (P == 0.f && isinf(s)) return s + q;
  return fmaf(P, s, q);
}

// -rate * softplus(decay), and -rate * sigmoid(decay), its derivative
__device__ __forceinline__ float decay_rate(float rate, float decay) {
  return -rate * (fmaxf(decay, 0.f) + log1pf(expf(-fabsf(decay))));
}

// One number's gates.  Where a is near 1 it is 1 - q, q = 1 - e^-v (v = -la) by its series: an exponential by itself is off by some 2^-23 of
// a, and a state that some thousand tokens stay in adds that up.  The series' rest is below 4e-8 of q up to v = 0.4; beyond, a state is
// gone before errors add up.  1 - a^2 = q (1 + a) loses nothing in either case.
struct Gates {
  float sr, la, a, om;
  __device__ __forceinline__ Gates(float k, float r) {
    sr = sigmoid_approx(r);
    la = k * sr;
    const float v = -la;
    float p = 1.f / 5040;
    p = fmaf(p, v, -1.f / 720);
    p = fmaf(p, v, 1.f / 120);
    p = fmaf(p, v, -1.f / 24);
    p = fmaf(p, v, 1.f / 6);
    p = fmaf(p, v, -0.5f);
    p = fmaf(p, v, 1.f);
    const float e = exp2_approx(kLog2E * la), q = v < 0.4f ? p * v : 1.f - e;
    a = v < 0.4f ? 1.f - q : e;
    om = q * (1.f + a);
  }
  // 1 / sqrt(1 - a^2), 0 where a is 1: it comes with factors that vanish faster
  __device__ __forceinline__ float inv() const { return om == 0.f ? 0.f : rsqrt_approx(om); }
};

template <typename T, bool VEC>
struct Lane {
  int c, apart;        // first channel, distance of the second
  bool ok0, ok1;
  int j0, j1;          // their places among the strip's 64
  __device__ __forceinline__ Lane(int strip, int channels) {
    const int l = threadIdx.x % 32;
    j0 = VEC ? 2 * l : l;
    apart = VEC ? 1 : 32;
    j1 = j0 + apart;
    c = strip * kStrip + j0;
    ok0 = c < channels;
    ok1 = c + apart < channels;
  }
};

struct Shared {
  float P[kRuns][kStrip], q[kRuns][kStrip], in[kRuns][kStrip];
  float2 seen[kRuns][kStrip];
  unsigned ticket;
};

// Which tile this CTA works on: (place in its sequence, strip and batch entry).
__device__ __forceinline__ int2 take_tile(const Scan& p, Shared& sh) {
  const unsigned units = (unsigned)p.strips * p.batch;
  if (p.tiles == 1) return make_int2(0, (int)blockIdx.x);
  if (threadIdx.x == 0) sh.ticket = atomicAdd(p.counter, 1u) + 1u;
  __syncthreads();
  return make_int2((int)(sh.ticket / units), (int)(sh.ticket % units));
}

// What stands before tile `k` of the unit, into sh.seen: warp w looks at tile k - 1 - w, for its state or else its pair; the farthest
// one waits for the state, so that one look is enough.
__device__ __forceinline__ void look_back(const Scan& p, Shared& sh, int64_t first, int k, int j0, int j1) {
  const int w = threadIdx.x / 32, nw = blockDim.x / 32;
  if (w < k) {
    const int64_t at = (first + k - 1 - w) * kStrip;
    const bool far = w == nw - 1;
    unsigned s0, s1;
    unsigned long long p0 = ~0ull, p1 = ~0ull;
    const long long t0 = clock64();
    while (true) {
      s0 = load_word(p.states + at + j0);
      s1 = load_word(p.states + at + j1);
      if (!far) {
        p0 = load_word(p.pairs + at + j0);
        p1 = load_word(p.pairs + at + j1);
      }
      if ((s0 != kNone || (unsigned)p0 != kNone) && (s1 != kNone || (unsigned)p1 != kNone)) break;
      if (clock64() - t0 > p.wait_clocks) {
        if (p.status) *p.status = STATUS_WAIT_TIMEOUT_LOOK_BACK;
        break;
      }
      __nanosleep(20);
    }
    const float fresh = __uint_as_float(kFresh);
    sh.seen[w][j0] = s0 != kNone ? make_float2(fresh, __uint_as_float(s0))
                                 : make_float2(__uint_as_float((unsigned)p0), __uint_as_float((unsigned)(p0 >> 32)));
    sh.seen[w][j1] = s1 != kNone ? make_float2(fresh, __uint_as_float(s1))
                                 : make_float2(__uint_as_float((unsigned)p1), __uint_as_float((unsigned)(p1 >> 32)));
  }
}

// The state entering a tile from what look_back() saw.
__device__ __forceinline__ float fold_seen(const Shared& sh, int k, int j) {
  float s = 0.f;
  for (int w = min(k, (int)blockDim.x / 32) - 1; w >= 0; --w) s = pass(sh.seen[w][j].x, sh.seen[w][j].y, s);
  return s;
}

__device__ __forceinline__ void publish_pair(const Scan& p, int64_t tile, int j, float P, float q) {
  store_word(p.pairs + tile * kStrip + j, (unsigned long long)word(P) | (unsigned long long)__float_as_uint(q) << 32);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kRuns, 2) gated_scan_kernel(const Scan p) {
  using Raw = typename Two<T>::Raw;
  __shared__ Shared sh;
  const int2 which = take_tile(p, sh);
  const int k = which.x, strip = which.y % p.strips, b = which.y / p.strips;
  const int w = threadIdx.x / 32, nw = blockDim.x / 32;
  const int t0 = k * kTile + w * kRun;
  const int here = min(kRun, p.seqlen - t0);   // tokens of this run that are there
  const Lane<T, VEC> ln(strip, p.channels);
  const int64_t tile = (int64_t)which.y * p.tiles;   // the sequence's first

  Raw rx[kRun], ri[kRun], rr[kRun];
  {
    const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + (int64_t)t0 * p.xs[1] + ln.c;
    const T* i = static_cast<const T*>(p.i) + b * p.is[0] + (int64_t)t0 * p.is[1] + ln.c;
    const T* r = static_cast<const T*>(p.r) + b * p.rs[0] + (int64_t)t0 * p.rs[1] + ln.c;
#pragma unroll
    for (int t = 0; t < kRun; ++t) {
      const bool there = t < here;
      rr[t] = load_two<T, VEC>(r + t * p.rs[1], ln.apart, there && ln.ok0, there && ln.ok1);
      ri[t] = load_two<T, VEC>(i + t * p.is[1], ln.apart, there && ln.ok0, there && ln.ok1);
      rx[t] = load_two<T, VEC>(x + t * p.xs[1], ln.apart, there && ln.ok0, there && ln.ok1);
    }
  }
  unsigned marks = 0;
  if (p.reset) {
    const unsigned char* m = p.reset + b * p.ms[0] + (int64_t)t0 * p.ms[1];
#pragma unroll
    for (int t = 0; t < kRun; ++t)
      if (t < here && m[t * p.ms[1]]) marks |= 1u << t;
  }
  const float k0 = ln.ok0 ? decay_rate(p.rate, p.decay[ln.c]) : 0.f;
  const float k1 = ln.ok1 ? decay_rate(p.rate, p.decay[ln.c + ln.apart]) : 0.f;

  float a[kRun][2], u[kRun][2];
  float P[2] = {1.f, 1.f}, q[2] = {0.f, 0.f};
  const float fresh = __uint_as_float(kFresh);
#pragma unroll
  for (int t = 0; t < kRun; ++t) {
    const float2 xv = Two<T>::up(rx[t]), iv = Two<T>::up(ri[t]), rv = Two<T>::up(rr[t]);
    const Gates g0(k0, rv.x), g1(k1, rv.y);
    a[t][0] = g0.a; a[t][1] = g1.a;
    u[t][0] = (g0.om * g0.inv()) * (sigmoid_approx(iv.x) * xv.x);
    u[t][1] = (g1.om * g1.inv()) * (sigmoid_approx(iv.y) * xv.y);
    if (t >= here) a[t][0] = a[t][1] = 1.f, u[t][0] = u[t][1] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool cut = marks >> t & 1;
      P[e] = cut ? fresh : P[e] * a[t][e];
      q[e] = cut ? u[t][e] : fmaf(a[t][e], q[e], u[t][e]);
    }
  }
  sh.P[w][ln.j0] = P[0]; sh.P[w][ln.j1] = P[1];
  sh.q[w][ln.j0] = q[0]; sh.q[w][ln.j1] = q[1];
  __syncthreads();

  const int j = threadIdx.x, cj = strip * kStrip + j;
  const bool fold = j < kStrip;
  const bool last = k == p.tiles - 1;
  auto first_state = [&]() { return p.init && cj < p.channels ? p.init[(int64_t)b * p.channels + cj] : 0.f; };
  float tp = 1.f, tq = 0.f;   // the tile's pair
  if (fold) {
    for (int v = 0; v < nw; ++v) {
      tq = pass(sh.P[v][j], sh.q[v][j], tq);
      tp = __float_as_uint(sh.P[v][j]) == kFresh ? fresh : tp * sh.P[v][j];
    }
    if (k > 0 && !last) publish_pair(p, tile + k, j, tp, tq);
  }
  if (k > 0) {
    look_back(p, sh, tile, k, ln.j0, ln.j1);
    __syncthreads();
  }
  if (fold) {
    float s = k == 0 ? first_state() : fold_seen(sh, k, j);
    const float out = pass(tp, tq, s);
    if (!last) store_word(p.states + (tile + k) * kStrip + j, word(out));
    if (last && p.fin && cj < p.channels) p.fin[(int64_t)b * p.channels + cj] = out;
    for (int v = 0; v < nw; ++v) {
      sh.in[v][j] = s;
      const int t = k * kTile + v * kRun;
      if (p.pieces && t % kPiece == 0 && t < p.seqlen && cj < p.channels)
        p.pieces[((int64_t)b * p.npieces + t / kPiece) * p.channels + cj] = s;
      s = pass(sh.P[v][j], sh.q[v][j], s);
    }
  }
  __syncthreads();

  float h0 = sh.in[w][ln.j0], h1 = sh.in[w][ln.j1];
  T* y = static_cast<T*>(p.y) + b * p.ys[0] + (int64_t)t0 * p.ys[1] + ln.c;
#pragma unroll
  for (int t = 0; t < kRun; ++t) {
    const bool cut = marks >> t & 1;
    h0 = cut ? u[t][0] : fmaf(a[t][0], h0, u[t][0]);
    h1 = cut ? u[t][1] : fmaf(a[t][1], h1, u[t][1]);
    store_two<T, VEC>(y + t * p.ys[1], ln.apart, t < here && ln.ok0, t < here && ln.ok1, h0, h1);
  }
}

// The gradient: the same walk from the last tile to the first, what passes from a token to the one before it being a[t] g[t].
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kRuns, 1) gated_scan_grad_kernel(const Scan p) {
  using Raw = typename Two<T>::Raw;
  constexpr int L = kRunGrad;
  __shared__ Shared sh;
  __shared__ float qb[kRuns][kStrip], back[kRuns][kStrip];   // pairs and entering numbers of the way back
  const int2 which = take_tile(p, sh);
  const int kb = which.x, k = p.tiles - 1 - kb, strip = which.y % p.strips, b = which.y / p.strips;
  const int w = threadIdx.x / 32, nw = blockDim.x / 32;
  const int t0 = k * kTileGrad + w * L;
  const int here = min(L, p.seqlen - t0);
  const Lane<T, VEC> ln(strip, p.channels);
  const int64_t tile = (int64_t)which.y * p.tiles;

  Raw rx[L], ri[L], rr[L], rd[L];
  {
    const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + (int64_t)t0 * p.xs[1] + ln.c;
    const T* i = static_cast<const T*>(p.i) + b * p.is[0] + (int64_t)t0 * p.is[1] + ln.c;
    const T* r = static_cast<const T*>(p.r) + b * p.rs[0] + (int64_t)t0 * p.rs[1] + ln.c;
    const T* d = static_cast<const T*>(p.dy) + b * p.dys[0] + (int64_t)t0 * p.dys[1] + ln.c;
#pragma unroll
    for (int t = 0; t < L; ++t) {
      const bool there = t < here;
      rr[t] = load_two<T, VEC>(r + t * p.rs[1], ln.apart, there && ln.ok0, there && ln.ok1);
      ri[t] = load_two<T, VEC>(i + t * p.is[1], ln.apart, there && ln.ok0, there && ln.ok1);
      rx[t] = load_two<T, VEC>(x + t * p.xs[1], ln.apart, there && ln.ok0, there && ln.ok1);
      rd[t] = load_two<T, VEC>(d + t * p.dys[1], ln.apart, there && ln.ok0, there && ln.ok1);
    }
  }
  unsigned marks = 0;
  if (p.reset) {
    const unsigned char* m = p.reset + b * p.ms[0] + (int64_t)t0 * p.ms[1];
#pragma unroll
    for (int t = 0; t < L; ++t)
      if (t < here && m[t * p.ms[1]]) marks |= 1u << t;
  }
  const int j = threadIdx.x, cj = strip * kStrip + j;
  const bool fold = j < kStrip;
  float s = 0.f;   // state entering the tile
  if (fold && cj < p.channels) s = p.pieces[((int64_t)b * p.npieces + k) * p.channels + cj];
  const float k0 = ln.ok0 ? decay_rate(p.rate, p.decay[ln.c]) : 0.f;
  const float k1 = ln.ok1 ? decay_rate(p.rate, p.decay[ln.c + ln.apart]) : 0.f;
  const float fresh = __uint_as_float(kFresh);

  float a[L][2], u[L][2];
  float P[2] = {1.f, 1.f}, q[2] = {0.f, 0.f}, c[2] = {0.f, 0.f};
#pragma unroll
  for (int t = 0; t < L; ++t) {
    const float2 xv = Two<T>::up(rx[t]), iv = Two<T>::up(ri[t]), rv = Two<T>::up(rr[t]);
    const Gates g0(k0, rv.x), g1(k1, rv.y);
    a[t][0] = g0.a; a[t][1] = g1.a;
    u[t][0] = (g0.om * g0.inv()) * (sigmoid_approx(iv.x) * xv.x);
    u[t][1] = (g1.om * g1.inv()) * (sigmoid_approx(iv.y) * xv.y);
    if (t >= here) a[t][0] = a[t][1] = 1.f, u[t][0] = u[t][1] = 0.f;
    const bool cut = marks >> t & 1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      P[e] = cut ? fresh : P[e] * a[t][e];
      q[e] = cut ? u[t][e] : fmaf(a[t][e], q[e], u[t][e]);
    }
  }
#pragma unroll
  for (int t = L - 1; t >= 0; --t) {
    const float2 dv = Two<T>::up(rd[t]);
    const bool cut = marks >> t & 1;
    c[0] = cut ? 0.f : a[t][0] * (dv.x + c[0]);
    c[1] = cut ? 0.f : a[t][1] * (dv.y + c[1]);
  }
  sh.P[w][ln.j0] = P[0]; sh.P[w][ln.j1] = P[1];
  sh.q[w][ln.j0] = q[0]; sh.q[w][ln.j1] = q[1];
  qb[w][ln.j0] = c[0]; qb[w][ln.j1] = c[1];
  __syncthreads();

  const bool last = kb == p.tiles - 1;   // of the way back: the sequence's first
  float tp = 1.f, tq = 0.f;
  if (fold) {
    for (int v = nw - 1; v >= 0; --v) {
      tq = pass(sh.P[v][j], qb[v][j], tq);
      tp = __float_as_uint(sh.P[v][j]) == kFresh ? fresh : tp * sh.P[v][j];
    }
    if (kb > 0 && !last) publish_pair(p, tile + kb, j, tp, tq);
    for (int v = 0; v < nw; ++v) {
      sh.in[v][j] = s;
      s = pass(sh.P[v][j], sh.q[v][j], s);
    }
  }
  if (kb > 0) {
    look_back(p, sh, tile, kb, ln.j0, ln.j1);
    __syncthreads();
  }
  if (fold) {
    float g = 0.f;
    if (kb > 0) g = fold_seen(sh, kb, j);
    else if (p.dfinal && cj < p.channels) g = p.dfinal[(int64_t)b * p.channels + cj];
    const float out = pass(tp, tq, g);
    if (!last) store_word(p.states + (tile + kb) * kStrip + j, word(out));
    if (last && p.dinit && cj < p.channels) p.dinit[(int64_t)b * p.channels + cj] = out;
    for (int v = nw - 1; v >= 0; --v) {
      back[v][j] = g;
      g = pass(sh.P[v][j], qb[v][j], g);
    }
  }
  __syncthreads();

  float h[2] = {sh.in[w][ln.j0], sh.in[w][ln.j1]};
#pragma unroll
  for (int t = 0; t < L; ++t) {   // u[t] becomes the state before t
    const bool cut = marks >> t & 1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float before = h[e];
      h[e] = cut ? u[t][e] : fmaf(a[t][e], before, u[t][e]);
      u[t][e] = before;
    }
  }
  c[0] = back[w][ln.j0];
  c[1] = back[w][ln.j1];
  float dd[2] = {0.f, 0.f};
  T* dx = static_cast<T*>(p.dx) + b * p.dxs[0] + (int64_t)t0 * p.dxs[1] + ln.c;
  T* di = static_cast<T*>(p.di) + b * p.dis[0] + (int64_t)t0 * p.dis[1] + ln.c;
  T* dr = static_cast<T*>(p.dr) + b * p.drs[0] + (int64_t)t0 * p.drs[1] + ln.c;
#pragma unroll
  for (int t = L - 1; t >= 0; --t) {
    const float2 xv = Two<T>::up(rx[t]), iv = Two<T>::up(ri[t]), rv = Two<T>::up(rr[t]), dv = Two<T>::up(rd[t]);
    const bool cut = marks >> t & 1;
    float ox[2], oi[2], orr[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const Gates gt(e ? k1 : k0, e ? rv.y : rv.x);
      const float xe = e ? xv.y : xv.x;
      const float si = sigmoid_approx(e ? iv.y : iv.x), inv = gt.inv(), beta = gt.om * inv;
      const float g = (e ? dv.y : dv.x) + c[e];
      const float gs = g * si, gb = gs * beta;
      ox[e] = gb;
      oi[e] = gb * xe * (1.f - si);
      const float through = cut ? 0.f : g * u[t][e] * gt.a;         // what a's share of h brings
      const float root = gs * xe, steep = gt.a * gt.a * inv;        // and b's: -root * steep
      orr[e] = (1.f - gt.sr) * (through * gt.la - root * (steep * gt.la));
      if (t < here) {
        dd[e] += through * gt.sr - root * (steep * gt.sr);
        c[e] = cut ? 0.f : gt.a * g;
      }
    }
    const bool ok0 = t < here && ln.ok0, ok1 = t < here && ln.ok1;
    store_two<T, VEC>(dx + t * p.dxs[1], ln.apart, ok0, ok1, ox[0], ox[1]);
    store_two<T, VEC>(di + t * p.dis[1], ln.apart, ok0, ok1, oi[0], oi[1]);
    store_two<T, VEC>(dr + t * p.drs[1], ln.apart, ok0, ok1, orr[0], orr[1]);
  }
  sh.q[w][ln.j0] = dd[0];
  sh.q[w][ln.j1] = dd[1];
  __syncthreads();
  if (fold && cj < p.channels) {
    float sum = 0.f;
    for (int v = 0; v < nw; ++v) sum += sh.q[v][j];
    p.part[((int64_t)b * p.tiles + k) * p.channels + cj] = sum;
  }
}

struct FinishDecay {
  const float* decay;
  float* out;
  float rate;
  __device__ __forceinline__ void operator()(int c, float v) const { out[c] = v * (-rate / (1.f + expf(-decay[c]))); }
};

// One token.  V channels per thread.
template <typename T, int V>
__global__ void __launch_bounds__(128) gated_step_kernel(const T* __restrict__ x, const T* __restrict__ i, const T* __restrict__ r,
                                                         const float* __restrict__ decay, const float* state, float* state_out,
                                                         T* y, int batch, int channels, int64_t xs, int64_t is, int64_t rs,
                                                         int64_t ys, float rate) {
  const int vecs = channels / V;
  const int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= (int64_t)batch * vecs) return;
  const int b = (int)(n / vecs), c = (int)(n % vecs) * V;
  T xv[V], iv[V], rv[V], yv[V];
  float dv[V], sv[V];
  auto copy = [](auto* to, const auto* from) {   // V numbers at once
    if constexpr (V == 1) to[0] = from[0];
    else if constexpr (sizeof(*to) == 2) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from);
    else *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
  };
  copy(xv, x + b * xs + c);
  copy(iv, i + b * is + c);
  copy(rv, r + b * rs + c);
  copy(sv, state + (int64_t)b * channels + c);
  copy(dv, decay + c);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const Gates g(decay_rate(rate, dv[e]), Cvt<T>::to_f(rv[e]));
    sv[e] = fmaf(g.a, sv[e], (g.om * g.inv()) * (sigmoid_approx(Cvt<T>::to_f(iv[e])) * Cvt<T>::to_f(xv[e])));
    yv[e] = Cvt<T>::from_f(sv[e]);
  }
  copy(state_out + (int64_t)b * channels + c, sv);
  copy(y + b * ys + c, yv);
}

int strips_of(int channels) { return (channels + kStrip - 1) / kStrip; }
int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

struct Sizes {
  int64_t tiles, units, words, part;   // tiles of a sequence, sequences of 64 channels, bytes
};
Sizes sizes_of(const SsdGatedScanArgs& a, bool grad) {
  Sizes z;
  const int tile = grad ? kTileGrad : kTile;
  z.tiles = (a.seqlen + (int64_t)tile - 1) / tile;
  z.units = (int64_t)a.batch * strips_of(a.channels);
  z.words = z.tiles == 1 ? 0 : 256 + z.units * z.tiles * kStrip * 12;
  z.part = grad ? (int64_t)a.batch * z.tiles * a.channels * 4 : 0;
  return z;
}

int check(const SsdGatedScanArgs* a, bool grad) {
  if (!a) return SSD_ERR_NULL_POINTER;
  if (a->batch <= 0 || a->seqlen <= 0 || a->channels <= 0 || a->wait_limit_ms < 0 || !(a->rate > 0.f && a->rate < INFINITY)) return SSD_ERR_BAD_SHAPE;
  if (a->dtype != SSD_DTYPE_F32 && a->dtype != SSD_DTYPE_F16 && a->dtype != SSD_DTYPE_BF16) return SSD_ERR_UNSUPPORTED;
  const Sizes z = sizes_of(*a, grad);
  if (a->seqlen > 0x7fffff00 || z.tiles * z.units > 0x7fffffff) return SSD_ERR_TOO_LARGE;
  return SSD_OK;
}

template <typename T>
int run_scan(const SsdGatedScanArgs& a, bool grad, cudaStream_t stream) {
  const Sizes z = sizes_of(a, grad);
  Scan p = {};
  p.x = a.x; p.i = a.input_gate; p.r = a.decay_gate; p.dy = a.dy;
  p.y = a.y; p.dx = a.dx; p.di = a.dinput_gate; p.dr = a.ddecay_gate;
  p.decay = a.decay; p.init = a.initial_state; p.dfinal = a.dfinal_state;
  p.reset = a.reset;
  p.fin = a.final_state; p.pieces = a.pieces; p.dinit = a.dinitial_state;
  p.status = a.status;
  p.wait_clocks = a.wait_limit_ms > 0 ? (long long)a.wait_limit_ms * 2000000LL : 2000000000LL;
  p.rate = a.rate;
  p.batch = a.batch; p.seqlen = a.seqlen; p.channels = a.channels;
  p.strips = strips_of(a.channels); p.tiles = (int)z.tiles; p.npieces = (a.seqlen + kPiece - 1) / kPiece;
  char* ws = static_cast<char*>(a.workspace);
  if (z.words) {
    p.counter = reinterpret_cast<unsigned*>(ws);
    p.pairs = reinterpret_cast<unsigned long long*>(ws + 256);
    p.states = reinterpret_cast<unsigned*>(ws + 256 + z.units * z.tiles * kStrip * 8);
    if (cudaMemsetAsync(ws, 0xff, (size_t)z.words, stream) != cudaSuccess) return SSD_ERR_CUDA;
  }
  p.part = reinterpret_cast<float*>(ws + up256(z.words));
  bool pairs = a.channels % 2 == 0;   // two channels at once: every row starts on their boundary
  auto strides = [&](int64_t (&to)[2], const int64_t (&from)[2], const void* at) {
    for (int d = 0; d < 2; ++d) {
      to[d] = from[d];
      pairs = pairs && from[d] % 2 == 0;
    }
    pairs = pairs && reinterpret_cast<uintptr_t>(at) % (2 * sizeof(T)) == 0;
  };
  strides(p.xs, a.x_stride, a.x);
  strides(p.is, a.input_gate_stride, a.input_gate);
  strides(p.rs, a.decay_gate_stride, a.decay_gate);
  for (int d = 0; d < 2; ++d) p.ms[d] = a.reset_stride[d];
  if (grad) {
    strides(p.dys, a.dy_stride, a.dy);
    strides(p.dxs, a.dx_stride, a.dx);
    strides(p.dis, a.dinput_gate_stride, a.dinput_gate);
    strides(p.drs, a.ddecay_gate_stride, a.ddecay_gate);
  } else {
    strides(p.ys, a.y_stride, a.y);
  }
  const unsigned grid = (unsigned)(z.tiles * z.units);
  const int run = grad ? kRunGrad : kRun;
  const int threads = z.tiles > 1 ? 32 * kRuns : 32 * std::max(2, (a.seqlen + run - 1) / run);   // (64 fold a strip)
  if (!grad) return launch(pairs ? gated_scan_kernel<T, true> : gated_scan_kernel<T, false>, grid, threads, 0, stream, p);
  if (const int rc = launch(pairs ? gated_scan_grad_kernel<T, true> : gated_scan_grad_kernel<T, false>, grid, threads, 0, stream, p))
    return rc;
  return launch_column_sum(p.part, a.batch * z.tiles, a.channels, a.channels, FinishDecay{a.decay, a.ddecay, a.rate}, stream);
}

template <typename T>
int run_step(const SsdGatedStepArgs& a, cudaStream_t stream) {
  auto fits = [](const void* p, int64_t stride, size_t bytes) {   // rows of four at once
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride % 4 == 0;
  };
  const bool four = a.channels % 4 == 0 && fits(a.x, a.x_stride, 4 * sizeof(T)) && fits(a.input_gate, a.input_gate_stride, 4 * sizeof(T)) &&
                    fits(a.decay_gate, a.decay_gate_stride, 4 * sizeof(T)) && fits(a.y, a.y_stride, 4 * sizeof(T)) &&
                    fits(a.state, 0, 16) && fits(a.state_out, 0, 16) && fits(a.decay, 0, 16);
  const int64_t threads = (int64_t)a.batch * (four ? a.channels / 4 : a.channels);
  if ((threads + 127) / 128 > 0x7fffffff) return SSD_ERR_TOO_LARGE;
  return launch(four ? gated_step_kernel<T, 4> : gated_step_kernel<T, 1>, (unsigned)((threads + 127) / 128), 128, 0, stream,
                static_cast<const T*>(a.x), static_cast<const T*>(a.input_gate), static_cast<const T*>(a.decay_gate), a.decay, a.state,
                a.state_out, static_cast<T*>(a.y), a.batch, a.channels, a.x_stride, a.input_gate_stride, a.decay_gate_stride, a.y_stride,
                a.rate);
}

}  // namespace
}  // namespace ssd

extern "C" size_t ssd_b200_gated_scan_workspace_bytes(const SsdGatedScanArgs* args, int32_t backward) {
  if (ssd::check(args, backward != 0) != SSD_OK) return 0;
  const ssd::Sizes z = ssd::sizes_of(*args, backward != 0);
  return (size_t)(ssd::up256(z.words) + z.part);
}

extern "C" int ssd_b200_gated_scan(const SsdGatedScanArgs* args, void* stream) {
  if (const int rc = ssd::check(args, false)) return rc;
  const SsdGatedScanArgs& a = *args;
  if (!a.x || !a.input_gate || !a.decay_gate || !a.decay || !a.y) return SSD_ERR_NULL_POINTER;
  const size_t need = ssd_b200_gated_scan_workspace_bytes(args, 0);
  if (need && (!a.workspace || a.workspace_bytes < need || reinterpret_cast<uintptr_t>(a.workspace) % 256)) return SSD_ERR_WORKSPACE;
  return ssd::by_type(a.dtype, [&](auto t) { return ssd::run_scan<decltype(t)>(a, false, static_cast<cudaStream_t>(stream)); });
}

extern "C" int ssd_b200_gated_scan_backward(const SsdGatedScanArgs* args, void* stream) {
  if (const int rc = ssd::check(args, true)) return rc;
  const SsdGatedScanArgs& a = *args;
  if (!a.x || !a.input_gate || !a.decay_gate || !a.decay || !a.dy || !a.pieces || !a.dx || !a.dinput_gate || !a.ddecay_gate || !a.ddecay)
    return SSD_ERR_NULL_POINTER;
  const size_t need = ssd_b200_gated_scan_workspace_bytes(args, 1);
  if (need && (!a.workspace || a.workspace_bytes < need || reinterpret_cast<uintptr_t>(a.workspace) % 256)) return SSD_ERR_WORKSPACE;
  return ssd::by_type(a.dtype, [&](auto t) { return ssd::run_scan<decltype(t)>(a, true, static_cast<cudaStream_t>(stream)); });
}

extern "C" int ssd_b200_gated_step(const SsdGatedStepArgs* args, void* stream) {
  if (!args) return SSD_ERR_NULL_POINTER;
  const SsdGatedStepArgs& a = *args;
  if (!a.x || !a.input_gate || !a.decay_gate || !a.decay || !a.state || !a.state_out || !a.y) return SSD_ERR_NULL_POINTER;
  if (a.batch <= 0 || a.channels <= 0 || !(a.rate > 0.f && a.rate < INFINITY)) return SSD_ERR_BAD_SHAPE;
  return ssd::by_type(a.dtype, [&](auto t) { return ssd::run_step<decltype(t)>(a, static_cast<cudaStream_t>(stream)); });
}
