// Per-channel gated linear recurrence, its gradient, and one token of it:
//   log a[t] = -rate * softplus(decay[c]) * sigmoid(r[t]),   u[t] = sqrt(1 - a[t]^2) * sigmoid(i[t]) * x[t],
//   h[t] = a[t] * h[t-1] + u[t]   (h[t-1] is left out where reset[t] is set),   y = h
// with x, i, r, y [b,s,d] (channels contiguous) and h, decay fp32.  The gradient, g[t] being that of h[t]:
//   g[t] = dy[t] + a[t+1] g[t+1],   dx = g b si,   di = g b x si (1 - si),
//   dr = (g a h[t-1] - g si x a^2 / b) la (1 - sr),   ddecay = -rate sigmoid(decay) sum_t (...) sr,   dh[0] = a[1] g[1]
// with b = sqrt(1 - a^2), si = sigmoid(i), sr = sigmoid(r), la = log a.
//
// Tokens fall into runs (one warp: kRun tokens of 64 channels, two a lane, their a and u in registers), runs into tiles (one CTA at a
// time), tiles into sequences.  A run, a tile: h_out = P h_in + q.  The runs' pairs (P, q) meet in shared memory, the tiles' in scratch: a
// tile publishes its pair, finds the state entering it by a look back at the states and pairs before it, publishes the state
// leaving it, and goes through its tokens again, from registers.  So every input is read once and every output written once.
// CTAs stay on the chip and take tiles from a counter, time first; the next tile's inputs are on their way (TMA) while one is worked on.
// What a tile waits for has a lower number, and the lowest one that is not done waits for nothing.
// A state is only ever folded through whole tiles' pairs, h <- P h + q, one tile after the other, wherever the look back begins:
// results do not depend on what was published when.
// Entering states of 64-token pieces are kept for the gradient, which makes every h again in fp32 instead of reading y.
// 8 x 2 048 x 2 048 bf16: forward 62 us (4.3 TB/s of algorithmic traffic, 67 % of the copy bandwidth), gradient 135 (53 %); 131 072 x 2 048:
// 494 us; where a strip's gates are not all MILD (below) 79, 142 and 618.  Bound: latency with sixteen warps an SM, whose registers the tokens' a and u fill; issue slots are half used, the
// special-function unit too (four functions a number, five in the gradient).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tc_common.cuh"
#include "tc_ptx.cuh"
#include "vec_io.cuh"

namespace ssd {
namespace {

constexpr int kStrip = 64, kPiece = 64;
// Tokens of a run, runs of a tile (warps of a CTA), CTAs that an SM holds (two tiles' inputs a CTA in shared memory).
// Long runs: what a run costs besides its tokens is some 250 instructions a warp (8 x 2 048 x 2 048 bf16: forward 64 us, with 12 runs of 8
// tokens 87, with three CTAs of 8 runs of 8 72; gradient 146 us, with 16 runs of 4 244).  fp32: as many numbers of shared memory hold half the
// tokens (4 x 2 048 x 2 048: two CTAs of 64 tokens 52 us, one of 128 54).
template <typename T, bool GRAD> struct Geometry;
template <typename T> struct Geometry<T, false> {
  static constexpr int kRun = sizeof(T) == 2 ? 16 : 8, kRuns = 8, kCtas = 2;
};
template <typename T> struct Geometry<T, true> {
  static constexpr int kRun = sizeof(T) == 2 ? 8 : 4, kRuns = sizeof(T) == 2 ? 8 : 16, kCtas = sizeof(T) == 2 ? 2 : 1;
};
constexpr int kTileGrad = kPiece;   // tokens of a tile
constexpr int tile_of(bool fp32) { return fp32 ? 64 : 128; }

struct Scan {
  const void *x, *i, *r, *dy;
  void *y, *dx, *di, *dr;
  const float *decay, *init, *dfinal;
  const float* rates;            // rate * softplus(decay) of every channel, where prepare_kernel has left them
  const unsigned char* reset;
  float *fin, *pieces, *part, *dinit;
  unsigned* counter;             // scratch, all bits set at launch: counter, pairs [tile][64], states [tile][64]
  unsigned long long *pairs, *states;
  int32_t* status;
  long long wait_clocks;
  float rate;
  int batch, seqlen, channels, strips, tiles, npieces;
  unsigned total;                // tiles of all sequences
  int inject, enter_ahead;       // enter_ahead: a gradient's entering states come with the inputs
  int early;                     // a forward's tile is sent for two tiles ahead, not half a one
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
__device__ __forceinline__ unsigned long long two_words(unsigned lo, unsigned hi) { return (unsigned long long)lo | (unsigned long long)hi << 32; }
__device__ __forceinline__ unsigned long long load_word(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_word(unsigned long long* p, unsigned long long v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

// State behind a run or a tile (P, q) that `s` enters.  Where P has underflowed an infinite state stays one, as token by token.
__device__ __forceinline__ float pass(float P, float q, float s) {
  float r = fmaf(P, s, q);
  if (P == 0.f) {
    if (__float_as_uint(P) == kFresh) r = q;
    else if (isinf(s)) r = s + q;
  }
  return r;
}

// rate * softplus(decay): what -log a is at most
__device__ __forceinline__ float decay_rate(float rate, float decay) {
  return rate * (fmaxf(decay, 0.f) + log1pf(expf(-fabsf(decay))));
}

// The gates of two channels.  v = -log a; where a is near 1 it is 1 - q, q = 1 - e^-v by a polynomial (the minimax one of fifth degree on
// [0, 1/2], 1.4e-9 of q): an exponential by itself is off by some 2^-23 of a, and a state that some thousand tokens stay in adds that
// up.  Beyond 1/2 a state is gone before errors add up.  1 - a^2 = q (1 + a) loses nothing in either case.
// MILD: v stays below 1/2 however far the gate opens (rate * softplus(decay) does), as it does where layers are initialised.
constexpr float kMild = 0.5f;
__device__ __forceinline__ Pair sigmoid(Pair v) { return each(each(v * both(-kLog2E), exp2_approx) + both(1.f), rcp_approx); }
// 1 / sqrt(v), of the smallest normal number where v is less; of a NaN a NaN
__device__ __forceinline__ float inv_root(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00800000;" : "=f"(r) : "f"(v));
  return rsqrt_approx(r);
}

__device__ __forceinline__ float not_above_zero(float v) {   // (a NaN stays one)
  float r;
  asm("min.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
  return r;
}

template <bool MILD>
struct Gates {
  Pair sr, v, a, om;
  __device__ __forceinline__ Gates(Pair k, Pair r) {
    const Pair one = both(1.f);
    sr = sigmoid(r);
    v = k * sr;
    Pair p = fma(both(-0.001121634905f), v, both(0.008187385975f));
    p = fma(p, v, both(-0.04162908913f));
    p = fma(p, v, both(0.1666622408f));
    p = fma(p, v, both(-0.4999998075f));
    p = fma(p, v, both(0.9999999986f));
    Pair q = p * v;
    a = fma(q, both(-1.f), one);
    if constexpr (!MILD) {
      const float2 vv = halves(v), e = halves(each(v * both(-kLog2E), exp2_approx)), qq = halves(q), aa = halves(a);
      const bool m0 = vv.x < kMild, m1 = vv.y < kMild;
      q = pair(m0 ? qq.x : 1.f - e.x, m1 ? qq.y : 1.f - e.y);
      a = pair(m0 ? aa.x : e.x, m1 ? aa.y : e.y);
    }
    om = q * (a + one);
  }
  // 1 / sqrt(1 - a^2); where a is 1 a large number, which comes with factors that are zero
  __device__ __forceinline__ Pair inv() const { return each(om, inv_root); }
};

// Pairs of a run or a tile, of a lane's two channels.
struct Share {
  Pair P, q;
};
__device__ __forceinline__ Pair pass(Share f, Pair s) {
  const float2 P = halves(f.P), q = halves(f.q), h = halves(s);
  return pair(pass(P.x, q.x, h.x), pass(P.y, q.y, h.y));
}
// `s` through shares first, first + step, .. (n of them).  One multiply-add each unless that gives a NaN, which it does not where
// infinities are left out by a reset or an underflow: then by the rule.
template <typename At>
__device__ __forceinline__ Pair through(Pair s, int n, At at) {
  Pair r = s;
#pragma unroll 4
  for (int v = 0; v < n; ++v) {
    const Share f = at(v);
    r = fma(f.P, r, f.q);
  }
  const float2 h = halves(r);
  if (isnan(h.x) || isnan(h.y)) {
    r = s;
    for (int v = 0; v < n; ++v) r = pass(at(v), r);
  }
  return r;
}
__device__ __forceinline__ bool is_fresh(Pair P) { return P.v == two_words(kFresh, kFresh); }

template <int RUNS, int SIDES>
struct Shared {
  Share run[2][SIDES][RUNS][32];    // of the runs, tiles in turn; the gradient's other side is that of the way back
  Share seen[RUNS][32];             // of the tiles before this one, the nearest first
  int4 which[2];                    // place in its sequence (-1: there is no tile left), unit, strip, batch entry
  int dead;                         // a wait ran out: no further one, and no further tile
  alignas(8) uint64_t full[2];
  alignas(16) float rate[2][kStrip], enter[2][kStrip];   // of the tiles' channels: rates, and (gradient) the states entering them
};

struct Maps {
  CUtensorMap at[4];
};

// Takes the next tile's number and sends for its inputs (one thread).
template <typename T, bool TMA, int N, int TILE>
__device__ __forceinline__ void send_for(const Scan& p, const Maps& maps, int4* which, uint64_t* full, unsigned turn, T* stage, bool backwards,
                                         float* rate, float* enter) {
  const unsigned t = p.tiles == 1 ? blockIdx.x + turn * gridDim.x : atomicAdd(p.counter, 1u) + 1u;
  if (t >= p.total) {
    which->x = -1;
    ptx::mbar_arrive(full);
    return;
  }
  const unsigned units = (unsigned)p.strips * p.batch;
  const int place = (int)(t / units), unit = (int)(t % units), strip = unit % p.strips, b = unit / p.strips;
  *which = make_int4(place, unit, strip, b);
  if (!TMA) {
    ptx::mbar_arrive(full);
    return;
  }
  const int k = backwards ? p.tiles - 1 - place : place;
  const uint32_t rates = p.rates ? kStrip * 4 : 0, states = p.enter_ahead ? (uint32_t)min(kStrip, p.channels - strip * kStrip) * 4 : 0;
  ptx::mbar_expect_tx(full, N * TILE * kStrip * (uint32_t)sizeof(T) + rates + states);
  auto numbers = [&](float* to, const float* from, uint32_t bytes) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ptx::smem_u32(to)), "l"(from), "r"(bytes),
                 "r"(ptx::smem_u32(full)) : "memory");
  };
  if (rates) numbers(rate, p.rates + strip * kStrip, rates);
  if (states) numbers(enter, p.pieces + ((int64_t)b * p.npieces + k) * p.channels + strip * kStrip, states);
#pragma unroll
  for (int n = 0; n < N; ++n)
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                     ptx::smem_u32(stage + n * TILE * kStrip)),
                 "l"(&maps.at[n]), "r"(ptx::smem_u32(full)), "r"(strip * kStrip), "r"(k * TILE), "r"(b)
                 : "memory");
}

template <typename S>
__device__ __forceinline__ void wait_for(const Scan& p, S& sh, uint64_t* full, unsigned parity) {
  if (ptx::mbar_try_wait(full, parity)) return;
  const long long t0 = clock64();
  while (!ptx::mbar_try_wait(full, parity)) {
    if (*(volatile int*)&sh.dead) return;
    if (clock64() - t0 > p.wait_clocks) {
      *(volatile int*)&sh.dead = 1;
      if (p.status) *p.status = STATUS_WAIT_TIMEOUT_TMA;
      return;
    }
  }
}

// Behind a wait that ran out the CTA leaves, once its own transfers have ended or the limit has passed again (one thread).
template <typename S>
__device__ __forceinline__ void drain(const Scan& p, S& sh, unsigned turn) {
  const long long t0 = clock64();
  for (unsigned t = turn; t < turn + 2; ++t)
    while (!ptx::mbar_try_wait(&sh.full[t & 1], t >> 1 & 1) && clock64() - t0 < p.wait_clocks) {
    }
}

// One operand's tile where TMA cannot read it (rows that do not start on 16 bytes), by all threads: fp32 by copies that are waited for
// later, 16-bit numbers, which no asynchronous copy takes one by one, through registers.
template <typename T, int TILE, int RUNS>
__device__ __forceinline__ void fill(T* to, const void* from, int b, int t0, int seqlen, const int64_t* st, int c, int channels) {
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const T* at = static_cast<const T*>(from) + b * st[0] + (int64_t)(t0 + w) * st[1] + c + lane;
  constexpr int kRows = TILE / RUNS, kBatch = 4;
#pragma unroll
  for (int r0 = 0; r0 < kRows; r0 += kBatch) {
    T v[kBatch][2];
#pragma unroll
    for (int r = 0; r < kBatch; ++r, at += RUNS * st[1]) {
      const int t = w + (r0 + r) * RUNS;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool there = t0 + t < seqlen && c + lane + 32 * e < channels;
        if constexpr (sizeof(T) == 4)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(ptx::smem_u32(to + t * kStrip + lane + 32 * e)),
                       "l"(there ? at + 32 * e : static_cast<const T*>(from)), "r"(there ? 4 : 0) : "memory");
        else
          v[r][e] = there ? at[32 * e] : Cvt<T>::from_f(0.f);
      }
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int r = 0; r < kBatch; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) to[(w + (r0 + r) * RUNS) * kStrip + lane + 32 * e] = v[r][e];
    }
  }
}

// Tokens of a run that are marked, a bit each.
template <int L>
__device__ __forceinline__ unsigned marks_of(const Scan& p, int b, int t0, int here) {
  if (!p.reset) return 0;
  const int t = threadIdx.x % 32;
  return __ballot_sync(~0u, t < here && p.reset[b * p.ms[0] + (int64_t)(t0 + t) * p.ms[1]]);
}

// The share of the whole tile, runs in their order (or, for the way back, from the last to the first).
template <int RUNS>
__device__ __forceinline__ Share whole(const Share (&run)[RUNS][32], bool backwards) {
  const int lane = threadIdx.x % 32;
  auto at = [&](int v) { return run[backwards ? RUNS - 1 - v : v][lane]; };
  Share all = {both(1.f), through(both(0.f), RUNS, at)};
  bool f0 = false, f1 = false;
#pragma unroll
  for (int v = 0; v < RUNS; ++v) {
    const Pair P = at(v).P;
    f0 |= (unsigned)P.v == kFresh;
    f1 |= (unsigned)(P.v >> 32) == kFresh;
    all.P = all.P * P;
  }
  const float2 P = halves(all.P);
  const float fresh = __uint_as_float(kFresh);
  all.P = pair(f0 ? fresh : P.x, f1 ? fresh : P.y);
  return all;
}

__device__ __forceinline__ void publish(const Scan& p, int64_t tile, Share f) {
  const float2 P = halves(f.P), q = halves(f.q);
  unsigned long long* at = p.pairs + tile * kStrip + 2 * (threadIdx.x % 32);
  store_word(at, two_words(word(P.x), __float_as_uint(q.x)));
  store_word(at + 1, two_words(word(P.y), __float_as_uint(q.y)));
}
__device__ __forceinline__ void publish(const Scan& p, int64_t tile, Pair s) {
  const float2 h = halves(s);
  store_word(p.states + tile * (kStrip / 2) + threadIdx.x % 32, two_words(word(h.x), word(h.y)));
}

// What stands before tile `k` of the unit, into sh.seen: warp w looks at tile k - 1 - w, for its state or else its pair; the farthest
// one waits for the state, so that one look is enough.
template <int RUNS, int SIDES>
__device__ __forceinline__ void look_back(const Scan& p, Shared<RUNS, SIDES>& sh, int64_t first, int k) {
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  if (w >= k) return;
  const int64_t tile = first + k - 1 - w;
  const unsigned long long *at = p.pairs + tile * kStrip + 2 * lane, *state = p.states + tile * (kStrip / 2) + lane;
  unsigned long long s, p0 = ~0ull, p1 = ~0ull;
  auto there = [](unsigned long long v) { return (unsigned)v != kNone && (unsigned)(v >> 32) != kNone; };
  long long t0 = 0;
  while (true) {
    s = load_word(state);
    if (w != RUNS - 1) {
      p0 = load_word(at);
      p1 = load_word(at + 1);
    }
    if (there(s) || ((unsigned)p0 != kNone && (unsigned)p1 != kNone)) break;
    if (*(volatile int*)&sh.dead) break;
    if (t0 == 0) t0 = clock64();
    if (clock64() - t0 > p.wait_clocks) {
      *(volatile int*)&sh.dead = 1;
      if (p.status) *p.status = STATUS_WAIT_TIMEOUT_LOOK_BACK;
      break;
    }
    __nanosleep(20);
  }
  auto lo = [](unsigned long long v) { return __uint_as_float((unsigned)v); };
  auto hi = [](unsigned long long v) { return __uint_as_float((unsigned)(v >> 32)); };
  const float fresh = __uint_as_float(kFresh);
  sh.seen[w][lane] = there(s) ? Share{both(fresh), pair(lo(s), hi(s))} : Share{pair(lo(p0), lo(p1)), pair(hi(p0), hi(p1))};
}

// The state entering a tile from what look_back() saw: from the nearest place that nothing before it matters to.
template <int RUNS, int SIDES>
__device__ __forceinline__ Pair fold_seen(const Shared<RUNS, SIDES>& sh, int k) {
  const int n = min(k, RUNS), lane = threadIdx.x % 32;
  int w = 0;
  while (w < n - 1 && !is_fresh(sh.seen[w][lane].P)) ++w;
  return through(both(0.f), w + 1, [&](int v) { return sh.seen[w - v][lane]; });
}

constexpr size_t stage_numbers(int n, int tile) { return (size_t)n * tile * kStrip; }

__device__ __forceinline__ Pair own_pair(const float* strip) {   // of a strip's numbers this lane's two
  const float2 f = *reinterpret_cast<const float2*>(strip + 2 * (threadIdx.x % 32));
  return pair(f.x, f.y);
}

// Lane l of a warp works on channels 2 l and 2 l + 1 of the strip.
struct Lane {
  int c;
  bool ok0, ok1;
  __device__ __forceinline__ Lane(int strip, int channels) {
    c = strip * kStrip + 2 * (threadIdx.x % 32);
    ok0 = c < channels;
    ok1 = c + 1 < channels;
  }
  __device__ __forceinline__ Pair get(const float* row) const { return pair(ok0 ? row[c] : 0.f, ok1 ? row[c + 1] : 0.f); }
  __device__ __forceinline__ void put(float* row, Pair v) const {
    const float2 h = halves(v);
    if (ok0) row[c] = h.x;
    if (ok1) row[c + 1] = h.y;
  }
  __device__ __forceinline__ Pair rates(const Scan& p) const {
    if (p.rates) {
      const float2 f = *reinterpret_cast<const float2*>(p.rates + c);
      return pair(f.x, f.y);
    }
    return pair(ok0 ? decay_rate(p.rate, p.decay[c]) : 0.f, ok1 ? decay_rate(p.rate, p.decay[c + 1]) : 0.f);
  }
  // two channels of an output's row, at once where the row starts on their boundary
  template <typename T, bool TMA>
  __device__ __forceinline__ void store(T* row, Pair v) const {
    const float2 h = halves(v);
    const typename Two<T>::Raw raw = Two<T>::down(h.x, h.y);
    if constexpr (TMA) {
      if (ok0) *reinterpret_cast<typename Two<T>::Raw*>(row) = raw;   // (channels are even)
    } else {
      if (ok0) row[0] = Two<T>::lo(raw);
      if (ok1) row[1] = Two<T>::hi(raw);
    }
  }
};

// TMA: every tensor's rows start on 16 bytes.
template <typename T, bool TMA>
__global__ void __launch_bounds__(32 * Geometry<T, false>::kRuns, Geometry<T, false>::kCtas)
gated_scan_kernel(const __grid_constant__ Scan p, const __grid_constant__ Maps maps) {
  using Raw = typename Two<T>::Raw;
  constexpr int L = Geometry<T, false>::kRun, kRuns = Geometry<T, false>::kRuns, kTile = tile_of(sizeof(T) == 4), kStage = (int)stage_numbers(3, kTile);
  static_assert(L * kRuns == kTile && kPiece % L == 0, "runs make a tile, pieces start at runs");
  extern __shared__ __align__(128) unsigned char smem[];
  T* const stages = reinterpret_cast<T*>(smem);
  Shared<kRuns, 1>& sh = *reinterpret_cast<Shared<kRuns, 1>*>(smem + 2 * kStage * sizeof(T));
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    sh.dead = 0;
    ptx::mbar_init(&sh.full[0], 1);
    ptx::mbar_init(&sh.full[1], 1);
    ptx::fence_mbar_init();
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (prepare_kernel's words and rates)
    asm volatile("fence.proxy.async;" ::: "memory");
    send_for<T, TMA, 3, kTile>(p, maps, &sh.which[0], &sh.full[0], 0, stages, false, sh.rate[0], nullptr);
  }
  __syncthreads();

  // without TMA: a tile's inputs by all threads, fp32 a tile ahead
  constexpr bool kLate = sizeof(T) == 4;
  auto fetch = [&](int s) {
    const int4 of = sh.which[s];
    if (of.x < 0) return;
    T* const to = stages + s * kStage;
    fill<T, kTile, kRuns>(to, p.x, of.w, of.x * kTile, p.seqlen, p.xs, of.z * kStrip, p.channels);
    fill<T, kTile, kRuns>(to + kTile * kStrip, p.i, of.w, of.x * kTile, p.seqlen, p.is, of.z * kStrip, p.channels);
    fill<T, kTile, kRuns>(to + 2 * kTile * kStrip, p.r, of.w, of.x * kTile, p.seqlen, p.rs, of.z * kStrip, p.channels);
  };
  if constexpr (!TMA && kLate) fetch(0);
  for (unsigned turn = 0;; ++turn) {
    const int s = turn & 1;
    T* const stage = stages + s * kStage;
    wait_for(p, sh, &sh.full[s], turn >> 1 & 1);
    if (p.inject && sh.which[s].x == 0 && sh.which[s].y == 0) break;   // (SsdGatedScanArgs::inject_lost_tile)
    if (p.early && turn == 0 && threadIdx.x == 32 * (kRuns - 1))   // (when every CTA has its first)
      send_for<T, TMA, 3, kTile>(p, maps, &sh.which[1], &sh.full[1], 1, stages + kStage, false, sh.rate[1], nullptr);
    const int4 which = sh.which[s];
    if (which.x < 0) break;
    const int k = which.x, unit = which.y, strip = which.z, b = which.w;
    const int t0 = k * kTile + w * L;
    const int here = min(L, p.seqlen - t0);   // tokens of this run that are there
    const Lane ln(strip, p.channels);
    const int64_t first = (int64_t)unit * p.tiles;
    if constexpr (!TMA) {
      if constexpr (kLate) asm volatile("cp.async.wait_all;" ::: "memory");
      else fetch(s);
      __syncthreads();
    }
    const Raw* const raw = reinterpret_cast<const Raw*>(stage + w * L * kStrip) + lane;
    auto rx = [&](int t) { return raw[t * 32]; };
    auto ri = [&](int t) { return raw[t * 32 + kTile * 32]; };
    auto rr = [&](int t) { return raw[t * 32 + 2 * kTile * 32]; };
    const unsigned marks = marks_of<L>(p, b, t0, here);
    const Pair rate = TMA && p.rates ? own_pair(sh.rate[s]) : ln.rates(p);

    Pair a[L], u[L];
    Share own = {both(1.f), both(0.f)};
    if (here > 0) {
      Raw least = ri(0);
#pragma unroll
      for (int t = 1; t < L; ++t) least = Two<T>::least(least, ri(t));
      const float2 kk = halves(rate), ll = Two<T>::up(least);
      // u = x om / (sqrt(om) (1 + e^-i)), one reciprocal square root of om (1 + e^-i)^2.  Where a run holds a gate that is all but shut that
      // would overflow: its gates are taken at kShut at least, times e^(i - kShut), which is 1 for the others (and in the general loop, as a loop
      // more costs the first one 2 %).  So a number is rounded in one way, whatever its neighbours are.
      constexpr float kShut = -40.f;
      const bool open = ll.x > kShut && ll.y > kShut;
      if (__all_sync(~0u, open && kk.x < kMild && kk.y < kMild)) {
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const Gates<true> g(rate, pair_of<T>(rr(t)));
          const Pair d = each(pair_of<T>(ri(t)) * both(-kLog2E), exp2_approx) + both(1.f);
          a[t] = g.a;
          u[t] = (pair_of<T>(rx(t)) * g.om) * each(g.om * (d * d), inv_root);
        }
      } else {
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const Gates<false> g(rate, pair_of<T>(rr(t)));
          const Pair i = pair_of<T>(ri(t)), less = each(each(i + both(-kShut), not_above_zero) * both(kLog2E), exp2_approx);
          const Pair d = each(each(i, [](float v) { return fmaxf(v, kShut); }) * both(-kLog2E), exp2_approx) + both(1.f);
          a[t] = g.a;
          u[t] = ((pair_of<T>(rx(t)) * less) * g.om) * each(g.om * (d * d), inv_root);
        }
      }
      if (here < L) {
#pragma unroll
        for (int t = 0; t < L; ++t)
          if (t >= here) a[t] = both(1.f), u[t] = both(0.f);
      }
      if (marks == 0) {
#pragma unroll
        for (int t = 0; t < L; ++t) {
          own.P = own.P * a[t];
          own.q = fma(a[t], own.q, u[t]);
        }
      } else {
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const bool cut = marks >> t & 1;
          own.P = own.P * a[t];
          own.q = fma(a[t], own.q, u[t]);
          if (cut) own = {both(__uint_as_float(kFresh)), u[t]};
        }
      }
    }
    auto& run = sh.run[s][0];
    run[w][lane] = own;
    if (__syncthreads_or(*(volatile int*)&sh.dead)) {
      if (threadIdx.x == 0) drain(p, sh, turn);
      break;
    }

    // (the inputs of this tile and of the one before have been read)
    if (threadIdx.x == 32 * (kRuns - 1)) {
      const int to = p.early ? s : s ^ 1;
      send_for<T, TMA, 3, kTile>(p, maps, &sh.which[to], &sh.full[to], p.early ? turn + 2 : turn + 1, stages + to * kStage, false, sh.rate[to],
                                      nullptr);
    }
    if constexpr (!TMA && kLate) {
      wait_for(p, sh, &sh.full[s ^ 1], (turn + 1) >> 1 & 1);
      fetch(s ^ 1);
    }
    const bool last = k == p.tiles - 1;
    Share tile = {};
    if (w == 0) {
      tile = whole(run, false);
      if (k > 0 && !last) publish(p, first + k, tile);
    }
    Pair h = both(0.f);
    if (k > 0) {
      look_back(p, sh, first, k);
      __syncthreads();
      h = fold_seen(sh, k);
    } else if (p.init) {
      h = ln.get(p.init + (int64_t)b * p.channels);
    }
    if (w == 0) {
      const Pair out = pass(tile, h);
      if (!last) publish(p, first + k, out);
      else if (p.fin) ln.put(p.fin + (int64_t)b * p.channels, out);
    }
    h = through(h, w, [&](int v) { return run[v][lane]; });
    if (here <= 0) continue;
    if (p.pieces && t0 % kPiece == 0) ln.put(p.pieces + ((int64_t)b * p.npieces + t0 / kPiece) * p.channels, h);

    T* y = static_cast<T*>(p.y) + b * p.ys[0] + (int64_t)t0 * p.ys[1] + ln.c;
    if (marks == 0 && here == L) {
#pragma unroll
      for (int t = 0; t < L; ++t, y += p.ys[1]) {
        h = fma(a[t], h, u[t]);
        ln.template store<T, TMA>(y, h);
      }
    } else {
#pragma unroll
      for (int t = 0; t < L; ++t, y += p.ys[1]) {
        h = fma(a[t], h, u[t]);
        if (marks >> t & 1) h = u[t];
        if (t < here) ln.template store<T, TMA>(y, h);
      }
    }
  }
}

// The gradient: the same walk from the last tile to the first, what passes from a token to the one before it being a[t] g[t].
// With w = b si, u = w x and m = a^2 / (1 - a^2):  dx = g w,  di = g u (1 - si),  dla = g (a h[t-1] - m u)  (without its first term at a
// reset),  dr = dla la (1 - sr),  and what decay's gradient sums up is dla la.
template <typename T, bool TMA>
__global__ void __launch_bounds__(32 * Geometry<T, true>::kRuns, Geometry<T, true>::kCtas)
gated_scan_grad_kernel(const __grid_constant__ Scan p, const __grid_constant__ Maps maps) {
  using Raw = typename Two<T>::Raw;
  constexpr int L = Geometry<T, true>::kRun, kRuns = Geometry<T, true>::kRuns, kStage = (int)stage_numbers(4, kTileGrad);
  static_assert(L * kRuns == kTileGrad, "runs make a tile");
  extern __shared__ __align__(128) unsigned char smem[];
  T* const stages = reinterpret_cast<T*>(smem);
  Shared<kRuns, 2>& sh = *reinterpret_cast<Shared<kRuns, 2>*>(smem + 2 * kStage * sizeof(T));
  __shared__ Pair sums[2][kRuns][32];
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    sh.dead = 0;
    ptx::mbar_init(&sh.full[0], 1);
    ptx::mbar_init(&sh.full[1], 1);
    ptx::fence_mbar_init();
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (prepare_kernel's words and rates)
    asm volatile("fence.proxy.async;" ::: "memory");
    send_for<T, TMA, 4, kTileGrad>(p, maps, &sh.which[0], &sh.full[0], 0, stages, true, sh.rate[0], sh.enter[0]);
  }
  __syncthreads();

  unsigned turn = 0;
  float* part = nullptr;   // where the sums of the tile before belong
  auto leave_sums = [&](int s) {   // (behind a barrier)
    if (part && w == 0) {
      Pair v = sums[s][0][lane];
#pragma unroll
      for (int n = 1; n < kRuns; ++n) v = v + sums[s][n][lane];
      *reinterpret_cast<float2*>(part) = halves(v);
    }
  };
  constexpr bool kLate = sizeof(T) == 4;
  auto fetch = [&](int s) {
    const int4 of = sh.which[s];
    if (of.x < 0) return;
    constexpr int n = kTileGrad * kStrip;
    T* const to = stages + s * kStage;
    const int at = (p.tiles - 1 - of.x) * kTileGrad;
    fill<T, kTileGrad, kRuns>(to, p.x, of.w, at, p.seqlen, p.xs, of.z * kStrip, p.channels);
    fill<T, kTileGrad, kRuns>(to + n, p.i, of.w, at, p.seqlen, p.is, of.z * kStrip, p.channels);
    fill<T, kTileGrad, kRuns>(to + 2 * n, p.r, of.w, at, p.seqlen, p.rs, of.z * kStrip, p.channels);
    fill<T, kTileGrad, kRuns>(to + 3 * n, p.dy, of.w, at, p.seqlen, p.dys, of.z * kStrip, p.channels);
  };
  if constexpr (!TMA && kLate) fetch(0);
  for (;; ++turn) {
    const int s = turn & 1;
    T* const stage = stages + s * kStage;
    wait_for(p, sh, &sh.full[s], turn >> 1 & 1);
    if (p.inject && sh.which[s].x == 0 && sh.which[s].y == 0) break;   // (SsdGatedScanArgs::inject_lost_tile)
    const int4 which = sh.which[s];
    if (which.x < 0) break;
    const int kb = which.x, k = p.tiles - 1 - kb, unit = which.y, strip = which.z, b = which.w;
    const int t0 = k * kTileGrad + w * L;
    const int here = min(L, p.seqlen - t0);
    const Lane ln(strip, p.channels);
    const int64_t first = (int64_t)unit * p.tiles;
    if constexpr (!TMA) {
      if constexpr (kLate) asm volatile("cp.async.wait_all;" ::: "memory");
      else fetch(s);
      __syncthreads();
    }
    const Raw* const raw = reinterpret_cast<const Raw*>(stage + w * L * kStrip) + lane;
    constexpr int kNext = kTileGrad * 32;
    auto x = [&](int t) { return pair_of<T>(raw[t * 32]); };
    auto ri = [&](int t) { return pair_of<T>(raw[t * 32 + kNext]); };
    auto rr = [&](int t) { return pair_of<T>(raw[t * 32 + 2 * kNext]); };
    auto dy = [&](int t) { return pair_of<T>(raw[t * 32 + 3 * kNext]); };
    const unsigned marks = marks_of<L>(p, b, t0, here);
    // the state entering the tile
    Pair h = TMA && p.enter_ahead ? own_pair(sh.enter[s]) : ln.get(p.pieces + ((int64_t)b * p.npieces + k) * p.channels);
    const Pair rate = TMA && p.rates ? own_pair(sh.rate[s]) : ln.rates(p), minus = both(-1.f), one = both(1.f);

    Pair a[L], sr[L], si[L], wt[L], m[L];
    Share own = {both(1.f), both(0.f)};
    Pair c = both(0.f);
    if (here > 0) {
      auto gates = [&](auto mild) {
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const Gates<decltype(mild)::value> g(rate, rr(t));
          const Pair inv = g.inv();
          a[t] = g.a;
          sr[t] = g.sr;
          si[t] = sigmoid(ri(t));
          wt[t] = (g.om * inv) * si[t];
          const Pair ai = g.a * inv;
          m[t] = ai * ai;
        }
      };
      const float2 kk = halves(rate);
      if (__all_sync(~0u, kk.x < kMild && kk.y < kMild)) gates(std::true_type());
      else gates(std::false_type());
      if (here < L) {
#pragma unroll
        for (int t = 0; t < L; ++t)
          if (t >= here) a[t] = one, sr[t] = si[t] = wt[t] = m[t] = both(0.f);
      }
      if (marks == 0) {
#pragma unroll
        for (int t = 0; t < L; ++t) {
          own.P = own.P * a[t];
          own.q = fma(a[t], own.q, wt[t] * x(t));
        }
#pragma unroll
        for (int t = L - 1; t >= 0; --t) c = a[t] * (dy(t) + c);
      } else {
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const Pair u = wt[t] * x(t);
          own.P = own.P * a[t];
          own.q = fma(a[t], own.q, u);
          if (marks >> t & 1) own = {both(__uint_as_float(kFresh)), u};
        }
#pragma unroll
        for (int t = L - 1; t >= 0; --t) {
          c = a[t] * (dy(t) + c);
          if (marks >> t & 1) c = both(0.f);
        }
      }
    }
    auto &run = sh.run[s][0], &back = sh.run[s][1];
    run[w][lane] = own;
    back[w][lane] = {own.P, c};
    if (__syncthreads_or(*(volatile int*)&sh.dead)) {
      if (threadIdx.x == 0) drain(p, sh, turn);
      break;
    }

    // (the inputs of the tile before have been read)
    if (threadIdx.x == 32 * (kRuns - 1))
      send_for<T, TMA, 4, kTileGrad>(p, maps, &sh.which[s ^ 1], &sh.full[s ^ 1], turn + 1, stages + (s ^ 1) * kStage, true, sh.rate[s ^ 1], sh.enter[s ^ 1]);
    if constexpr (!TMA && kLate) {
      wait_for(p, sh, &sh.full[s ^ 1], (turn + 1) >> 1 & 1);
      fetch(s ^ 1);
    }
    leave_sums(s ^ 1);
    part = p.part + ((int64_t)b * p.tiles + k) * ((int64_t)p.strips * kStrip) + ln.c;
    const bool last = kb == p.tiles - 1;   // of the way back: the sequence's first
    Share tile = {};
    if (w == 0) {
      tile = whole(back, true);
      if (kb > 0 && !last) publish(p, first + kb, tile);
    }
    c = both(0.f);
    if (kb > 0) {
      look_back(p, sh, first, kb);
      __syncthreads();
      c = fold_seen(sh, kb);
    } else if (p.dfinal) {
      c = ln.get(p.dfinal + (int64_t)b * p.channels);
    }
    if (w == 0) {
      const Pair out = pass(tile, c);
      if (!last) publish(p, first + kb, out);
      else if (p.dinit) ln.put(p.dinit + (int64_t)b * p.channels, out);
    }
    h = through(h, w, [&](int v) { return run[v][lane]; });
    c = through(c, kRuns - 1 - w, [&](int v) { return back[kRuns - 1 - v][lane]; });

    Pair sum = both(0.f);
    // ALL: every token of the run is there and none is marked
    auto again = [&](auto all) {
      constexpr bool ALL = decltype(all)::value;
#pragma unroll
      for (int t = 0; t < L; ++t) {   // m becomes a h[t-1] - m u
        const Pair u = wt[t] * x(t);
        Pair before = a[t] * h;
        if (!ALL && (marks >> t & 1)) before = both(0.f);
        h = before + u;
        m[t] = fma(m[t] * minus, u, before);
      }
      T* dx = static_cast<T*>(p.dx) + b * p.dxs[0] + (int64_t)(t0 + L - 1) * p.dxs[1] + ln.c;
      T* di = static_cast<T*>(p.di) + b * p.dis[0] + (int64_t)(t0 + L - 1) * p.dis[1] + ln.c;
      T* dr = static_cast<T*>(p.dr) + b * p.drs[0] + (int64_t)(t0 + L - 1) * p.drs[1] + ln.c;
#pragma unroll
      for (int t = L - 1; t >= 0; --t, dx -= p.dxs[1], di -= p.dis[1], dr -= p.drs[1]) {
        const Pair g = dy(t) + c;
        const Pair dv = (g * m[t]) * (rate * sr[t]);   // -dla la
        const Pair gw = g * wt[t];
        sum = sum + dv;
        c = a[t] * g;
        if (!ALL && (marks >> t & 1)) c = both(0.f);
        if (ALL || t < here) {
          ln.template store<T, TMA>(dx, gw);
          ln.template store<T, TMA>(di, (gw * x(t)) * fma(si[t], minus, one));
          ln.template store<T, TMA>(dr, dv * fma(sr[t], one, minus));
        }
      }
    };
    if (marks == 0 && here == L) again(std::true_type());
    else if (here > 0) again(std::false_type());
    sums[s][w][lane] = sum;
  }
  __syncthreads();
  leave_sums((turn - 1) & 1);
}

// From the sum of -dla la: la is -rate softplus(decay) sr, so d la / d decay is la sigmoid(decay) / softplus(decay), a ratio that goes
// to 1 where both vanish.
struct FinishDecay {
  const float* decay;
  float* out;
  __device__ __forceinline__ void operator()(int c, float v) const {
    const float plus = decay_rate(1.f, decay[c]);
    out[c] = plus < 1e-30f ? -v : -v * (1.f / (1.f + expf(-decay[c])) / plus);
  }
};

// Ahead of a scan: sets its words, and works every channel's rate out.
__global__ void __launch_bounds__(256) prepare_kernel(uint4* words, int64_t n, const float* decay, float* rates, int channels, int padded, float rate) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = i0; i < n; i += step) words[i] = make_uint4(kNone, kNone, kNone, kNone);
  for (int64_t c = i0; c < padded; c += step) rates[c] = c < channels ? decay_rate(rate, decay[c]) : 0.f;
}

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
  if constexpr (V == 1) {   // (as one of two)
    const Gates<false> g(both(decay_rate(rate, dv[0])), both(Cvt<T>::to_f(rv[0])));
    const Pair u = (g.om * g.inv()) * both(sigmoid_approx(Cvt<T>::to_f(iv[0])) * Cvt<T>::to_f(xv[0]));
    sv[0] = halves(fma(g.a, both(sv[0]), u)).x;
    yv[0] = Cvt<T>::from_f(sv[0]);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const Gates<false> g(pair(decay_rate(rate, dv[e]), decay_rate(rate, dv[e + 1])), pair(Cvt<T>::to_f(rv[e]), Cvt<T>::to_f(rv[e + 1])));
      const Pair x2 = pair(Cvt<T>::to_f(xv[e]), Cvt<T>::to_f(xv[e + 1])), i2 = pair(Cvt<T>::to_f(iv[e]), Cvt<T>::to_f(iv[e + 1]));
      const float2 h = halves(fma(g.a, pair(sv[e], sv[e + 1]), (g.om * g.inv()) * (sigmoid(i2) * x2)));
      sv[e] = h.x;
      sv[e + 1] = h.y;
      yv[e] = Cvt<T>::from_f(h.x);
      yv[e + 1] = Cvt<T>::from_f(h.y);
    }
  }
  copy(state_out + (int64_t)b * channels + c, sv);
  copy(y + b * ys + c, yv);
}

int strips_of(int channels) { return (channels + kStrip - 1) / kStrip; }
int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

struct Sizes {
  int64_t tiles, units, words, rates, part;   // tiles of a sequence, sequences of 64 channels, bytes
};
Sizes sizes_of(const SsdGatedScanArgs& a, bool grad) {
  Sizes z;
  const int tile = grad ? kTileGrad : tile_of(a.dtype == SSD_DTYPE_F32);
  z.tiles = (a.seqlen + (int64_t)tile - 1) / tile;
  z.units = (int64_t)a.batch * strips_of(a.channels);
  z.words = z.tiles == 1 ? 0 : 256 + z.units * z.tiles * kStrip * 12;
  // (a CTA that works on one tile works its channels' rates out by itself)
  z.rates = z.tiles * z.units > 148 ? up256((int64_t)strips_of(a.channels) * kStrip * 4) : 0;
  z.part = grad ? z.units * z.tiles * kStrip * 4 : 0;
  return z;
}

int check(const SsdGatedScanArgs* a, bool grad) {
  if (!a) return SSD_ERR_NULL_POINTER;
  if (a->batch <= 0 || a->seqlen <= 0 || a->channels <= 0 || a->wait_limit_ms < 0 || !(a->rate > 0.f && a->rate < INFINITY)) return SSD_ERR_BAD_SHAPE;
  if (a->dtype != SSD_DTYPE_F32 && a->dtype != SSD_DTYPE_F16 && a->dtype != SSD_DTYPE_BF16) return SSD_ERR_UNSUPPORTED;
  if (a->seqlen > 0x7fffff00 || a->channels > 0x7fffff00) return SSD_ERR_TOO_LARGE;   // (tiles and strips round them up)
  const Sizes z = sizes_of(*a, grad);
  if (z.tiles * z.units > 0x7fffffff) return SSD_ERR_TOO_LARGE;
  return SSD_OK;
}

// [b,s,d] as TMA sees it, a box of 64 channels of `rows` tokens; what lies outside reads as zero.
template <typename T>
bool operand_map(CUtensorMap* map, const void* base, const SsdGatedScanArgs& a, const int64_t (&st)[2], int rows) {
  const tc::EncodeFn encode = tc::encode_fn();
  if (!encode) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a.channels, (cuuint64_t)a.seqlen, (cuuint64_t)a.batch};
  const cuuint64_t strides[2] = {(cuuint64_t)st[1] * sizeof(T), (cuuint64_t)st[0] * sizeof(T)};
  const cuuint32_t box[3] = {kStrip, (cuuint32_t)rows, 1}, each[3] = {1, 1, 1};
  const CUtensorMapDataType type = a.dtype == SSD_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : a.dtype == SSD_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(map, type, 3, const_cast<void*>(base), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
  p.inject = a.inject_lost_tile;
  p.batch = a.batch; p.seqlen = a.seqlen; p.channels = a.channels;
  p.strips = strips_of(a.channels); p.tiles = (int)z.tiles; p.npieces = (a.seqlen + kPiece - 1) / kPiece;
  char* ws = static_cast<char*>(a.workspace);
  if (z.words) {
    p.counter = reinterpret_cast<unsigned*>(ws);
    p.pairs = reinterpret_cast<unsigned long long*>(ws + 256);
    p.states = reinterpret_cast<unsigned long long*>(ws + 256 + z.units * z.tiles * kStrip * 8);
  }
  float* const rates = z.rates ? reinterpret_cast<float*>(ws + up256(z.words)) : nullptr;
  p.rates = rates;
  p.part = reinterpret_cast<float*>(ws + up256(z.words) + z.rates);
  // by TMA: every row starts on 16 bytes
  bool tma = a.channels * sizeof(T) % 16 == 0;
  auto strides = [&](int64_t (&to)[2], const int64_t (&from)[2], const void* at) {
    for (int d = 0; d < 2; ++d) {
      to[d] = (d == 0 ? a.batch : a.seqlen) == 1 ? 16 : from[d];   // (the stride of a single one may be anything)
      const int64_t bytes = to[d] * (int64_t)sizeof(T);
      tma = tma && bytes % 16 == 0 && bytes > 0 && bytes < (int64_t)1 << 40;
    }
    tma = tma && reinterpret_cast<uintptr_t>(at) % 16 == 0;
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
  p.total = (unsigned)(z.tiles * z.units);
  Maps maps = {};
  if (tma) {
    const int tile = grad ? kTileGrad : tile_of(sizeof(T) == 4);
    tma = operand_map<T>(&maps.at[0], a.x, a, p.xs, tile) && operand_map<T>(&maps.at[1], a.input_gate, a, p.is, tile) &&
          operand_map<T>(&maps.at[2], a.decay_gate, a, p.rs, tile) &&
          (!grad || operand_map<T>(&maps.at[3], a.dy, a, p.dys, tile));
  }
  using Fwd = Geometry<T, false>;
  using Bwd = Geometry<T, true>;
  const unsigned grid = std::min(p.total, 148u * (grad ? Bwd::kCtas : Fwd::kCtas));
  // Where many tiles of one sequence are worked on at a time their numbers are taken as late as their inputs allow, so that a tile does not
  // wait for one that is started after it; with fewer the inputs' way counts for more.  One sequence of 2^26 numbers bf16 (2^25 fp32), us, taken
  // two tiles ahead and late: 9.25 tiles at a time 138.5 131.7 (109.7 104.4), 7 132.0 130.0 (104.7 101.7), 6 129.9 128.5 (103.0 100.8), 5 127.4 126.7
  // (100.3 100.1), 4.6 125.8 125.3 (99.6 100.1), 4 124.8 125.0 (98.2 100.2), 3 122.4 124.0 (95.8 100.2), 2 119.9 121.5 (92.4 98.6).
  // (Copies by threads are late ones.)
  p.early = 2 * (int64_t)grid <= 9 * z.units && (tma || sizeof(T) == 2);
  p.enter_ahead = grad && tma && reinterpret_cast<uintptr_t>(a.pieces) % 16 == 0 && a.channels % 4 == 0;
  auto go = [&](auto kernel, int threads, size_t smem) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return (int)SSD_ERR_CUDA;
    if (!z.words && !z.rates) return launch(kernel, grid, threads, smem, stream, p, maps);
    const int64_t n = z.words / 16, padded = z.rates ? (int64_t)p.strips * kStrip : 0;
    const unsigned blocks = (unsigned)std::min<int64_t>(148 * 4, (std::max(n, padded) + 255) / 256);
    if (const int rc = launch(prepare_kernel, blocks, 256, 0, stream, reinterpret_cast<uint4*>(ws), n, a.decay, rates, a.channels, (int)padded, a.rate))
      return rc;
    return launch_early(kernel, grid, threads, smem, stream, p, maps);
  };
  if (!grad) {
    const size_t smem = 2 * stage_numbers(3, tile_of(sizeof(T) == 4)) * sizeof(T) + sizeof(Shared<Fwd::kRuns, 1>);
    return tma ? go(gated_scan_kernel<T, true>, 32 * Fwd::kRuns, smem) : go(gated_scan_kernel<T, false>, 32 * Fwd::kRuns, smem);
  }
  const size_t smem = 2 * stage_numbers(4, kTileGrad) * sizeof(T) + sizeof(Shared<Bwd::kRuns, 2>);
  if (const int rc = tma ? go(gated_scan_grad_kernel<T, true>, 32 * Bwd::kRuns, smem) : go(gated_scan_grad_kernel<T, false>, 32 * Bwd::kRuns, smem)) return rc;
  return launch_column_sum(p.part, a.batch * z.tiles, (int64_t)p.strips * kStrip, a.channels, FinishDecay{a.decay, a.ddecay}, stream);
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
  return (size_t)(ssd::up256(z.words) + z.rates + z.part);
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
