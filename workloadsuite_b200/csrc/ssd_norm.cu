// RMS norms between blocks and their gradients (formulas: ssd_b200.h).
// A row (of a group) is one warp's or one CTA's, eight numbers a thread and step, worked on in registers (but for what ptxas spills of the
// gradients' sixteen and thirty-two numbers a thread, up to 1.1 KB): every input is read once, every output written once.  CTAs stay and take rows in turn; the inputs of the next rows are on their way (cp.async) while one is worked on, each
// thread's into places that nobody else reads, so that waiting for its own copies is all the synchronisation they need.
// The gradients against vectors are sums over rows: a CTA adds those of its rows up in registers and leaves
// them to column_sum_kernel, so that their order is fixed.
// Bound: HBM and, between a row's halves, its sums.  16 384 rows of 2 048 fp16 with residual: 52 us (5.2 TB/s, 80 % of the copy bandwidth), gradient 51;
// gated, 8 192 rows of 8 x 1 024 bf16: 68 (91 %) and 124 (84 %).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "vec_io.cuh"

namespace ssd {
namespace {

// Eight numbers of a row: neighbours (VEC: 16-byte pieces), or blockDim.x apart where rows do not start on such a boundary.
// Those behind the row's end read as zero.
template <bool VEC>
__device__ __forceinline__ int place(int it, int e) {
  return VEC ? (it * (int)blockDim.x + (int)threadIdx.x) * 8 + e : (it * 8 + e) * (int)blockDim.x + (int)threadIdx.x;
}
struct Eight {
  Pair v[4];
  __device__ __forceinline__ Pair& operator[](int e) { return v[e]; }
  __device__ __forceinline__ Pair operator[](int e) const { return v[e]; }
};
template <typename F>
__device__ __forceinline__ void four(F f) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f(e);
}
__device__ __forceinline__ Pair words_to_pair(uint32_t lo, uint32_t hi) { return pair(__uint_as_float(lo), __uint_as_float(hi)); }
template <typename T>
__device__ __forceinline__ Eight widen(const uint4& a, const uint4& b) {
  Eight r;
  if constexpr (sizeof(T) == 2) {
    r[0] = pair_of<T>(a.x); r[1] = pair_of<T>(a.y); r[2] = pair_of<T>(a.z); r[3] = pair_of<T>(a.w);
  } else {
    r[0] = words_to_pair(a.x, a.y); r[1] = words_to_pair(a.z, a.w); r[2] = words_to_pair(b.x, b.y); r[3] = words_to_pair(b.z, b.w);
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ Eight get8(const T* __restrict__ row, int it, int d) {
  if constexpr (VEC) {
    const int at = place<true>(it, 0);
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (at < d) {
      a = *reinterpret_cast<const uint4*>(row + at);
      if (sizeof(T) == 4) b = *reinterpret_cast<const uint4*>(row + at + 4);
    }
    return widen<T>(a, b);
  } else {
    Eight r;
    four([&](int e) {
      const int i0 = place<false>(it, 2 * e), i1 = place<false>(it, 2 * e + 1);
      r[e] = pair(i0 < d ? Cvt<T>::to_f(row[i0]) : 0.f, i1 < d ? Cvt<T>::to_f(row[i1]) : 0.f);
    });
    return r;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void put8(T* row, int it, int d, const Eight& v) {
  if constexpr (VEC) {
    const int at = place<true>(it, 0);
    if (at < d) {
      if constexpr (sizeof(T) == 2) {
        auto word = [&](int e) { return Two<T>::down(halves(v[e]).x, halves(v[e]).y); };
        *reinterpret_cast<uint4*>(row + at) = make_uint4(word(0), word(1), word(2), word(3));
      } else {
        const float2 a = halves(v[0]), b = halves(v[1]), c = halves(v[2]), e = halves(v[3]);
        *reinterpret_cast<float4*>(row + at) = make_float4(a.x, a.y, b.x, b.y);
        *reinterpret_cast<float4*>(row + at + 4) = make_float4(c.x, c.y, e.x, e.y);
      }
    }
  } else {
    four([&](int e) {
      const float2 f = halves(v[e]);
      const int i0 = place<false>(it, 2 * e), i1 = place<false>(it, 2 * e + 1);
      if (i0 < d) row[i0] = Cvt<T>::from_f(f.x);
      if (i1 < d) row[i1] = Cvt<T>::from_f(f.y);
    });
  }
}

// A vector of d numbers, fp32 or T.
struct Vector {
  const void* p;
  int in_dtype;
  template <typename T, bool VEC>
  __device__ __forceinline__ Eight get(int first, int it, int d) const {
    return in_dtype ? get8<T, VEC>(static_cast<const T*>(p) + first, it, d) : get8<float, VEC>(static_cast<const float*>(p) + first, it, d);
  }
};

// Sum over the threads of a row, in all of them, in a fixed order.  `turn` alternates between two places, so that one barrier a sum is
// enough.
struct RowSum {
  float (*place)[16];   // [2]: up to sixteen warps
  int turn;
  __device__ __forceinline__ float operator()(Pair s) {
    const float2 h = halves(s);
    float v = h.x + h.y;
#pragma unroll
    for (int k = 16; k > 0; k /= 2) v += __shfl_xor_sync(~0u, v, k);
    if (blockDim.x > 32) {
      float* const at = place[turn];
      turn ^= 1;
      if (threadIdx.x % 32 == 0) at[threadIdx.x / 32] = v;
      __syncthreads();
      v = 0.f;
      for (int w = 0; w < (int)blockDim.x / 32; w += 4) {   // (places of warps that are not there hold zero)
        const float4 a = *reinterpret_cast<const float4*>(at + w);
        v += (a.x + a.y) + (a.z + a.w);
      }
    }
    return v;
  }
};
__device__ __forceinline__ void clear(float (&sums)[2][16]) {
  const int t = threadIdx.y * blockDim.x + threadIdx.x;
  if (t < 32) sums[t / 16][t % 16] = 0.f;
  __syncthreads();
}

// One operand's rows, as a CTA goes through them.
template <typename T>
struct Rows {
  T* at;
  int64_t by;
  __device__ __forceinline__ Rows(T* p, int64_t stride)
      : at(p ? p + ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * stride : nullptr), by((int64_t)gridDim.x * blockDim.y * stride) {}
  __device__ __forceinline__ T* next() {
    T* const r = at;
    at += by;
    return r;
  }
};
template <typename T>
__device__ __forceinline__ Rows<const T> rows_in(const void* p, int64_t stride, int first = 0) {
  return Rows<const T>(p ? static_cast<const T*>(p) + first : nullptr, stride);
}
template <typename T>
__device__ __forceinline__ Rows<T> rows_out(void* p, int64_t stride, int first = 0) {
  return Rows<T>(p ? static_cast<T*>(p) + first : nullptr, stride);
}

struct Norm {
  const void *x, *z, *res, *dy, *dres_out;
  void *y, *res_out, *dx, *dz, *dres;
  Vector w, post, scale;
  float *inv, *inv_post, *part;
  int64_t rows, xs, zs, rs, ys, ros, dys, dros, dxs, dzs, drs;
  int d, groups, norm_first, vectors;   // d: of a group; vectors: of d * groups partial sums a row of `part` holds
  float eps, inv_d;
  // what the norm behind the block and the scale multiply by
  template <typename T, bool VEC>
  __device__ __forceinline__ Eight outer(int it) const {
    if (!post.p) return scale.get<T, VEC>(0, it, d);
    Eight o = post.get<T, VEC>(0, it, d);
    if (scale.p) {
      const Eight s = scale.get<T, VEC>(0, it, d);
      four([&](int e) { o[e] = o[e] * s[e]; });
    }
    return o;
  }
};

// The inputs of the rows to come: a thread's sixteen-byte pieces (PIECES a row), STAGES rows ahead.
template <int PIECES, int STAGES>
struct Ahead {
  uint32_t base;
  __device__ __forceinline__ Ahead() {
    extern __shared__ __align__(16) unsigned char smem[];
    base = (uint32_t)__cvta_generic_to_shared(smem) + (threadIdx.y * blockDim.x + threadIdx.x) * 16;
  }
  __device__ __forceinline__ uint32_t at(int stage, int piece) const {
    return base + (uint32_t)((stage * PIECES + piece) * (int)(blockDim.x * blockDim.y) * 16);
  }
  // pieces first, first + 1 .. of a row's numbers of this thread
  template <typename T, int I>
  __device__ __forceinline__ void send(int stage, int first, const T* row, int d) const {
#pragma unroll
    for (int it = 0; it < I; ++it) {
      const int n = place<true>(it, 0);
      if (n < d) {
#pragma unroll
        for (int q = 0; q < (int)sizeof(T) / 2; ++q)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(stage, first + it * (int)sizeof(T) / 2 + q)), "l"(row + n + 8 * q / ((int)sizeof(T) / 2)) : "memory");
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ Eight get(int stage, int first, int it, int d) const {
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (place<true>(it, 0) < d) {
      auto load = [&](uint4& v, int q) {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at(stage, first + it * (int)sizeof(T) / 2 + q)) : "memory");
      };
      load(a, 0);
      if (sizeof(T) == 4) load(b, 1);
    }
    return widen<T>(a, b);
  }
};
// Rows ahead: fewer of large rows, as CTAs that do not fit cost more than a row ahead; where the widest CTA (512 threads) does not hold
// two, rows are read where they are needed.
constexpr int stages_of(int pieces) { return pieces <= 4 ? 4 : pieces <= 8 ? 3 : pieces <= 13 ? 2 : 0; }

// Goes through a CTA's rows (a row per warp, blockDim.y of them, or one per CTA): send(stage) asks for the next row's inputs, work(stage, row)
// takes them.
template <bool AHEAD, int STAGES, typename Send, typename Work>
__device__ __forceinline__ void for_rows(int64_t rows, Send send, Work work) {
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y, ahead = row;
  auto ask = [&](int stage) {
    if (ahead < rows) send(stage);
    ahead += step;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (AHEAD) {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) ask(s);
  }
  int stage = 0;
  for (; row < rows; row += step) {
    if constexpr (AHEAD) {
      ask(stage == 0 ? STAGES - 1 : stage - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    }
    work(stage, row);
    if (++stage == STAGES) stage = 0;
  }
  if constexpr (AHEAD) asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ float inv_rms(float sum, const Norm& p) { return rsqrtf(fmaf(sum, p.inv_d, p.eps)); }

// OUTER: with post_weight or scale.
template <typename T, typename R, int I, bool VEC, bool OUTER>
struct Forward {
  // Two sums a row (OUTER): what counts is how many rows an SM has in hand, and rows ahead take the room of CTAs (2 560 numbers, fp32
  // residual: 50 us for 8 192 rows without, 56 with).  One sum: 52 and 52 at 2 048, 91 and 98 at 8 192.
  static constexpr int kPieces = I * (int)(sizeof(T) + sizeof(R)) / 2, kStages = OUTER ? 0 : stages_of(kPieces);
  static constexpr bool kAhead = VEC && kStages > 0;
  static constexpr bool kKeep = I <= 2 && !OUTER;   // the weight stays in registers
};
template <typename T, typename R, int I, bool VEC, bool OUTER>
__global__ void __launch_bounds__(I == 1 ? 128 : 512) rms_norm_kernel(const Norm p) {
  using F = Forward<T, R, I, VEC, OUTER>;
  constexpr int kRes = I * (int)sizeof(T) / 2;
  __shared__ __align__(16) float sums[2][16];
  clear(sums);
  RowSum row_sum{sums, 0};
  const Ahead<F::kPieces, F::kStages> ahead;
  Eight w[I];
  if constexpr (F::kKeep) {
#pragma unroll
    for (int it = 0; it < I; ++it) w[it] = p.w.get<T, VEC>(0, it, p.d);
  }
  auto x = rows_in<T>(p.x, p.xs);
  auto res = rows_in<R>(p.res, p.rs);
  auto res_out = rows_out<R>(p.res_out, p.ros);
  auto y = rows_out<T>(p.y, p.ys);
  for_rows<F::kAhead, F::kStages>(
      p.rows,
      [&](int s) {
        ahead.template send<T, I>(s, 0, x.next(), p.d);
        if (p.res) ahead.template send<R, I>(s, kRes, res.next(), p.d);
      },
      [&](int s, int64_t row) {
        Eight v[I];
        const T* const xr = F::kAhead ? nullptr : x.next();
#pragma unroll
        for (int it = 0; it < I; ++it) v[it] = F::kAhead ? ahead.template get<T>(s, 0, it, p.d) : get8<T, VEC>(xr, it, p.d);
        if constexpr (OUTER) {
          float inv = 1.f;
          if (p.post.p) {
            Pair ss = both(0.f);
#pragma unroll
            for (int it = 0; it < I; ++it) four([&](int e) { ss = fma(v[it][e], v[it][e], ss); });
            inv = inv_rms(row_sum(ss), p);
            if (p.inv_post && threadIdx.x == 0) p.inv_post[row] = inv;
          }
#pragma unroll
          for (int it = 0; it < I; ++it) {
            const Eight ps = p.outer<T, VEC>(it);
            four([&](int e) { v[it][e] = v[it][e] * both(inv) * ps[e]; });
          }
        }
        if (p.res) {
          const R* const rr = F::kAhead ? nullptr : res.next();
          R* const ro = res_out.next();
#pragma unroll
          for (int it = 0; it < I; ++it) {
            const Eight old = F::kAhead ? ahead.template get<R>(s, kRes, it, p.d) : get8<R, VEC>(rr, it, p.d);
            four([&](int e) {   // as it is stored
              const float2 f = halves(old[e] + v[it][e]);
              v[it][e] = pair_of<R>(Two<R>::down(f.x, f.y));
            });
            put8<R, VEC>(ro, it, p.d, v[it]);
          }
        }
        Pair ss = both(0.f);
#pragma unroll
        for (int it = 0; it < I; ++it) four([&](int e) { ss = fma(v[it][e], v[it][e], ss); });
        const float inv = inv_rms(row_sum(ss), p);
        if (p.inv && threadIdx.x == 0) p.inv[row] = inv;
        T* const yr = y.next();
#pragma unroll
        for (int it = 0; it < I; ++it) {
          if constexpr (!F::kKeep) w[it] = p.w.get<T, VEC>(0, it, p.d);
          four([&](int e) { v[it][e] = v[it][e] * both(inv) * w[it][e]; });
          put8<T, VEC>(yr, it, p.d, v[it]);
        }
      });
}

// Partial sums of this warp's or CTA's rows.
template <int I, bool VEC>
__device__ __forceinline__ void leave(const Norm& p, int which, const Eight (&sum)[I]) {
  const int64_t all = (int64_t)p.d * p.groups;
  float* to = p.part + (((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * p.vectors + which) * all + (int64_t)blockIdx.y * p.d;
#pragma unroll
  for (int it = 0; it < I; ++it)
    four([&](int e) {
      const float2 f = halves(sum[it][e]);
      if (place<VEC>(it, 2 * e) < p.d) to[place<VEC>(it, 2 * e)] = f.x;
      if (place<VEC>(it, 2 * e + 1) < p.d) to[place<VEC>(it, 2 * e + 1)] = f.y;
    });
}

template <typename T, typename R, int I, bool VEC, bool OUTER>
struct Backward {
  static constexpr int kPieces = I * (int)(sizeof(T) + 2 * sizeof(R) + (OUTER ? sizeof(T) : 0)) / 2, kStages = stages_of(kPieces);
  static constexpr bool kAhead = VEC && kStages > 0;
  static constexpr bool kKeep = I <= 2;
};
template <typename T, typename R, int I, bool VEC, bool OUTER>
__global__ void __launch_bounds__(I == 1 ? 128 : 512) rms_norm_grad_kernel(const Norm p) {
  using F = Backward<T, R, I, VEC, OUTER>;
  constexpr int kOut = I * (int)sizeof(T) / 2, kIn = kOut + I * (int)sizeof(R) / 2, kX = kIn + I * (int)sizeof(R) / 2;
  __shared__ __align__(16) float sums[2][16];
  clear(sums);
  RowSum row_sum{sums, 0};
  const Ahead<F::kPieces, F::kStages> ahead;
  Eight dw[I], acc[I], w[I], ps[I];
#pragma unroll
  for (int it = 0; it < I; ++it) {
    four([&](int e) { dw[it][e] = acc[it][e] = both(0.f); });
    if constexpr (F::kKeep) {
      w[it] = p.w.get<T, VEC>(0, it, p.d);
      if constexpr (OUTER) ps[it] = p.outer<T, VEC>(it);
    }
  }
  auto dy = rows_in<T>(p.dy, p.dys), x = rows_in<T>(p.x, p.xs);
  auto of = p.res_out ? rows_in<R>(p.res_out, p.ros) : rows_in<R>(p.x, p.xs);   // (of x: R is T)
  auto dres_out = rows_in<R>(p.dres_out, p.dros);
  auto dres = rows_out<R>(p.dres, p.drs);
  auto dx = rows_out<T>(p.dx, p.dxs);
  float inv_now = 0.f, inv_post_now = 1.f;   // the next row's, asked for a row ahead
  auto rates = [&](int64_t row) {
    if (row >= p.rows) return;
    inv_now = p.inv[row];
    if (OUTER && p.post.p) inv_post_now = p.inv_post[row];
  };
  rates((int64_t)blockIdx.x * blockDim.y + threadIdx.y);
  for_rows<F::kAhead, F::kStages>(
      p.rows,
      [&](int s) {
        ahead.template send<T, I>(s, 0, dy.next(), p.d);
        ahead.template send<R, I>(s, kOut, of.next(), p.d);
        if (p.dres_out) ahead.template send<R, I>(s, kIn, dres_out.next(), p.d);
        if constexpr (OUTER) ahead.template send<T, I>(s, kX, x.next(), p.d);
      },
      [&](int s, int64_t row) {
        Eight g[I], v[I];
        const T* const gr = F::kAhead ? nullptr : dy.next();
        const R *const vr = F::kAhead ? nullptr : of.next(), *const ir = F::kAhead ? nullptr : dres_out.next();
        const T* const xr = F::kAhead ? nullptr : x.next();
        const float inv = inv_now, invp = inv_post_now;
        rates(row + (int64_t)gridDim.x * blockDim.y);
        Pair c = both(0.f);
#pragma unroll
        for (int it = 0; it < I; ++it) {
          if constexpr (F::kAhead) {
            g[it] = ahead.template get<T>(s, 0, it, p.d);
            v[it] = ahead.template get<R>(s, kOut, it, p.d);
          } else {
            g[it] = get8<T, VEC>(gr, it, p.d);
            v[it] = get8<R, VEC>(vr, it, p.d);
          }
          if constexpr (!F::kKeep) w[it] = p.w.get<T, VEC>(0, it, p.d);
          four([&](int e) {
            v[it][e] = v[it][e] * both(inv);
            dw[it][e] = fma(g[it][e], v[it][e], dw[it][e]);
            g[it][e] = g[it][e] * w[it][e];
            c = fma(g[it][e], v[it][e], c);
          });
        }
        const Pair mean = both(-row_sum(c) * p.inv_d);
        R* const dres_at = p.dres ? dres.next() : nullptr;
#pragma unroll
        for (int it = 0; it < I; ++it) {
          four([&](int e) { g[it][e] = both(inv) * fma(v[it][e], mean, g[it][e]); });
          if (p.dres_out) {
            const Eight in = F::kAhead ? ahead.template get<R>(s, kIn, it, p.d) : get8<R, VEC>(ir, it, p.d);
            four([&](int e) { g[it][e] = g[it][e] + in[e]; });
          }
          if (p.dres) put8<R, VEC>(dres_at, it, p.d, g[it]);
        }
        if constexpr (OUTER) {
          Pair c2 = both(0.f);
#pragma unroll
          for (int it = 0; it < I; ++it) {
            v[it] = F::kAhead ? ahead.template get<T>(s, kX, it, p.d) : get8<T, VEC>(xr, it, p.d);
            if constexpr (!F::kKeep) ps[it] = p.outer<T, VEC>(it);
            four([&](int e) {
              v[it][e] = v[it][e] * both(invp);
              acc[it][e] = fma(g[it][e], v[it][e], acc[it][e]);
              g[it][e] = g[it][e] * ps[it][e];
              c2 = fma(g[it][e], v[it][e], c2);
            });
          }
          if (p.post.p) {
            const Pair mean2 = both(-row_sum(c2) * p.inv_d);
#pragma unroll
            for (int it = 0; it < I; ++it) four([&](int e) { g[it][e] = both(invp) * fma(v[it][e], mean2, g[it][e]); });
          }
        }
        T* const dxr = dx.next();
#pragma unroll
        for (int it = 0; it < I; ++it) put8<T, VEC>(dxr, it, p.d, g[it]);
      });
  leave<I, VEC>(p, 0, dw);
  if constexpr (OUTER) leave<I, VEC>(p, 1, acc);
}

__device__ __forceinline__ Pair sigmoid(Pair v) { return each(each(v * both(-kLog2E), exp2_approx) + both(1.f), rcp_approx); }

template <typename T, int I, bool VEC>
struct Gated {
  static constexpr int kPieces = I * (int)sizeof(T), kStages = stages_of(kPieces);
  static constexpr bool kAhead = VEC && kStages > 0;
};
template <typename T, int I, bool VEC>
__global__ void __launch_bounds__(I == 1 ? 128 : 512) gated_rms_norm_kernel(const Norm p) {
  using F = Gated<T, I, VEC>;
  constexpr int kZ = I * (int)sizeof(T) / 2;
  __shared__ __align__(16) float sums[2][16];
  clear(sums);
  RowSum row_sum{sums, 0};
  const Ahead<F::kPieces, F::kStages> ahead;
  const int first = blockIdx.y * p.d;
  auto x = rows_in<T>(p.x, p.xs, first), z = rows_in<T>(p.z, p.zs, first);
  auto y = rows_out<T>(p.y, p.ys, first);
  Eight w[I];
  if constexpr (I <= 2) {
#pragma unroll
    for (int it = 0; it < I; ++it) w[it] = p.w.get<T, VEC>(first, it, p.d);
  }
  for_rows<F::kAhead, F::kStages>(
      p.rows,
      [&](int s) {
        ahead.template send<T, I>(s, 0, x.next(), p.d);
        ahead.template send<T, I>(s, kZ, z.next(), p.d);
      },
      [&](int s, int64_t row) {
        Eight v[I], g[I];
        const T *const xr = F::kAhead ? nullptr : x.next(), *const zr = F::kAhead ? nullptr : z.next();
        Pair ss = both(0.f);
#pragma unroll
        for (int it = 0; it < I; ++it) {
          v[it] = F::kAhead ? ahead.template get<T>(s, 0, it, p.d) : get8<T, VEC>(xr, it, p.d);
          g[it] = F::kAhead ? ahead.template get<T>(s, kZ, it, p.d) : get8<T, VEC>(zr, it, p.d);
          four([&](int e) {
            g[it][e] = g[it][e] * sigmoid(g[it][e]);
            if (!p.norm_first) v[it][e] = v[it][e] * g[it][e];
            ss = fma(v[it][e], v[it][e], ss);
          });
        }
        const float inv = inv_rms(row_sum(ss), p);
        if (p.inv && threadIdx.x == 0) p.inv[row * p.groups + blockIdx.y] = inv;
        T* const yr = y.next();
#pragma unroll
        for (int it = 0; it < I; ++it) {
          if constexpr (I > 2) w[it] = p.w.get<T, VEC>(first, it, p.d);
          four([&](int e) {
            v[it][e] = v[it][e] * both(inv) * w[it][e];
            if (p.norm_first) v[it][e] = v[it][e] * g[it][e];
          });
          put8<T, VEC>(yr, it, p.d, v[it]);
        }
      });
}

template <typename T, int I, bool VEC>
struct GatedBackward {
  static constexpr int kPieces = I * 3 * (int)sizeof(T) / 2, kStages = stages_of(kPieces);
  static constexpr bool kAhead = VEC && kStages > 0;
};
template <typename T, int I, bool VEC>
__global__ void __launch_bounds__(I == 1 ? 128 : 512) gated_rms_norm_grad_kernel(const Norm p) {
  using F = GatedBackward<T, I, VEC>;
  constexpr int kZ = I * (int)sizeof(T) / 2, kG = 2 * kZ;
  __shared__ __align__(16) float sums[2][16];
  clear(sums);
  RowSum row_sum{sums, 0};
  const Ahead<F::kPieces, F::kStages> ahead;
  const int first = blockIdx.y * p.d;
  auto xs = rows_in<T>(p.x, p.xs, first), zs = rows_in<T>(p.z, p.zs, first), gs = rows_in<T>(p.dy, p.dys, first);
  auto dx = rows_out<T>(p.dx, p.dxs, first), dz = rows_out<T>(p.dz, p.dzs, first);
  Eight dw[I], w[I];
#pragma unroll
  for (int it = 0; it < I; ++it) {
    four([&](int e) { dw[it][e] = both(0.f); });
    if constexpr (I <= 2) w[it] = p.w.get<T, VEC>(first, it, p.d);
  }
  const Pair one = both(1.f), minus = both(-1.f);
  float inv_now = 0.f;   // the next row's, asked for a row ahead
  auto rate = [&](int64_t row) {
    if (row < p.rows) inv_now = p.inv[row * p.groups + blockIdx.y];
  };
  rate((int64_t)blockIdx.x * blockDim.y + threadIdx.y);
  for_rows<F::kAhead, F::kStages>(
      p.rows,
      [&](int s) {
        ahead.template send<T, I>(s, 0, xs.next(), p.d);
        ahead.template send<T, I>(s, kZ, zs.next(), p.d);
        ahead.template send<T, I>(s, kG, gs.next(), p.d);
      },
      [&](int s, int64_t row) {
        Eight x[I], z[I], g[I], sg[I];
        const T *const xr = F::kAhead ? nullptr : xs.next(), *const zr = F::kAhead ? nullptr : zs.next(), *const gr = F::kAhead ? nullptr : gs.next();
        const float inv = inv_now;
        rate(row + (int64_t)gridDim.x * blockDim.y);
        Pair c = both(0.f);
#pragma unroll
        for (int it = 0; it < I; ++it) {
          x[it] = F::kAhead ? ahead.template get<T>(s, 0, it, p.d) : get8<T, VEC>(xr, it, p.d);
          z[it] = F::kAhead ? ahead.template get<T>(s, kZ, it, p.d) : get8<T, VEC>(zr, it, p.d);
          g[it] = F::kAhead ? ahead.template get<T>(s, kG, it, p.d) : get8<T, VEC>(gr, it, p.d);
          if constexpr (I > 2) w[it] = p.w.get<T, VEC>(first, it, p.d);
          four([&](int e) {
            sg[it][e] = sigmoid(z[it][e]);
            const Pair gate = z[it][e] * sg[it][e];
            if (p.norm_first) {
              x[it][e] = x[it][e] * both(inv);      // the normalised row
              dw[it][e] = fma(g[it][e] * gate, x[it][e], dw[it][e]);
              g[it][e] = g[it][e] * w[it][e];
              c = fma(g[it][e] * gate, x[it][e], c);
            } else {
              const Pair vh = x[it][e] * gate * both(inv);
              dw[it][e] = fma(g[it][e], vh, dw[it][e]);
              g[it][e] = g[it][e] * w[it][e];
              c = fma(g[it][e], vh, c);
            }
          });
        }
        const Pair mean = both(-row_sum(c) * p.inv_d);
        T *const dxr = dx.next(), *const dzr = dz.next();
#pragma unroll
        for (int it = 0; it < I; ++it) {
          four([&](int e) {
            const Pair sv = sg[it][e], gate = z[it][e] * sv, slope = sv * fma(z[it][e], fma(sv, minus, one), one);
            if (p.norm_first) {
              const Pair vh = x[it][e];
              z[it][e] = g[it][e] * vh * slope;
              x[it][e] = both(inv) * fma(vh, mean, g[it][e] * gate);
            } else {
              const Pair dv = both(inv) * fma(x[it][e] * gate * both(inv), mean, g[it][e]);
              z[it][e] = dv * x[it][e] * slope;
              x[it][e] = dv * gate;
            }
          });
          put8<T, VEC>(dxr, it, p.d, x[it]);
          put8<T, VEC>(dzr, it, p.d, z[it]);
        }
      });
  leave<I, VEC>(p, 0, dw);
}

// Sums over rows to gradients of vectors: column c of the first d is dweight's; one of the next d is that of post_weight * scale.
template <typename T>
struct FinishVectors {
  int d, in_dtype;   // (bits as in SsdNormArgs)
  void *dw, *dpost, *dscale;
  const void *post, *scale;
  __device__ __forceinline__ float get(const void* v, int bit, int c) const {
    return in_dtype & bit ? Cvt<T>::to_f(static_cast<const T*>(v)[c]) : static_cast<const float*>(v)[c];
  }
  __device__ __forceinline__ void put(void* v, int bit, int c, float f) const {
    if (!v) return;
    if (in_dtype & bit) static_cast<T*>(v)[c] = Cvt<T>::from_f(f);
    else static_cast<float*>(v)[c] = f;
  }
  __device__ __forceinline__ void operator()(int c, float v) const {
    if (c < d) {
      put(dw, 1, c, v);
    } else {
      c -= d;
      put(dpost, 2, c, scale ? v * get(scale, 4, c) : v);
      put(dscale, 4, c, post ? v * get(post, 2, c) : v);
    }
  }
};

struct Shape {
  int threads, rows, steps;      // threads of a row, rows of a CTA, eights of a thread
  unsigned most;                 // CTAs a group, of a gradient: each leaves its sums over rows
};
// Eight numbers a thread up to 512 a row, then sixteen, from 4 096 (a gradient: 8 192) on 32.  Rows of a warp go four to a CTA.
Shape shape_of(int64_t rows, int d, int groups, bool grad) {
  Shape s;
  const int eights = (d + 7) / 8;
  s.steps = eights <= 64 ? 1 : eights <= (grad ? 1024 : 512) ? 2 : 4;
  s.threads = ((eights + s.steps - 1) / s.steps + 31) / 32 * 32;
  s.rows = s.threads == 32 ? 4 : 1;
  const int64_t an_sm = std::max(1, 1024 / (s.threads * s.rows));
  s.most = (unsigned)std::min((rows + s.rows - 1) / s.rows, std::max<int64_t>(1, 148 * an_sm / groups));
  return s;
}

int check(const SsdNormArgs* a, bool gated, bool grad) {
  if (!a) return SSD_ERR_NULL_POINTER;
  if (!gated && a->z) return SSD_ERR_UNSUPPORTED;   // (the workspace's size is asked for by it)
  const int groups = gated ? a->groups : 1;
  if (a->rows <= 0 || a->d <= 0 || groups <= 0 || a->d % groups != 0 || !(a->eps >= 0.f && a->eps < INFINITY)) return SSD_ERR_BAD_SHAPE;
  if (a->d / groups > 16384 || groups > 65535) return SSD_ERR_TOO_LARGE;
  if (!a->x || !a->weight) return SSD_ERR_NULL_POINTER;
  if (gated && !a->z) return SSD_ERR_NULL_POINTER;
  if (!gated && !a->residual && (a->post_weight || a->scale) && !grad) return SSD_ERR_UNSUPPORTED;
  if (grad) {
    if (!a->dy || !a->dx || !a->inv_rms || (gated && !a->dz)) return SSD_ERR_NULL_POINTER;
    if (!gated && (a->post_weight || a->scale) && !a->residual_out) return SSD_ERR_UNSUPPORTED;
    if (!gated && a->post_weight && !a->inv_rms_post) return SSD_ERR_NULL_POINTER;
    if (!gated && !a->residual_out && (a->dresidual || a->dresidual_out)) return SSD_ERR_UNSUPPORTED;
    if (!a->workspace || a->workspace_bytes < ssd_b200_norm_workspace_bytes(a) || reinterpret_cast<uintptr_t>(a->workspace) % 16)
      return SSD_ERR_WORKSPACE;
  } else if (!a->y || (!gated && a->residual && !a->residual_out)) {
    return SSD_ERR_NULL_POINTER;
  }
  return SSD_OK;
}

// How many CTAs of a kernel an SM holds: asked for once a thread, kernel, device and size (as long as no other one takes its place).
struct Resident {
  const void* kernel;
  int device, threads, smem, an_sm;
  bool is(const Resident& o) const { return kernel == o.kernel && device == o.device && threads == o.threads && smem == o.smem; }
};
Resident& resident(const Resident& r) {
  static thread_local Resident known[128] = {};
  return known[(reinterpret_cast<uintptr_t>(r.kernel) / 16 * 31 + (unsigned)r.device * 7 + (unsigned)r.threads + (unsigned)r.smem / 512) % 128];
}

template <typename T>
struct Launch {
  Norm p = {};
  Shape s;
  bool vec = true;
  unsigned grid = 0;
  cudaStream_t stream;
  Launch(const SsdNormArgs& a, bool gated, bool grad, cudaStream_t st) : stream(st) {
    p.rows = a.rows; p.groups = gated ? a.groups : 1; p.d = a.d / p.groups; p.eps = a.eps; p.inv_d = 1.f / (float)p.d; p.norm_first = a.norm_first;
    p.x = a.x; p.z = a.z; p.res = a.residual; p.y = a.y; p.res_out = a.residual_out; p.inv = a.inv_rms; p.inv_post = a.inv_rms_post;
    p.xs = a.x_stride; p.zs = a.z_stride; p.rs = a.residual_stride; p.ys = a.y_stride; p.ros = a.residual_out_stride;
    p.w = {a.weight, a.vectors_in_dtype & 1};
    if (!gated) {
      p.post = {a.post_weight, a.vectors_in_dtype & 2};
      p.scale = {a.scale, a.vectors_in_dtype & 4};
    }
    s = shape_of(a.rows, p.d, p.groups, grad);
    const int R = a.residual_dtype == SSD_DTYPE_F32 ? 4 : 2;
    vec = p.d % 8 == 0;
    rows_of(a.x, a.x_stride, sizeof(T));
    vector_of(p.w);
    vector_of(p.post);
    vector_of(p.scale);
    if (gated) rows_of(a.z, a.z_stride, sizeof(T));
    else rows_of(a.residual_out, a.residual_out_stride, R);
    if (grad) {
      p.dy = a.dy; p.dres_out = a.dresidual_out; p.dx = a.dx; p.dz = a.dz; p.dres = a.dresidual;
      p.dys = a.dy_stride; p.dros = a.dresidual_out_stride; p.dxs = a.dx_stride; p.dzs = a.dz_stride; p.drs = a.dresidual_stride;
      p.part = static_cast<float*>(a.workspace);
      p.vectors = !gated && (a.post_weight || a.scale) ? 2 : 1;
      rows_of(a.dy, a.dy_stride, sizeof(T));
      rows_of(a.dx, a.dx_stride, sizeof(T));
      if (gated) rows_of(a.dz, a.dz_stride, sizeof(T));
      else rows_of(a.dresidual, a.dresidual_stride, R), rows_of(a.dresidual_out, a.dresidual_out_stride, R);
    } else {
      rows_of(a.y, a.y_stride, sizeof(T));
      if (!gated) rows_of(a.residual, a.residual_stride, R);
    }
  }
  // (sixteen bytes at once)
  void rows_of(const void* at, int64_t stride, int bytes) {
    if (at) vec = vec && reinterpret_cast<uintptr_t>(at) % 16 == 0 && stride * bytes % 16 == 0;
  }
  void vector_of(const Vector& v) { vec = vec && reinterpret_cast<uintptr_t>(v.p) % 16 == 0; }

  // As many CTAs as the chip holds at once, where there are rows for them (a gradient: and sums).
  template <typename K>
  int go(K kernel, int pieces, int stages) {
    const size_t smem = vec ? (size_t)pieces * stages * s.threads * s.rows * 16 : 0;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return SSD_ERR_CUDA;
    const Resident want = {reinterpret_cast<const void*>(kernel), device, s.threads * s.rows, (int)smem, 0};
    Resident& known = resident(want);
    if (!known.is(want)) {
      int an_sm = 0;
      // (the most there is, so that no later call's size takes it back)
      if ((smem && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 << 10) != cudaSuccess) ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&an_sm, kernel, want.threads, smem) != cudaSuccess || an_sm < 1)
        return SSD_ERR_CUDA;
      known = want;
      known.an_sm = an_sm;
    }
    const int64_t all = (p.rows + s.rows - 1) / s.rows, fit = std::max(1, 148 * known.an_sm / p.groups);
    grid = (unsigned)std::min<int64_t>(std::min(all, fit), p.part ? s.most : fit);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, (unsigned)p.groups);
    cfg.blockDim = dim3((unsigned)s.threads, (unsigned)s.rows);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? SSD_OK : SSD_ERR_CUDA;
  }
  template <typename F>
  int by_steps(F f) {
    if (s.steps == 1) return f(std::integral_constant<int, 1>());
    if (s.steps == 2) return f(std::integral_constant<int, 2>());
    return f(std::integral_constant<int, 4>());
  }
  template <typename R, bool OUTER>
  int forward() {
    return by_steps([&](auto i) {
      constexpr int I = decltype(i)::value;
      using F = Forward<T, R, I, true, OUTER>;
      return go(vec ? rms_norm_kernel<T, R, I, true, OUTER> : rms_norm_kernel<T, R, I, false, OUTER>, F::kPieces, F::kStages);
    });
  }
  template <typename R, bool OUTER>
  int backward() {
    return by_steps([&](auto i) {
      constexpr int I = decltype(i)::value;
      using F = Backward<T, R, I, true, OUTER>;
      return go(vec ? rms_norm_grad_kernel<T, R, I, true, OUTER> : rms_norm_grad_kernel<T, R, I, false, OUTER>, F::kPieces, F::kStages);
    });
  }
  int gated() {
    return by_steps([&](auto i) {
      constexpr int I = decltype(i)::value;
      using F = Gated<T, I, true>;
      return go(vec ? gated_rms_norm_kernel<T, I, true> : gated_rms_norm_kernel<T, I, false>, F::kPieces, F::kStages);
    });
  }
  int gated_backward() {
    return by_steps([&](auto i) {
      constexpr int I = decltype(i)::value;
      using F = GatedBackward<T, I, true>;
      return go(vec ? gated_rms_norm_grad_kernel<T, I, true> : gated_rms_norm_grad_kernel<T, I, false>, F::kPieces, F::kStages);
    });
  }
  int vectors(const SsdNormArgs& a) const {
    if (!a.dweight && !a.dpost_weight && !a.dscale) return SSD_OK;
    const int all = a.d * p.vectors;
    return launch_column_sum(p.part, (int64_t)grid * s.rows, all, all,
                             FinishVectors<T>{a.d, a.vectors_in_dtype, a.dweight, a.dpost_weight, a.dscale, a.post_weight, a.scale}, stream);
  }
};

}  // namespace
}  // namespace ssd

extern "C" size_t ssd_b200_norm_workspace_bytes(const SsdNormArgs* a) {
  if (!a || a->rows <= 0 || a->d <= 0) return 0;
  const int groups = a->z ? a->groups : 1;
  if (groups <= 0 || a->d % groups != 0 || a->d / groups > 16384) return 0;
  const ssd::Shape s = ssd::shape_of(a->rows, a->d / groups, groups, true);
  return (size_t)s.most * s.rows * a->d * (!a->z && (a->post_weight || a->scale) ? 2 : 1) * sizeof(float);
}

extern "C" int ssd_b200_rms_norm(const SsdNormArgs* args, void* stream) {
  if (const int rc = ssd::check(args, false, false)) return rc;
  const SsdNormArgs& a = *args;
  return ssd::by_type(a.dtype, [&](auto t) -> int {
    using T = decltype(t);
    ssd::Launch<T> l(a, false, false, static_cast<cudaStream_t>(stream));
    const bool outer = a.post_weight || a.scale;
    if (!a.residual || a.residual_dtype == a.dtype) return outer ? l.template forward<T, true>() : l.template forward<T, false>();
    if (a.residual_dtype != SSD_DTYPE_F32) return (int)SSD_ERR_UNSUPPORTED;
    return outer ? l.template forward<float, true>() : l.template forward<float, false>();
  });
}

extern "C" int ssd_b200_rms_norm_backward(const SsdNormArgs* args, void* stream) {
  if (const int rc = ssd::check(args, false, true)) return rc;
  const SsdNormArgs& a = *args;
  return ssd::by_type(a.dtype, [&](auto t) -> int {
    using T = decltype(t);
    ssd::Launch<T> l(a, false, true, static_cast<cudaStream_t>(stream));
    const bool outer = a.post_weight || a.scale;
    int rc = SSD_ERR_UNSUPPORTED;
    if (!a.residual_out || a.residual_dtype == a.dtype) rc = outer ? l.template backward<T, true>() : l.template backward<T, false>();
    else if (a.residual_dtype == SSD_DTYPE_F32) rc = outer ? l.template backward<float, true>() : l.template backward<float, false>();
    return rc ? rc : l.vectors(a);
  });
}

extern "C" int ssd_b200_gated_rms_norm(const SsdNormArgs* args, void* stream) {
  if (const int rc = ssd::check(args, true, false)) return rc;
  return ssd::by_type(args->dtype, [&](auto t) { return ssd::Launch<decltype(t)>(*args, true, false, static_cast<cudaStream_t>(stream)).gated(); });
}

extern "C" int ssd_b200_gated_rms_norm_backward(const SsdNormArgs* args, void* stream) {
  if (const int rc = ssd::check(args, true, true)) return rc;
  return ssd::by_type(args->dtype, [&](auto t) -> int {
    ssd::Launch<decltype(t)> l(*args, true, true, static_cast<cudaStream_t>(stream));
    const int rc = l.gated_backward();
    return rc ? rc : l.vectors(*args);
  });
}
