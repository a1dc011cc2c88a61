// Gradient of the causal depthwise conv1d + SiLU (ssd_conv1d.cu):
//   pre[t] = bias + sum_k w[k] x[t-(K-1)+k],   dpre[t] = dy[t] s(pre) (1 + pre (1 - s(pre))),  s the sigmoid
//   dx[t] = sum_k w[k] dpre[t+(K-1)-k],   dw[k] = sum_t dpre[t] x[t-(K-1)+k],   dbias = sum_t dpre[t]
// A warp walks a run of tokens of 64 channels, two a lane: x and dpre of the last K tokens in registers, dx[t-(K-1)] written once
// dpre[t] is known, so x and dy are read once but for K-1 tokens on either side of a run.  A CTA's runs follow one another; it leaves
// its sums for dw and dbias to column_sum_kernel, in a fixed order.
#include <algorithm>
#include <type_traits>

#include "vec_io.cuh"

namespace ssd {
namespace {

constexpr int kWarps = 8, kAhead = 8, kCtas = 2;

struct ConvGrad {
  const void *x, *w, *bias, *dy;
  void* dx;
  float* part;   // [batch][CTAs of a sequence][K + 1][channels]
  int seqlen, channels, run, ctas;
  int64_t xs[2], dys[2], dxs[2];
};

template <typename T, int K>
__global__ void __launch_bounds__(32 * kWarps, kCtas) conv1d_silu_grad_kernel(const ConvGrad p) {
  using Raw = typename Two<T>::Raw;
  __shared__ Pair sums[kWarps][K + 1][32];
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const int c = blockIdx.y * 64 + 2 * lane;
  const int cta = blockIdx.x % p.ctas, b = blockIdx.x / p.ctas;
  const bool ok = c < p.channels;
  const int64_t begin = ((int64_t)cta * kWarps + w) * p.run;
  const int t_begin = (int)min((int64_t)p.seqlen, begin), t_end = (int)min((int64_t)p.seqlen, begin + p.run);
  const Pair zero = both(0.f), one = both(1.f), minus = both(-1.f);

  Pair wk[K], bs = zero, dw[K], db = zero;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const T* at = static_cast<const T*>(p.w) + (int64_t)c * K + k;
    wk[k] = ok ? pair(Cvt<T>::to_f(at[0]), Cvt<T>::to_f(at[K])) : zero;
    dw[k] = zero;
  }
  if (ok && p.bias) bs = pair(Cvt<T>::to_f(static_cast<const T*>(p.bias)[c]), Cvt<T>::to_f(static_cast<const T*>(p.bias)[c + 1]));
  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + c;
  const T* dy = static_cast<const T*>(p.dy) + b * p.dys[0] + c;
  T* dx = static_cast<T*>(p.dx) + b * p.dxs[0] + c;
  auto row = [&](const T* at, int64_t stride, int t) {
    return ok && t >= 0 && t < p.seqlen ? *reinterpret_cast<const Raw*>(at + (int64_t)t * stride) : Two<T>::zero();
  };

  if (t_begin < t_end) {
    // x and dpre of token t_begin + n in places n & 7: no row is ever moved
    Pair xw[kAhead], dp[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) dp[n] = zero, xw[n] = n > kAhead - K ? pair_of<T>(row(x, p.xs[1], t_begin - kAhead + n)) : zero;
    const int t_last = min(t_end + K - 1, p.seqlen + K - 1);   // dpre of the K - 1 tokens behind the run, zero behind the sequence
    Raw rx[kAhead], rd[kAhead];
    auto ask = [&](int t0) {
      if (ok && t0 + kAhead <= p.seqlen) {
        const T *xa = x + (int64_t)t0 * p.xs[1], *da = dy + (int64_t)t0 * p.dys[1];
#pragma unroll
        for (int n = 0; n < kAhead; ++n, xa += p.xs[1], da += p.dys[1]) {
          rx[n] = *reinterpret_cast<const Raw*>(xa);
          rd[n] = *reinterpret_cast<const Raw*>(da);
        }
      } else {
#pragma unroll
        for (int n = 0; n < kAhead; ++n) rx[n] = row(x, p.xs[1], t0 + n), rd[n] = row(dy, p.dys[1], t0 + n);
      }
    };
    // one token; ALL: it is the run's, and so are those that its dx is of
    auto token = [&](auto all, int n, int t, Pair xv, Pair g, T* to) {
      constexpr bool ALL = decltype(all)::value;
      auto at = [&](int back) { return (n + kAhead - back) % kAhead; };
      xw[n] = xv;
      Pair pre = bs;
#pragma unroll
      for (int k = 0; k < K; ++k) pre = fma(wk[k], xw[at(K - 1 - k)], pre);
      const Pair s = each(each(pre * both(-kLog2E), exp2_approx) + one, rcp_approx);
      Pair d = (g * s) * fma(pre, fma(s, minus, one), one);
      if (!ALL && t >= p.seqlen) d = zero;
      dp[n] = d;
      if (ALL || t < t_end) {
        db = db + d;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k] = fma(d, xw[at(K - 1 - k)], dw[k]);
      }
      Pair o = wk[0] * d;
#pragma unroll
      for (int k = 1; k < K; ++k) o = fma(wk[k], dp[at(k)], o);
      const int u = t - (K - 1);
      if (ok && (ALL || (u >= t_begin && u < t_end))) {
        const float2 h = halves(o);
        *reinterpret_cast<Raw*>(to) = Two<T>::down(h.x, h.y);
      }
    };
    ask(t_begin);
    for (int t0 = t_begin; t0 < t_last; t0 += kAhead) {
      Raw cx[kAhead], cd[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) cx[n] = rx[n], cd[n] = rd[n];
      if (t0 + kAhead < t_last) ask(t0 + kAhead);
      T* to = dx + (int64_t)(t0 - (K - 1)) * p.dxs[1];
      if (t0 > t_begin && t0 + kAhead <= t_end) {
#pragma unroll
        for (int n = 0; n < kAhead; ++n, to += p.dxs[1]) token(std::true_type(), n, t0 + n, pair_of<T>(cx[n]), pair_of<T>(cd[n]), to);
      } else {
#pragma unroll
        for (int n = 0; n < kAhead; ++n, to += p.dxs[1])
          if (t0 + n < t_last) token(std::false_type(), n, t0 + n, pair_of<T>(cx[n]), pair_of<T>(cd[n]), to);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) sums[w][k][lane] = dw[k];
  sums[w][K][lane] = db;
  __syncthreads();
  for (int i = threadIdx.x; i < (K + 1) * 32; i += 32 * kWarps) {
    const int k = i / 32, l = i % 32, cc = blockIdx.y * 64 + 2 * l;
    if (cc >= p.channels) continue;
    Pair v = sums[0][k][l];
#pragma unroll
    for (int u = 1; u < kWarps; ++u) v = v + sums[u][k][l];
    *reinterpret_cast<float2*>(p.part + ((int64_t)blockIdx.x * (K + 1) + k) * p.channels + cc) = halves(v);
  }
}

template <typename T>
struct FinishConv {
  T *dw, *db;
  int channels, taps;
  __device__ __forceinline__ void operator()(int i, float v) const {
    const int k = i / channels, c = i % channels;
    if (k < taps) dw[(int64_t)c * taps + k] = Cvt<T>::from_f(v);
    else if (db) db[c] = Cvt<T>::from_f(v);
  }
};

struct Cut {
  int run, ctas;   // tokens of a warp, CTAs of a sequence
};
// Long runs read fewer tokens twice (K - 1 on either side); shorter ones where there are few CTAs.
Cut cut_of(int batch, int seqlen, int channels) {
  Cut c;
  const int64_t strips = (int64_t)batch * ((channels + 63) / 64);
  for (c.run = 128; c.run > 8; c.run /= 2) {
    if (strips * ((seqlen + (int64_t)kWarps * c.run - 1) / (kWarps * c.run)) >= 148 * 4) break;
  }
  c.ctas = (int)(((int64_t)seqlen + kWarps * c.run - 1) / (kWarps * c.run));
  return c;
}

template <typename T>
int run_grad(ConvGrad p, void* dw, void* db, int batch, int taps, cudaStream_t stream) {
  const dim3 grid((unsigned)(batch * p.ctas), (unsigned)((p.channels + 63) / 64));
  int rc = SSD_ERR_UNSUPPORTED;
  switch (taps) {
    case 2: rc = launch(conv1d_silu_grad_kernel<T, 2>, grid, 32 * kWarps, 0, stream, p); break;
    case 3: rc = launch(conv1d_silu_grad_kernel<T, 3>, grid, 32 * kWarps, 0, stream, p); break;
    case 4: rc = launch(conv1d_silu_grad_kernel<T, 4>, grid, 32 * kWarps, 0, stream, p); break;
  }
  if (rc) return rc;
  const int all = (taps + 1) * p.channels;
  return launch_column_sum(p.part, (int64_t)batch * p.ctas, all, all, FinishConv<T>{static_cast<T*>(dw), static_cast<T*>(db), p.channels, taps}, stream);
}

}  // namespace
}  // namespace ssd

extern "C" size_t ssd_b200_conv1d_silu_workspace_bytes(int32_t batch, int32_t seqlen, int32_t channels, int32_t taps) {
  if (batch <= 0 || seqlen <= 0 || channels <= 0 || taps < 2 || taps > 4) return 0;
  return (size_t)batch * ssd::cut_of(batch, seqlen, channels).ctas * (taps + 1) * channels * sizeof(float);
}

extern "C" int ssd_b200_conv1d_silu_backward(const void* x, const void* weight, const void* bias, const void* dy, void* dx, void* dweight,
                                             void* dbias, void* workspace, size_t workspace_bytes, int32_t batch, int32_t seqlen,
                                             int32_t channels, int32_t taps, int32_t dtype, int64_t x_stride_b, int64_t x_stride_l,
                                             int64_t dy_stride_b, int64_t dy_stride_l, int64_t dx_stride_b, int64_t dx_stride_l,
                                             void* stream) {
  if (!x || !weight || !dy || !dx || !dweight || (bias && !dbias)) return SSD_ERR_NULL_POINTER;
  if (batch <= 0 || seqlen <= 0 || channels <= 0 || taps <= 0) return SSD_ERR_BAD_SHAPE;
  if (channels % 8 != 0 || taps < 2 || taps > 4) return SSD_ERR_UNSUPPORTED;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      workspace_bytes < ssd_b200_conv1d_silu_workspace_bytes(batch, seqlen, channels, taps))
    return SSD_ERR_WORKSPACE;
  const ssd::Cut cut = ssd::cut_of(batch, seqlen, channels);
  if ((int64_t)batch * cut.ctas > 0x7fffffff || (channels + 63) / 64 > 65535) return SSD_ERR_TOO_LARGE;
  // two channels at once: rows start on their boundary
  for (int64_t stride : {x_stride_b, x_stride_l, dy_stride_b, dy_stride_l, dx_stride_b, dx_stride_l})
    if (stride % 2) return SSD_ERR_MISALIGNED;
  const uintptr_t two = dtype == SSD_DTYPE_F32 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(x) % two || reinterpret_cast<uintptr_t>(dy) % two || reinterpret_cast<uintptr_t>(dx) % two)
    return SSD_ERR_MISALIGNED;
  ssd::ConvGrad p = {x, weight, bias, dy, dx, static_cast<float*>(workspace), seqlen, channels, cut.run, cut.ctas,
                     {x_stride_b, x_stride_l}, {dy_stride_b, dy_stride_l}, {dx_stride_b, dx_stride_l}};
  return ssd::by_type(dtype, [&](auto t) {
    return ssd::run_grad<decltype(t)>(p, dweight, bias ? dbias : nullptr, batch, taps, static_cast<cudaStream_t>(stream));
  });
}
