// Gradient of the causal depthwise conv1d + SiLU (ssd_conv1d.cu):
//   pre[t] = bias + sum_k w[k] x[t-(K-1)+k],   dpre[t] = dy[t] s(pre) (1 + pre (1 - s(pre))),  s the sigmoid
//   dx[t] = sum_k w[k] dpre[t+(K-1)-k],   dw[k] = sum_t dpre[t] x[t-(K-1)+k],   dbias = sum_t dpre[t]
// A warp walks a run of tokens of 64 channels, two a lane: x and dpre of the last K tokens in a ring of registers (no row is ever moved),
// dx[t-(K-1)] written once dpre[t] is known, so x and dy are read once but for K-1 tokens on either side of a run.  Blocks of eight tokens
// are on their way (TMA, a ring of its own for each warp) while one is worked on: registers do not hold enough of them to cover the memory's latency
// (4 x 8 192 x 5 120 bf16: a block ahead in registers 239 us).  A CTA's runs follow one another; it leaves
// its sums for dw and dbias to column_sum_kernel, in a fixed order.
// 4 x 8 192 x 5 120 bf16: 197 us (5.1 TB/s, 79 % of the copy bandwidth).  Bound: latency with sixteen warps an SM and 25 instructions an element.
// Sixteen warps are four CTAs of four: a CTA's last warp holds up fewer of them (two of eight 216 us; eight of two 199, but 8 x 2 048 x 2 048 53 for 50).
#include <algorithm>
#include <type_traits>

#include "tc_common.cuh"
#include "tc_ptx.cuh"
#include "vec_io.cuh"

namespace ssd {
namespace {

constexpr int kWarps = 4, kAhead = 8, kCtas = 4;
constexpr int stages_of(int bytes) { return bytes == 2 ? 4 : 3; }   // blocks of a warp's ring

struct ConvGrad {
  const void *x, *w, *bias, *dy;
  void* dx;
  float* part;   // [batch][CTAs of a sequence][K + 1][channels]
  int32_t* status;
  int seqlen, channels, run, ctas;
  int64_t xs[2], dys[2], dxs[2];
};

struct ConvMaps {
  CUtensorMap x, dy;
};

// TMA: rows of x and dy start on 16 bytes.
template <typename T, int K, bool TMA>
__global__ void __launch_bounds__(32 * kWarps, kCtas) conv1d_silu_grad_kernel(const __grid_constant__ ConvGrad p, const __grid_constant__ ConvMaps maps) {
  using Raw = typename Two<T>::Raw;
  constexpr int kStages = stages_of(sizeof(T)), kBlock = kAhead * 64;   // numbers of a block of one tensor
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t full[kWarps][kStages];
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
    auto block = [&](int t0, auto xv, auto g) {   // xv(n), g(n): x and dy of token t0 + n
      T* to = dx + (int64_t)(t0 - (K - 1)) * p.dxs[1];
      if (t0 > t_begin && t0 + kAhead <= t_end) {
#pragma unroll
        for (int n = 0; n < kAhead; ++n, to += p.dxs[1]) token(std::true_type(), n, t0 + n, xv(n), g(n), to);
      } else {
#pragma unroll
        for (int n = 0; n < kAhead; ++n, to += p.dxs[1])
          if (t0 + n < t_last) token(std::false_type(), n, t0 + n, xv(n), g(n), to);
      }
    };
    if constexpr (TMA) {
      T* const ring = reinterpret_cast<T*>(smem) + w * kStages * 2 * kBlock;
      auto send = [&](int stage, int t0) {   // (one lane; what lies behind the sequence or the last channel reads as zero)
        ptx::mbar_expect_tx(&full[w][stage], 2 * kBlock * sizeof(T));
#pragma unroll
        for (int n = 0; n < 2; ++n)
          asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                           ptx::smem_u32(ring + (2 * stage + n) * kBlock)),
                       "l"(n ? &maps.dy : &maps.x), "r"(ptx::smem_u32(&full[w][stage])), "r"(blockIdx.y * 64), "r"(t0), "r"(b)
                       : "memory");
      };
      if (lane == 0) {
#pragma unroll
        for (int n = 0; n < kStages; ++n) ptx::mbar_init(&full[w][n], 1);
        ptx::fence_mbar_init();
#pragma unroll
        for (int n = 0; n < kStages; ++n)
          if (t_begin + n * kAhead < t_last) send(n, t_begin + n * kAhead);
      }
      __syncwarp();
      int stage = 0;
      unsigned parity = 0;
      auto wait = [&](int s, unsigned par) {   // for about a second
        if (ptx::mbar_try_wait(&full[w][s], par)) return true;
        const long long since = clock64();
        while (!ptx::mbar_try_wait(&full[w][s], par))
          if (clock64() - since > 2000000000LL) return false;
        return true;
      };
      for (int t0 = t_begin; t0 < t_last; t0 += kAhead) {
        if (!__all_sync(~0u, wait(stage, parity))) {
          if (lane == 0) {   // it gives up, once the blocks it has sent for are there or do not come either
            if (p.status) *p.status = STATUS_WAIT_TIMEOUT_TMA;
            for (int n = 0, t = t0; n < kStages && t < t_last; ++n, t += kAhead) wait((stage + n) % kStages, parity ^ (stage + n >= kStages));
          }
          __syncwarp();
          break;
        }
        const Raw* const at = reinterpret_cast<const Raw*>(ring + 2 * stage * kBlock) + lane;
        block(t0, [&](int n) { return pair_of<T>(at[n * 32]); }, [&](int n) { return pair_of<T>(at[n * 32 + kBlock / 2]); });
        __syncwarp();
        if (lane == 0 && t0 + kStages * kAhead < t_last) send(stage, t0 + kStages * kAhead);
        if (++stage == kStages) stage = 0, parity ^= 1;
      }
    } else {
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
      ask(t_begin);
      for (int t0 = t_begin; t0 < t_last; t0 += kAhead) {
        Raw cx[kAhead], cd[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) cx[n] = rx[n], cd[n] = rd[n];
        if (t0 + kAhead < t_last) ask(t0 + kAhead);
        block(t0, [&](int n) { return pair_of<T>(cx[n]); }, [&](int n) { return pair_of<T>(cd[n]); });
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

// Strips of channels are a grid's second axis, and a run goes a few tokens past its end.
bool covered(int seqlen, int channels) { return channels <= 64 * 65535 && seqlen <= 0x7fffff00; }

struct Cut {
  int run, ctas;   // tokens of a warp, CTAs of a sequence
};
// Long runs read fewer tokens twice (K - 1 on either side); shorter ones where there are few CTAs.
Cut cut_of(int batch, int seqlen, int channels) {
  Cut c;
  const int64_t strips = (int64_t)batch * ((channels + 63) / 64);
  for (c.run = 256; c.run > 8; c.run /= 2) {
    if (strips * ((seqlen + (int64_t)kWarps * c.run - 1) / (kWarps * c.run)) >= 148 * 4) break;
  }
  c.ctas = (int)(((int64_t)seqlen + kWarps * c.run - 1) / (kWarps * c.run));
  return c;
}

template <typename T>
bool operand_map(CUtensorMap* map, const void* base, int batch, int seqlen, int channels, const int64_t* st, int dtype) {
  const tc::EncodeFn encode = tc::encode_fn();
  const int64_t sl = seqlen == 1 ? 16 : st[1], sb = batch == 1 ? 16 : st[0];   // (the stride of a single one may be anything)
  constexpr int64_t e = sizeof(T), most = (int64_t)1 << 40;
  if (!encode || reinterpret_cast<uintptr_t>(base) % 16 || sl * e % 16 || sb * e % 16 || sl <= 0 || sb <= 0 || sl * e >= most || sb * e >= most) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)channels, (cuuint64_t)seqlen, (cuuint64_t)batch}, strides[2] = {(cuuint64_t)(sl * e), (cuuint64_t)(sb * e)};
  const cuuint32_t box[3] = {64, kAhead, 1}, each[3] = {1, 1, 1};
  const CUtensorMapDataType type = dtype == SSD_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == SSD_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(map, type, 3, const_cast<void*>(base), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
int run_grad(ConvGrad p, void* dw, void* db, int batch, int taps, int dtype, cudaStream_t stream) {
  const dim3 grid((unsigned)(batch * p.ctas), (unsigned)((p.channels + 63) / 64));
  ConvMaps maps = {};
  const bool tma = operand_map<T>(&maps.x, p.x, batch, p.seqlen, p.channels, p.xs, dtype) &&
                   operand_map<T>(&maps.dy, p.dy, batch, p.seqlen, p.channels, p.dys, dtype);
  constexpr int smem = kWarps * stages_of(sizeof(T)) * 2 * kAhead * 64 * (int)sizeof(T);
  auto go = [&](auto k) {
    constexpr int K = decltype(k)::value;
    if (!tma) return launch(conv1d_silu_grad_kernel<T, K, false>, grid, 32 * kWarps, 0, stream, p, maps);
    if (cudaFuncSetAttribute(conv1d_silu_grad_kernel<T, K, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return (int)SSD_ERR_CUDA;
    return launch(conv1d_silu_grad_kernel<T, K, true>, grid, 32 * kWarps, smem, stream, p, maps);
  };
  int rc = SSD_ERR_UNSUPPORTED;
  switch (taps) {
    case 2: rc = go(std::integral_constant<int, 2>()); break;
    case 3: rc = go(std::integral_constant<int, 3>()); break;
    case 4: rc = go(std::integral_constant<int, 4>()); break;
  }
  if (rc) return rc;
  const int all = (taps + 1) * p.channels;
  return launch_column_sum(p.part, (int64_t)batch * p.ctas, all, all, FinishConv<T>{static_cast<T*>(dw), static_cast<T*>(db), p.channels, taps}, stream);
}

}  // namespace
}  // namespace ssd

extern "C" size_t ssd_b200_conv1d_silu_workspace_bytes(int32_t batch, int32_t seqlen, int32_t channels, int32_t taps) {
  if (batch <= 0 || seqlen <= 0 || channels <= 0 || taps < 2 || taps > 4 || !ssd::covered(seqlen, channels)) return 0;
  return (size_t)batch * ssd::cut_of(batch, seqlen, channels).ctas * (taps + 1) * channels * sizeof(float);
}

extern "C" int ssd_b200_conv1d_silu_backward(const void* x, const void* weight, const void* bias, const void* dy, void* dx, void* dweight,
                                             void* dbias, void* workspace, size_t workspace_bytes, int32_t batch, int32_t seqlen,
                                             int32_t channels, int32_t taps, int32_t dtype, int64_t x_stride_b, int64_t x_stride_l,
                                             int64_t dy_stride_b, int64_t dy_stride_l, int64_t dx_stride_b, int64_t dx_stride_l,
                                             int32_t* status, void* stream) {
  if (!x || !weight || !dy || !dx || !dweight || (bias && !dbias)) return SSD_ERR_NULL_POINTER;
  if (batch <= 0 || seqlen <= 0 || channels <= 0 || taps <= 0) return SSD_ERR_BAD_SHAPE;
  if (channels % 8 != 0 || taps < 2 || taps > 4) return SSD_ERR_UNSUPPORTED;
  if (!ssd::covered(seqlen, channels)) return SSD_ERR_TOO_LARGE;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      workspace_bytes < ssd_b200_conv1d_silu_workspace_bytes(batch, seqlen, channels, taps))
    return SSD_ERR_WORKSPACE;
  const ssd::Cut cut = ssd::cut_of(batch, seqlen, channels);
  if ((int64_t)batch * cut.ctas > 0x7fffffff) return SSD_ERR_TOO_LARGE;
  // two channels at once: rows start on their boundary
  for (int64_t stride : {x_stride_b, x_stride_l, dy_stride_b, dy_stride_l, dx_stride_b, dx_stride_l})
    if (stride % 2) return SSD_ERR_MISALIGNED;
  const uintptr_t two = dtype == SSD_DTYPE_F32 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(x) % two || reinterpret_cast<uintptr_t>(dy) % two || reinterpret_cast<uintptr_t>(dx) % two)
    return SSD_ERR_MISALIGNED;
  ssd::ConvGrad p = {x, weight, bias, dy, dx, static_cast<float*>(workspace), status, seqlen, channels, cut.run, cut.ctas,
                     {x_stride_b, x_stride_l}, {dy_stride_b, dy_stride_l}, {dx_stride_b, dx_stride_l}};
  return ssd::by_type(dtype, [&](auto t) {
    return ssd::run_grad<decltype(t)>(p, dweight, bias ? dbias : nullptr, batch, taps, dtype, static_cast<cudaStream_t>(stream));
  });
}
