// RMS norms between blocks and their gradients (formulas: ssd_b200.h).
// A row (of a group) is one warp's or one CTA's, eight numbers a thread and step, kept in registers: every input is read once, every
// output written once.  The gradients against vectors are sums over rows: a CTA adds those of its rows up in registers and leaves
// them to column_sum_kernel, so that their order is fixed.
#include <algorithm>
#include <cmath>

#include "vec_io.cuh"

namespace ssd {
namespace {

// Eight numbers of a row: neighbours (VEC: 16-byte pieces), or blockDim.x apart where rows do not start on such a boundary.
// Those behind the row's end read as zero.
template <bool VEC>
__device__ __forceinline__ int place(int it, int e) {
  return VEC ? (it * (int)blockDim.x + (int)threadIdx.x) * 8 + e : (it * 8 + e) * (int)blockDim.x + (int)threadIdx.x;
}
template <typename T, bool VEC>
__device__ __forceinline__ void get8(const T* __restrict__ row, int it, int d, float (&v)[8]) {
  if constexpr (VEC) {
    const int at = place<true>(it, 0);
    if (at < d) {
      if constexpr (sizeof(T) == 2) {
        const uint4 q = *reinterpret_cast<const uint4*>(row + at);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Two<T>::up(w[e]);
          v[2 * e] = f.x;
          v[2 * e + 1] = f.y;
        }
      } else {
        const float4 a = *reinterpret_cast<const float4*>(row + at), b = *reinterpret_cast<const float4*>(row + at + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = place<false>(it, e) < d ? Cvt<T>::to_f(row[place<false>(it, e)]) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void put8(T* row, int it, int d, const float (&v)[8]) {
  if constexpr (VEC) {
    const int at = place<true>(it, 0);
    if (at < d) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(row + at) = make_uint4(Two<T>::down(v[0], v[1]), Two<T>::down(v[2], v[3]), Two<T>::down(v[4], v[5]), Two<T>::down(v[6], v[7]));
      } else {
        *reinterpret_cast<float4*>(row + at) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (place<false>(it, e) < d) row[place<false>(it, e)] = Cvt<T>::from_f(v[e]);
  }
}

// A vector of d numbers, fp32 or T.
struct Vector {
  const void* p;
  int in_dtype;
  template <typename T, bool VEC>
  __device__ __forceinline__ void get(int first, int it, int d, float (&v)[8]) const {
    if (in_dtype) get8<T, VEC>(static_cast<const T*>(p) + first, it, d, v);
    else get8<float, VEC>(static_cast<const float*>(p) + first, it, d, v);
  }
};

// Sum over the threads of a row, in all of them.  `turn` alternates between two places, so that one barrier a sum is enough.
struct RowSum {
  float* place;   // [2][32]
  int turn;
  __device__ __forceinline__ float operator()(float v) {
#pragma unroll
    for (int k = 16; k > 0; k /= 2) v += __shfl_xor_sync(~0u, v, k);
    if (blockDim.x > 32) {
      float* s = place + 32 * turn;
      turn ^= 1;
      const int lane = threadIdx.x % 32;
      if (lane == 0) s[threadIdx.x / 32] = v;
      __syncthreads();
      v = lane < (int)blockDim.x / 32 ? s[lane] : 0.f;
#pragma unroll
      for (int k = 16; k > 0; k /= 2) v += __shfl_xor_sync(~0u, v, k);
    }
    return v;
  }
};

struct Norm {
  const void *x, *z, *res, *dy, *dres_out;
  void *y, *res_out, *dx, *dz, *dres;
  Vector w, post, scale;
  float *inv, *inv_post, *part;
  int64_t rows, xs, zs, rs, ys, ros, dys, dros, dxs, dzs, drs;
  int d, groups, norm_first, vectors;   // d: of a group; vectors: of d * groups partial sums a row of `part` holds
  float eps;
};

// A row per warp (blockDim.y of them) or per CTA.
template <typename F>
__device__ __forceinline__ void for_rows(const Norm& p, F f) {
  for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < p.rows; row += (int64_t)gridDim.x * blockDim.y) f(row);
}

template <typename T, typename R, int I, bool VEC>
__global__ void __launch_bounds__(I == 1 ? 256 : 512) rms_norm_kernel(const Norm p) {
  __shared__ float sums[64];
  RowSum row_sum{sums, 0};
  for_rows(p, [&](int64_t row) {
    float v[I][8], old[I][8];
#pragma unroll
    for (int it = 0; it < I; ++it) {
      get8<T, VEC>(static_cast<const T*>(p.x) + row * p.xs, it, p.d, v[it]);
      if (p.res) get8<R, VEC>(static_cast<const R*>(p.res) + row * p.rs, it, p.d, old[it]);
    }
    if (p.post.p) {
      float ss = 0.f;
#pragma unroll
      for (int it = 0; it < I; ++it)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[it][e], v[it][e], ss);
      const float inv = rsqrtf(row_sum(ss) / p.d + p.eps);
      if (p.inv_post && threadIdx.x == 0) p.inv_post[row] = inv;
#pragma unroll
      for (int it = 0; it < I; ++it) {
        float w[8];
        p.post.get<T, VEC>(0, it, p.d, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[it][e] *= inv * w[e];
      }
    }
    if (p.scale.p) {
#pragma unroll
      for (int it = 0; it < I; ++it) {
        float w[8];
        p.scale.get<T, VEC>(0, it, p.d, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[it][e] *= w[e];
      }
    }
    if (p.res) {
#pragma unroll
      for (int it = 0; it < I; ++it) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[it][e] = Cvt<R>::to_f(Cvt<R>::from_f(old[it][e] + v[it][e]));   // as it is stored
        put8<R, VEC>(static_cast<R*>(p.res_out) + row * p.ros, it, p.d, v[it]);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int it = 0; it < I; ++it)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[it][e], v[it][e], ss);
    const float inv = rsqrtf(row_sum(ss) / p.d + p.eps);
    if (p.inv && threadIdx.x == 0) p.inv[row] = inv;
#pragma unroll
    for (int it = 0; it < I; ++it) {
      float w[8];
      p.w.get<T, VEC>(0, it, p.d, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[it][e] *= inv * w[e];
      put8<T, VEC>(static_cast<T*>(p.y) + row * p.ys, it, p.d, v[it]);
    }
  });
}

// Partial sums of this warp's or CTA's rows.
template <int I, bool VEC>
__device__ __forceinline__ void leave(const Norm& p, int which, const float (&sum)[I][8]) {
  const int64_t all = (int64_t)p.d * p.groups;
  float* to = p.part + (((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * p.vectors + which) * all + (int64_t)blockIdx.y * p.d;
#pragma unroll
  for (int it = 0; it < I; ++it)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (place<VEC>(it, e) < p.d) to[place<VEC>(it, e)] = sum[it][e];
}

// OUTER: with post_weight or scale.
template <typename T, typename R, int I, bool VEC, bool OUTER>
__global__ void __launch_bounds__(I == 1 ? 256 : 512) rms_norm_grad_kernel(const Norm p) {
  __shared__ float sums[64];
  RowSum row_sum{sums, 0};
  float dw[I][8] = {}, both[I][8] = {};
  for_rows(p, [&](int64_t row) {
    float g[I][8], v[I][8], in[I][8];
    const float inv = p.inv[row];
#pragma unroll
    for (int it = 0; it < I; ++it) {
      get8<T, VEC>(static_cast<const T*>(p.dy) + row * p.dys, it, p.d, g[it]);
      if (p.res_out) get8<R, VEC>(static_cast<const R*>(p.res_out) + row * p.ros, it, p.d, v[it]);
      else get8<T, VEC>(static_cast<const T*>(p.x) + row * p.xs, it, p.d, v[it]);
      if (p.dres_out) get8<R, VEC>(static_cast<const R*>(p.dres_out) + row * p.dros, it, p.d, in[it]);
    }
    float c = 0.f;
#pragma unroll
    for (int it = 0; it < I; ++it) {
      float w[8];
      p.w.get<T, VEC>(0, it, p.d, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[it][e] *= inv;
        dw[it][e] = fmaf(g[it][e], v[it][e], dw[it][e]);
        g[it][e] *= w[e];
        c = fmaf(g[it][e], v[it][e], c);
      }
    }
    c = row_sum(c) / p.d;
#pragma unroll
    for (int it = 0; it < I; ++it) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[it][e] = inv * fmaf(-v[it][e], c, g[it][e]);
        if (p.dres_out) g[it][e] += in[it][e];
      }
      if (p.dres) put8<R, VEC>(static_cast<R*>(p.dres) + row * p.drs, it, p.d, g[it]);
    }
    if constexpr (OUTER) {
      const float invp = p.post.p ? p.inv_post[row] : 1.f;
      float c2 = 0.f;
#pragma unroll
      for (int it = 0; it < I; ++it) {
        float w[8];
        get8<T, VEC>(static_cast<const T*>(p.x) + row * p.xs, it, p.d, v[it]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[it][e] *= invp;
          both[it][e] = fmaf(g[it][e], v[it][e], both[it][e]);
        }
        if (p.scale.p) {
          p.scale.get<T, VEC>(0, it, p.d, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[it][e] *= w[e];
        }
        if (p.post.p) {
          p.post.get<T, VEC>(0, it, p.d, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            g[it][e] *= w[e];
            c2 = fmaf(g[it][e], v[it][e], c2);
          }
        }
      }
      if (p.post.p) {
        c2 = row_sum(c2) / p.d;
#pragma unroll
        for (int it = 0; it < I; ++it)
#pragma unroll
          for (int e = 0; e < 8; ++e) g[it][e] = invp * fmaf(-v[it][e], c2, g[it][e]);
      }
    }
#pragma unroll
    for (int it = 0; it < I; ++it) put8<T, VEC>(static_cast<T*>(p.dx) + row * p.dxs, it, p.d, g[it]);
  });
  leave<I, VEC>(p, 0, dw);
  if constexpr (OUTER) leave<I, VEC>(p, 1, both);
}

template <typename T, int I, bool VEC>
__global__ void __launch_bounds__(I == 1 ? 256 : 512) gated_rms_norm_kernel(const Norm p) {
  __shared__ float sums[64];
  RowSum row_sum{sums, 0};
  const int first = blockIdx.y * p.d;
  for_rows(p, [&](int64_t row) {
    float v[I][8], z[I][8];
#pragma unroll
    for (int it = 0; it < I; ++it) {
      get8<T, VEC>(static_cast<const T*>(p.x) + row * p.xs + first, it, p.d, v[it]);
      get8<T, VEC>(static_cast<const T*>(p.z) + row * p.zs + first, it, p.d, z[it]);
    }
    float ss = 0.f;
#pragma unroll
    for (int it = 0; it < I; ++it)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[it][e] *= sigmoid_approx(z[it][e]);
        if (!p.norm_first) v[it][e] *= z[it][e];
        ss = fmaf(v[it][e], v[it][e], ss);
      }
    const float inv = rsqrtf(row_sum(ss) / p.d + p.eps);
    if (p.inv && threadIdx.x == 0) p.inv[row * p.groups + blockIdx.y] = inv;
#pragma unroll
    for (int it = 0; it < I; ++it) {
      float w[8];
      p.w.get<T, VEC>(first, it, p.d, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[it][e] *= inv * w[e];
        if (p.norm_first) v[it][e] *= z[it][e];
      }
      put8<T, VEC>(static_cast<T*>(p.y) + row * p.ys + first, it, p.d, v[it]);
    }
  });
}

template <typename T, int I, bool VEC>
__global__ void __launch_bounds__(I == 1 ? 256 : 512) gated_rms_norm_grad_kernel(const Norm p) {
  __shared__ float sums[64];
  RowSum row_sum{sums, 0};
  const int first = blockIdx.y * p.d;
  float dw[I][8] = {};
  for_rows(p, [&](int64_t row) {
    float x[I][8], z[I][8], g[I][8];
    const float inv = p.inv[row * p.groups + blockIdx.y];
#pragma unroll
    for (int it = 0; it < I; ++it) {
      get8<T, VEC>(static_cast<const T*>(p.x) + row * p.xs + first, it, p.d, x[it]);
      get8<T, VEC>(static_cast<const T*>(p.z) + row * p.zs + first, it, p.d, z[it]);
      get8<T, VEC>(static_cast<const T*>(p.dy) + row * p.dys + first, it, p.d, g[it]);
    }
    float c = 0.f;
#pragma unroll
    for (int it = 0; it < I; ++it) {
      float w[8];
      p.w.get<T, VEC>(first, it, p.d, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float gate = z[it][e] * sigmoid_approx(z[it][e]);
        const float vh = inv * (p.norm_first ? x[it][e] : x[it][e] * gate);
        if (p.norm_first) {
          dw[it][e] = fmaf(g[it][e] * gate, vh, dw[it][e]);
          c = fmaf(g[it][e] * gate * w[e], vh, c);
        } else {
          dw[it][e] = fmaf(g[it][e], vh, dw[it][e]);
          c = fmaf(g[it][e] * w[e], vh, c);
        }
        g[it][e] *= w[e];
      }
    }
    c = row_sum(c) / p.d;
#pragma unroll
    for (int it = 0; it < I; ++it) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = sigmoid_approx(z[it][e]), gate = z[it][e] * s, slope = s * fmaf(z[it][e], 1.f - s, 1.f);
        if (p.norm_first) {
          const float vh = inv * x[it][e];
          z[it][e] = g[it][e] * vh * slope;
          x[it][e] = inv * fmaf(-vh, c, g[it][e] * gate);
        } else {
          const float dv = inv * fmaf(-inv * (x[it][e] * gate), c, g[it][e]);
          z[it][e] = dv * x[it][e] * slope;
          x[it][e] = dv * gate;
        }
      }
      put8<T, VEC>(static_cast<T*>(p.dx) + row * p.dxs + first, it, p.d, x[it]);
      put8<T, VEC>(static_cast<T*>(p.dz) + row * p.dzs + first, it, p.d, z[it]);
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
  unsigned grid;                 // CTAs a group
};
// Eight numbers a thread up to 2 048 a row, sixteen up to 8 192, 32 beyond.  Rows of a warp go four to a CTA.  Gradients: as many CTAs as
// stay on the chip, each with its sums over rows.
Shape shape_of(int64_t rows, int d, int groups, bool grad) {
  Shape s;
  const int eights = (d + 7) / 8;
  s.steps = eights <= 256 ? 1 : eights <= 1024 ? 2 : 4;
  s.threads = ((eights + s.steps - 1) / s.steps + 31) / 32 * 32;
  s.rows = s.threads == 32 ? 4 : 1;
  int64_t grid = (rows + s.rows - 1) / s.rows;
  const int64_t most = grad ? std::max(1, 148 * std::max(1, 1024 / (s.threads * s.rows)) / groups) : 0x7fffffff;
  s.grid = (unsigned)std::min(grid, most);
  return s;
}

int check(const SsdNormArgs* a, bool gated, bool grad) {
  if (!a) return SSD_ERR_NULL_POINTER;
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

template <typename T>
struct Launch {
  Norm p = {};
  Shape s;
  bool vec = true;
  cudaStream_t stream;
  Launch(const SsdNormArgs& a, bool gated, bool grad, cudaStream_t st) : stream(st) {
    p.rows = a.rows; p.groups = gated ? a.groups : 1; p.d = a.d / p.groups; p.eps = a.eps; p.norm_first = a.norm_first;
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

  template <typename K>
  int go(K kernel) const {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(s.grid, (unsigned)p.groups);
    cfg.blockDim = dim3((unsigned)s.threads, (unsigned)s.rows);
    cfg.stream = stream;
    return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? SSD_OK : SSD_ERR_CUDA;
  }
  template <typename R>
  int forward() const {
    if (s.steps == 1) return go(vec ? rms_norm_kernel<T, R, 1, true> : rms_norm_kernel<T, R, 1, false>);
    if (s.steps == 2) return go(vec ? rms_norm_kernel<T, R, 2, true> : rms_norm_kernel<T, R, 2, false>);
    return go(vec ? rms_norm_kernel<T, R, 4, true> : rms_norm_kernel<T, R, 4, false>);
  }
  template <typename R, bool OUTER>
  int backward() const {
    if (s.steps == 1) return go(vec ? rms_norm_grad_kernel<T, R, 1, true, OUTER> : rms_norm_grad_kernel<T, R, 1, false, OUTER>);
    if (s.steps == 2) return go(vec ? rms_norm_grad_kernel<T, R, 2, true, OUTER> : rms_norm_grad_kernel<T, R, 2, false, OUTER>);
    return go(vec ? rms_norm_grad_kernel<T, R, 4, true, OUTER> : rms_norm_grad_kernel<T, R, 4, false, OUTER>);
  }
  int gated() const {
    if (s.steps == 1) return go(vec ? gated_rms_norm_kernel<T, 1, true> : gated_rms_norm_kernel<T, 1, false>);
    if (s.steps == 2) return go(vec ? gated_rms_norm_kernel<T, 2, true> : gated_rms_norm_kernel<T, 2, false>);
    return go(vec ? gated_rms_norm_kernel<T, 4, true> : gated_rms_norm_kernel<T, 4, false>);
  }
  int gated_backward() const {
    if (s.steps == 1) return go(vec ? gated_rms_norm_grad_kernel<T, 1, true> : gated_rms_norm_grad_kernel<T, 1, false>);
    if (s.steps == 2) return go(vec ? gated_rms_norm_grad_kernel<T, 2, true> : gated_rms_norm_grad_kernel<T, 2, false>);
    return go(vec ? gated_rms_norm_grad_kernel<T, 4, true> : gated_rms_norm_grad_kernel<T, 4, false>);
  }
  int vectors(const SsdNormArgs& a) const {
    if (!a.dweight && !a.dpost_weight && !a.dscale) return SSD_OK;
    const int all = a.d * p.vectors;
    return launch_column_sum(p.part, (int64_t)s.grid * s.rows, all, all,
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
  return (size_t)s.grid * s.rows * a->d * (!a->z && (a->post_weight || a->scale) ? 2 : 1) * sizeof(float);
}

extern "C" int ssd_b200_rms_norm(const SsdNormArgs* args, void* stream) {
  if (const int rc = ssd::check(args, false, false)) return rc;
  const SsdNormArgs& a = *args;
  return ssd::by_type(a.dtype, [&](auto t) -> int {
    using T = decltype(t);
    const ssd::Launch<T> l(a, false, false, static_cast<cudaStream_t>(stream));
    if (!a.residual || a.residual_dtype == a.dtype) return l.template forward<T>();
    return a.residual_dtype == SSD_DTYPE_F32 ? l.template forward<float>() : (int)SSD_ERR_UNSUPPORTED;
  });
}

extern "C" int ssd_b200_rms_norm_backward(const SsdNormArgs* args, void* stream) {
  if (const int rc = ssd::check(args, false, true)) return rc;
  const SsdNormArgs& a = *args;
  return ssd::by_type(a.dtype, [&](auto t) -> int {
    using T = decltype(t);
    const ssd::Launch<T> l(a, false, true, static_cast<cudaStream_t>(stream));
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
    const ssd::Launch<decltype(t)> l(*args, true, true, static_cast<cudaStream_t>(stream));
    const int rc = l.gated_backward();
    return rc ? rc : l.vectors(*args);
  });
}
