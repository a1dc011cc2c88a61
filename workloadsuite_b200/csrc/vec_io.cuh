// Two consecutive numbers of a row, packed fp32 pairs, and sums over columns: what the kernels of the layer's pieces share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ssd_common.cuh"

namespace ssd {

// Two fp32 numbers that one instruction works on.
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ Pair both(float v) { return pair(v, v); }
__device__ __forceinline__ float2 halves(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
template <typename F>
__device__ __forceinline__ Pair each(Pair p, F f) {
  const float2 h = halves(p);
  return pair(f(h.x), f(h.y));
}

// Two numbers of type T as they lie in memory.
template <typename T> struct Two;
template <> struct Two<float> {
  using Raw = float2;
  static __device__ __forceinline__ Raw zero() { return make_float2(0.f, 0.f); }
  static __device__ __forceinline__ float2 up(Raw v) { return v; }
  static __device__ __forceinline__ Raw down(float a, float b) { return make_float2(a, b); }
  static __device__ __forceinline__ Raw join(float a, float b) { return make_float2(a, b); }
  static __device__ __forceinline__ float lo(Raw v) { return v.x; }
  static __device__ __forceinline__ float hi(Raw v) { return v.y; }
  static __device__ __forceinline__ Raw least(Raw a, Raw b) { return make_float2(fminf(a.x, b.x), fminf(a.y, b.y)); }
};
template <> struct Two<__half> {
  using Raw = uint32_t;
  static __device__ __forceinline__ Raw zero() { return 0u; }
  static __device__ __forceinline__ float2 up(Raw v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ Raw down(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ Raw join(__half a, __half b) { return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16; }
  static __device__ __forceinline__ __half lo(Raw v) { return __ushort_as_half((unsigned short)v); }
  static __device__ __forceinline__ __half hi(Raw v) { return __ushort_as_half((unsigned short)(v >> 16)); }
  static __device__ __forceinline__ Raw least(Raw a, Raw b) {
    const __half2 h = __hmin2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Two<__nv_bfloat16> {
  using Raw = uint32_t;
  static __device__ __forceinline__ Raw zero() { return 0u; }
  static __device__ __forceinline__ float2 up(Raw v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
  static __device__ __forceinline__ Raw down(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ Raw join(__nv_bfloat16 a, __nv_bfloat16 b) {
    return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16;
  }
  static __device__ __forceinline__ __nv_bfloat16 lo(Raw v) { return __ushort_as_bfloat16((unsigned short)v); }
  static __device__ __forceinline__ __nv_bfloat16 hi(Raw v) { return __ushort_as_bfloat16((unsigned short)(v >> 16)); }
  static __device__ __forceinline__ Raw least(Raw a, Raw b) {
    const __nv_bfloat162 h = __hmin2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename T>
__device__ __forceinline__ Pair pair_of(typename Two<T>::Raw v) {
  const float2 f = Two<T>::up(v);
  return pair(f.x, f.y);
}

// A lane's two channels: neighbours read at once (VEC), or `apart` elements from each other and each only if it is there.
// What is not there reads as `missing`.
template <typename T, bool VEC>
__device__ __forceinline__ typename Two<T>::Raw load_two(const T* p, int apart, bool ok0, bool ok1, float missing = 0.f) {
  if constexpr (VEC) {
    return ok0 ? *reinterpret_cast<const typename Two<T>::Raw*>(p) : Two<T>::down(missing, missing);
  } else {
    const T z = Cvt<T>::from_f(missing);
    const T a = ok0 ? p[0] : z, b = ok1 ? p[apart] : z;
    return Two<T>::join(a, b);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_two(T* p, int apart, bool ok0, bool ok1, Pair f) {
  const float2 h = halves(f);
  const typename Two<T>::Raw v = Two<T>::down(h.x, h.y);
  if constexpr (VEC) {
    if (ok0) *reinterpret_cast<typename Two<T>::Raw*>(p) = v;
  } else {
    if (ok0) p[0] = Two<T>::lo(v);
    if (ok1) p[apart] = Two<T>::hi(v);
  }
}

// Functions of the special-function unit: relative errors of 2^-22 and less, infinities and NaN as IEEE has them.  Numbers below the normal
// ones count as zero: what would keep them takes four more instructions.
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rsqrt_approx(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2E = 1.4426950408889634f;
// 1 / (1 + e^-v): exactly 0 at -infinity (and below -88), 1 at infinity
__device__ __forceinline__ float sigmoid_approx(float v) { return rcp_approx(1.f + exp2_approx(-kLog2E * v)); }

// out[c] = finish(c, sum over the rows r of part[r * stride + c]), in a fixed order.
// One block: 32 columns, 32 rows at a time.
template <typename Finish>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, int64_t rows, int64_t stride, int columns,
                                                          Finish finish) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, r0 = threadIdx.x / 32;
  float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
  if (c < columns) {
    int64_t r = r0;
    for (; r + 96 < rows; r += 128) {
      a0 += part[r * stride + c];
      a1 += part[(r + 32) * stride + c];
      a2 += part[(r + 64) * stride + c];
      a3 += part[(r + 96) * stride + c];
    }
    for (; r < rows; r += 32) a0 += part[r * stride + c];
  }
  s[r0][threadIdx.x % 32] = (a0 + a1) + (a2 + a3);
  __syncthreads();
  float v = s[threadIdx.x % 32][r0];
#pragma unroll
  for (int k = 16; k > 0; k /= 2) v += __shfl_xor_sync(~0u, v, k);
  const int cc = blockIdx.x * 32 + r0;
  if (threadIdx.x % 32 == 0 && cc < columns) finish(cc, v);
}

template <typename Finish>
int launch_column_sum(const float* part, int64_t rows, int64_t stride, int columns, Finish finish, cudaStream_t stream) {
  return launch(column_sum_kernel<Finish>, (unsigned)((columns + 31) / 32), 1024, 0, stream, part, rows, stride, columns, finish);
}

// f(a number of the type that `dtype` names)
template <typename F>
inline int by_type(int dtype, F f) {
  switch (dtype) {
    case SSD_DTYPE_F32: return f(float());
    case SSD_DTYPE_F16: return f(__half());
    case SSD_DTYPE_BF16: return f(__nv_bfloat16());
    default: return SSD_ERR_UNSUPPORTED;
  }
}

}  // namespace ssd
