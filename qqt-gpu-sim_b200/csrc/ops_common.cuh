// Shared device code of the training operators (layer norm, gated recurrence,
// policy loss): element types, block sums and NaN-keeping extremes.
//
// The library is built with -fmad=false for the simulator's arithmetic, so
// fused multiply-adds are written out (fmaf) where an operator wants them.
#pragma once

#include <cuda_bf16.h>

#include "qqt_common.cuh"

namespace qqt {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// VEC consecutive elements, moved by one access of their whole size.
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ Vec<T, VEC> ld_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, VEC>*>(p);
}
template <class T, int VEC>
__device__ __forceinline__ void st_vec(T* p, const Vec<T, VEC>& x) {
  *reinterpret_cast<Vec<T, VEC>*>(p) = x;
}
static inline bool aligned_to(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// 2^x and 1/x by the special-function unit (relative errors of about 2^-22).
__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Maximum that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(QQT_FULL, v, o);
  return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(QQT_FULL, v, o));
  return v;
}

// Sum over the block in a fixed order, known to every thread.  buf: 32 floats
// of shared memory, free to be reused after the call's closing barrier.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  const int nw = (blockDim.x + 31) >> 5;
  v = warp_sum_f(v);
  if (lane_id() == 0) buf[warp_id()] = v;
  __syncthreads();
  v = lane_id() < nw ? buf[lane_id()] : 0.f;
  v = warp_sum_f(v);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_max_nan(float v, float* buf) {
  const int nw = (blockDim.x + 31) >> 5;
  v = warp_max_nan(v);
  if (lane_id() == 0) buf[warp_id()] = v;
  __syncthreads();
  v = lane_id() < nw ? buf[lane_id()] : buf[0];
  v = warp_max_nan(v);
  __syncthreads();
  return v;
}

static inline int elem_bytes(int32_t dtype) { return dtype == QQT_F32 ? 4 : 2; }
static inline bool dtype_ok(int32_t dtype) { return dtype >= QQT_F32 && dtype <= QQT_BF16; }

// Runs f(T{}) with the element type of `dtype`.
template <class F>
static inline int with_dtype(int32_t dtype, F f) {
  switch (dtype) {
    case QQT_F32: return f(float{});
    case QQT_F16: return f(__half{});
    case QQT_BF16: return f(__nv_bfloat16{});
  }
  return QQT_E_ARG;
}

}  // namespace qqt
