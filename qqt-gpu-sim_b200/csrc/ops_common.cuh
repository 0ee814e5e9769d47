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

// VEC consecutive elements, moved by one access of their whole size; 16-bit
// elements stay packed in 32-bit words (a word a pair) until they are read.
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec;
template <int VEC>
struct alignas(4 * VEC) Vec<float, VEC> {
  float v[VEC];
  __device__ __forceinline__ float get(int j) const { return v[j]; }
  __device__ __forceinline__ void put(const float* f) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = f[j];
  }
};
template <>
struct alignas(2) Vec<__half, 1> {
  __half v;
  __device__ __forceinline__ float get(int) const { return __half2float(v); }
  __device__ __forceinline__ void put(const float* f) { v = __float2half_rn(f[0]); }
};
template <>
struct alignas(2) Vec<__nv_bfloat16, 1> {
  __nv_bfloat16 v;
  __device__ __forceinline__ float get(int) const { return __bfloat162float(v); }
  __device__ __forceinline__ void put(const float* f) { v = __float2bfloat16_rn(f[0]); }
};
template <int VEC>
struct alignas(2 * VEC) Vec<__half, VEC> {
  uint32_t w[VEC / 2];
  __device__ __forceinline__ float get(int j) const {
    const __half2 h = *reinterpret_cast<const __half2*>(&w[j / 2]);
    return j & 1 ? __high2float(h) : __low2float(h);
  }
  __device__ __forceinline__ void put(const float* f) {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
template <int VEC>
struct alignas(2 * VEC) Vec<__nv_bfloat16, VEC> {
  uint32_t w[VEC / 2];
  __device__ __forceinline__ float get(int j) const {   // a bfloat16 is a float's upper half
    return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
  __device__ __forceinline__ void put(const float* f) {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
// The access of that size: a vector type, so that a pair of 16-bit elements
// is not taken apart into two registers by the load.
template <int BYTES>
struct Word;
template <>
struct Word<2> {
  using type = unsigned short;
};
template <>
struct Word<4> {
  using type = unsigned;
};
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<16> {
  using type = uint4;
};
template <class T, int VEC>
__device__ __forceinline__ Vec<T, VEC> ld_vec(const T* p) {
  using W = typename Word<sizeof(T) * VEC>::type;
  const W w = *reinterpret_cast<const W*>(p);
  return *reinterpret_cast<const Vec<T, VEC>*>(&w);
}
template <class T, int VEC>
__device__ __forceinline__ void st_vec(T* p, const Vec<T, VEC>& x) {
  using W = typename Word<sizeof(T) * VEC>::type;
  *reinterpret_cast<W*>(p) = *reinterpret_cast<const W*>(&x);
}
template <class T, int VEC>
__device__ __forceinline__ Vec<T, VEC> vec_zero() {
  Vec<T, VEC> x;
  const float z[VEC] = {};
  x.put(z);
  return x;
}
static inline bool aligned_to(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// Pairs of floats, one instruction for both.
typedef float2 f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) { return make_float2(lo, hi); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { return __ffma2_rn(a, b, c); }

// Rows staged by bulk copies: one mbarrier per stage, armed with the bytes of
// its copies.  Waits are bounded; a wait that runs out is reported by the
// device error word.  The kernel then issues no further copy, waits (bounded)
// for those in flight and goes on to its end; what it writes is not valid.
constexpr uint32_t kStagePolls = 1u << 24;
__device__ __forceinline__ uint32_t stage_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void stage_init(uint64_t* bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(stage_addr(bar)) : "memory");
}
__device__ __forceinline__ void stage_init_done() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void stage_arm(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(stage_addr(bar)),
               "r"(bytes)
               : "memory");
}
// bytes: a multiple of 16; both addresses on 16 bytes.
__device__ __forceinline__ void stage_copy(void* dst, const void* src, uint32_t bytes,
                                           uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          stage_addr(dst)),
      "l"(src), "r"(bytes), "r"(stage_addr(bar))
      : "memory");
}
// False once `polls` polls have run out; the copy is then given as many again,
// so that it is not left in flight.
__device__ __forceinline__ bool stage_wait(uint64_t* bar, uint32_t parity,
                                           uint32_t polls = kStagePolls) {
  for (uint32_t i = 0; i < 2 * polls; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(stage_addr(bar)), "r"(parity)
        : "memory");
    if (ok) {
      if (i < polls) return true;
      break;
    }
  }
  flag_error(QQT_DEV_TIMEOUT);
  return false;
}

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

// Kernels of one call launched while the one before still runs: such a kernel
// waits for that one's results with before_me_done(); let_next_start() allows
// the next to be launched before this one ends.
__device__ __forceinline__ void before_me_done() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// early: the kernel before it in the stream is one of the same call's.  A
// failure is left for launch_status.
template <class... P, class... A>
static void launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                         bool early, A... args) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  (void)cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// SMs of the current device (148 where it cannot be asked).
static int sm_count() {
  static std::atomic<int> n{0};
  int v = n.load();
  if (v == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0)
      v = 148;
    n.store(v);
  }
  return v;
}

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
