// Layer norm over the last d values of each row, forward and backward
// (the norms of the MLP and CNN policies, train/model.py:77-101, 140-153, and
// of the memory policy).
//   y  = (x - mean) rstd w + b,   rstd = 1 / sqrt(var + eps)
//   dx = rstd (q - mean(q) - xh mean(q xh)),  q = dy w,  xh = (x - mean) rstd
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// All statistics and sums are float32; outputs are rounded once.

#include "ops_common.cuh"

namespace qqt {

template <class T>
__global__ void k_ln_fwd(const T* __restrict__ x, int64_t xs, int64_t d, const float* __restrict__ w,
                         const float* __restrict__ b, float eps, T* __restrict__ y,
                         float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float buf[32];
  const int64_t r = blockIdx.x;
  x += r * xs;
  y += r * d;
  float s = 0.f;
  for (int64_t j = threadIdx.x; j < d; j += blockDim.x) s += to_f(x[j]);
  const float mu = block_sum(s, buf) / (float)d;
  s = 0.f;
  for (int64_t j = threadIdx.x; j < d; j += blockDim.x) {
    const float c = to_f(x[j]) - mu;
    s = fmaf(c, c, s);
  }
  const float rs = 1.f / sqrtf(block_sum(s, buf) / (float)d + eps);
  for (int64_t j = threadIdx.x; j < d; j += blockDim.x)
    y[j] = from_f<T>(fmaf((to_f(x[j]) - mu) * rs, w[j], b ? b[j] : 0.f));
  if (threadIdx.x == 0) {
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

template <class T>
__global__ void k_ln_dx(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                        int64_t d, const float* __restrict__ mean, const float* __restrict__ rstd,
                        const float* __restrict__ w, T* __restrict__ dx) {
  __shared__ float buf[32];
  const int64_t r = blockIdx.x;
  x += r * xs;
  dy += r * dys;
  dx += r * d;
  const float mu = mean[r], rs = rstd[r];
  float s1 = 0.f, s2 = 0.f;
  for (int64_t j = threadIdx.x; j < d; j += blockDim.x) {
    const float q = to_f(dy[j]) * w[j];
    s1 += q;
    s2 = fmaf(q, (to_f(x[j]) - mu) * rs, s2);
  }
  s1 = block_sum(s1, buf) / (float)d;
  s2 = block_sum(s2, buf) / (float)d;
  for (int64_t j = threadIdx.x; j < d; j += blockDim.x) {
    const float q = to_f(dy[j]) * w[j];
    dx[j] = from_f<T>(rs * (q - s1 - (to_f(x[j]) - mu) * rs * s2));
  }
}

constexpr int kLnParts = 512;   // row groups of the weight gradient's first stage

template <class T>
__global__ void k_ln_dw_part(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x,
                             int64_t xs, int64_t rows, int64_t d, const float* __restrict__ mean,
                             const float* __restrict__ rstd, float* __restrict__ part) {
  const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= d) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = to_f(dy[r * dys + j]);
    sb += g;
    sw = fmaf(g, (to_f(x[r * xs + j]) - mean[r]) * rstd[r], sw);
  }
  part[(int64_t)blockIdx.y * 2 * d + j] = sw;
  part[(int64_t)blockIdx.y * 2 * d + d + j] = sb;
}

__global__ void k_ln_dw_sum(const float* __restrict__ part, int n_part, int64_t d,
                            float* __restrict__ dw, float* __restrict__ db) {
  const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= 2 * d) return;
  float s = 0.f;
  for (int p = 0; p < n_part; ++p) s += part[(int64_t)p * 2 * d + j];
  float* out = j < d ? dw : db;
  if (out) out[j < d ? j : j - d] = s;
}

static int ln_parts(int64_t rows) { return (int)(rows < kLnParts ? (rows > 0 ? rows : 1) : kLnParts); }

}  // namespace qqt

using namespace qqt;

extern "C" uint64_t qqt_layernorm_work_bytes(int64_t rows, int64_t d) {
  if (rows < 0 || d <= 0) return 0;
  return (uint64_t)ln_parts(rows) * 2 * (uint64_t)d * sizeof(float);
}

extern "C" int qqt_layernorm_forward(const void* x, int32_t dtype, int64_t rows, int64_t d,
                                     int64_t x_stride, const float* w, const float* b, float eps,
                                     void* y, float* mean, float* rstd, qqt_stream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || d <= 0 || x_stride < 0 || !(eps >= 0.f)) return QQT_E_ARG;
  if (rows > 0x7fffffffll || d > 0x7fffffffll) return QQT_E_LIMIT;
  if (rows == 0) return QQT_OK;
  if (!x || !w || !y) return QQT_E_ARG;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_ln_fwd<T><<<(unsigned)rows, 256, 0, (cudaStream_t)stream>>>((const T*)x, x_stride, d, w, b,
                                                                  eps, (T*)y, mean, rstd);
    return launch_status();
  });
}

extern "C" int qqt_layernorm_backward(const void* dy, int64_t dy_stride, const void* x,
                                      int64_t x_stride, int32_t dtype, int64_t rows, int64_t d,
                                      const float* mean, const float* rstd, const float* w,
                                      void* dx, float* dw, float* db, void* work,
                                      qqt_stream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || d <= 0 || x_stride < 0 || dy_stride < 0) return QQT_E_ARG;
  if (rows > 0x7fffffffll || d > 0x7fffffffll) return QQT_E_LIMIT;
  if (rows > 0 && (!dy || !x || !mean || !rstd || !w)) return QQT_E_ARG;
  if ((dw || db) && !work) return QQT_E_ARG;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    if (dx && rows > 0)
      k_ln_dx<T><<<(unsigned)rows, 256, 0, st>>>((const T*)dy, dy_stride, (const T*)x, x_stride, d,
                                                 mean, rstd, w, (T*)dx);
    if (dw || db) {
      const int parts = ln_parts(rows);
      k_ln_dw_part<T><<<dim3((unsigned)((d + 127) / 128), parts), 128, 0, st>>>(
          (const T*)dy, dy_stride, (const T*)x, x_stride, rows, d, mean, rstd, (float*)work);
      k_ln_dw_sum<<<(unsigned)((2 * d + 127) / 128), 128, 0, st>>>((const float*)work, parts, d, dw,
                                                                    db);
    }
    return launch_status();
  });
}
