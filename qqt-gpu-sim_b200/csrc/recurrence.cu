// Gated linear recurrence over T ticks of N sequences of width D, with resets
// at episode ends (the memory of a policy over its rollout).
//   f = sigmoid(gate_t),  k = 0 where reset_t else 1
//   h_t = f k h_{t-1} + (1 - f) x_t
// and its gradient, with e_t = dL/dh_t summed over every later use:
//   e_t = dh_t + f_{t+1} k_{t+1} e_{t+1}      (+ dh_last at the last tick)
//   dx_t = (1 - f) e_t,   dgate_t = f (1 - f) e_t (k h_{t-1} - x_t)
//   dh0 = f_1 k_1 e_1
// States are float32 whatever the type of the sequence.  The backward pass
// recomputes them from the state entering every kRecChunk ticks, which the
// forward pass saves in float32: rounded outputs are not read back.

#include "ops_common.cuh"

namespace qqt {

constexpr int kRecChunk = 64;

// f = sigmoid(g) and i = 1 - f = sigmoid(-g), each to float32 accuracy: with
// e = exp(-|g|) the larger of the two is 1/(1+e) and the smaller e/(1+e).
__device__ __forceinline__ void gates(float g, float& f, float& i) {
  const float e = expf(-fabsf(g));
  const float big = 1.f / (1.f + e);
  const float small = e * big;
  f = g < 0.f ? small : big;
  i = g < 0.f ? big : small;
}

struct RecSeq {            // one (T, N, D) sequence: element strides of t and n
  const void* p;
  int64_t ts, ns;
};

template <class T>
__global__ void k_rec_fwd(RecSeq x, RecSeq g, RecSeq reset, const float* __restrict__ h0, int64_t nT,
                          int64_t nN, int64_t nD, RecSeq h, float* __restrict__ h_last,
                          float* __restrict__ carry) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= nN * nD) return;
  const int64_t n = c / nD, d = c % nD;
  const T* xp = (const T*)x.p + n * x.ns + d;
  const T* gp = (const T*)g.p + n * g.ns + d;
  T* hp = (T*)h.p + n * h.ns + d;
  const uint8_t* rp = (const uint8_t*)reset.p + n * reset.ns;
  float s = h0 ? h0[c] : 0.f;
  for (int64_t t = 0; t < nT; ++t) {
    if (carry && t % kRecChunk == 0) carry[(t / kRecChunk) * nN * nD + c] = s;
    float f, i;
    gates(to_f(gp[t * g.ts]), f, i);
    const float prev = reset.p && rp[t * reset.ts] ? 0.f : s;
    s = fmaf(f, prev, i * to_f(xp[t * x.ts]));
    if (h.p) hp[t * h.ts] = from_f<T>(s);
  }
  if (h_last) h_last[c] = s;
}

template <class T>
__global__ void k_rec_bwd(RecSeq dh, const float* __restrict__ dh_last, RecSeq x, RecSeq g,
                          RecSeq reset, const float* __restrict__ carry, int64_t nT, int64_t nN,
                          int64_t nD, RecSeq dx, RecSeq dg, float* __restrict__ dh0) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= nN * nD) return;
  const int64_t n = c / nD, d = c % nD;
  const T* xp = (const T*)x.p + n * x.ns + d;
  const T* gp = (const T*)g.p + n * g.ns + d;
  const T* dhp = (const T*)dh.p + n * dh.ns + d;
  T* dxp = (T*)dx.p + n * dx.ns + d;
  T* dgp = (T*)dg.p + n * dg.ns + d;
  const uint8_t* rp = (const uint8_t*)reset.p + n * reset.ns;
  float e = dh_last ? dh_last[c] : 0.f;
  float prev[kRecChunk];
  for (int64_t k = (nT + kRecChunk - 1) / kRecChunk - 1; k >= 0; --k) {
    const int64_t t0 = k * kRecChunk;
    const int len = (int)(nT - t0 < kRecChunk ? nT - t0 : kRecChunk);
    float s = carry[k * nN * nD + c], f, i;
    for (int j = 0; j < len; ++j) {
      if (reset.p && rp[(t0 + j) * reset.ts]) s = 0.f;
      prev[j] = s;
      gates(to_f(gp[(t0 + j) * g.ts]), f, i);
      s = fmaf(f, s, i * to_f(xp[(t0 + j) * x.ts]));
    }
    for (int j = len - 1; j >= 0; --j) {
      const int64_t t = t0 + j;
      gates(to_f(gp[t * g.ts]), f, i);
      if (dh.p) e += to_f(dhp[t * dh.ts]);
      const float ie = i * e;
      dxp[t * dx.ts] = from_f<T>(ie);
      dgp[t * dg.ts] = from_f<T>(f * ie * (prev[j] - to_f(xp[t * x.ts])));
      e = reset.p && rp[t * reset.ts] ? 0.f : f * e;
    }
  }
  if (dh0) dh0[c] = e;
}

static bool rec_sizes_ok(int64_t T, int64_t N, int64_t D) { return T >= 0 && N >= 0 && D > 0; }

}  // namespace qqt

using namespace qqt;

extern "C" int64_t qqt_recurrence_chunks(int64_t T) { return T <= 0 ? 0 : (T + kRecChunk - 1) / kRecChunk; }

extern "C" uint64_t qqt_recurrence_work_bytes(int64_t T, int64_t N, int64_t D) {
  (void)T;
  (void)N;
  (void)D;
  return 16;
}

extern "C" int qqt_recurrence_forward(const QqtSeq* x, const QqtSeq* gate, const QqtSeq* reset,
                                      const float* h0, int32_t dtype, int64_t T, int64_t N,
                                      int64_t D, const QqtSeq* h, float* h_last, float* carry,
                                      void* work, qqt_stream_t stream) {
  (void)work;
  if (!x || !gate || !h || !dtype_ok(dtype) || !rec_sizes_ok(T, N, D)) return QQT_E_ARG;
  if (N * D == 0) return QQT_OK;
  if (T > 0 && (!x->p || !gate->p)) return QQT_E_ARG;
  const RecSeq none{nullptr, 0, 0};
  return with_dtype(dtype, [&](auto t) {
    using E = decltype(t);
    k_rec_fwd<E><<<(unsigned)((N * D + 127) / 128), 128, 0, (cudaStream_t)stream>>>(
        RecSeq{x->p, x->t_stride, x->n_stride}, RecSeq{gate->p, gate->t_stride, gate->n_stride},
        reset ? RecSeq{reset->p, reset->t_stride, reset->n_stride} : none, h0, T, N, D,
        RecSeq{h->p, h->t_stride, h->n_stride}, h_last, carry);
    return launch_status();
  });
}

extern "C" int qqt_recurrence_backward(const QqtSeq* dh, const float* dh_last, const QqtSeq* x,
                                       const QqtSeq* gate, const QqtSeq* reset, const float* carry,
                                       int32_t dtype, int64_t T, int64_t N, int64_t D,
                                       const QqtSeq* dx, const QqtSeq* dgate, float* dh0, void* work,
                                       qqt_stream_t stream) {
  (void)work;
  if (!x || !gate || !dx || !dgate || !dtype_ok(dtype) || !rec_sizes_ok(T, N, D)) return QQT_E_ARG;
  if (N * D == 0) return QQT_OK;
  if (T > 0 && (!x->p || !gate->p || !dx->p || !dgate->p || !carry)) return QQT_E_ARG;
  const RecSeq none{nullptr, 0, 0};
  return with_dtype(dtype, [&](auto t) {
    using E = decltype(t);
    k_rec_bwd<E><<<(unsigned)((N * D + 127) / 128), 128, 0, (cudaStream_t)stream>>>(
        dh ? RecSeq{dh->p, dh->t_stride, dh->n_stride} : none, dh_last,
        RecSeq{x->p, x->t_stride, x->n_stride}, RecSeq{gate->p, gate->t_stride, gate->n_stride},
        reset ? RecSeq{reset->p, reset->t_stride, reset->n_stride} : none, carry, T, N, D,
        RecSeq{dx->p, dx->t_stride, dx->n_stride}, RecSeq{dgate->p, dgate->t_stride, dgate->n_stride},
        dh0);
    return launch_status();
  });
}
