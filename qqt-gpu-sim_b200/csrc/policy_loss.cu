// Clipped policy loss with a KL term and an entropy bonus over masked
// categorical heads (train/ppo.py:397-424 with train/model.py:216-256), its
// gradient with respect to the logits, and the log-probabilities alone.
// A row's logits are split into n_heads segments; per head, over its legal
// categories,
//   m = max z,  S = sum exp(z - m),  E = sum exp(z - m) (z - m)
//   log p_j = z_j - m - log S,   H = log S - E / S
// and over the heads  logp = sum log p[action],  H = sum H.  Then
//   r = exp(logp - old),  pg = -min(r A, clip(r, 1 - lo, 1 + hi) A)
//   kl = expm1(q) - q,  q = ref - logp
//   loss = mean over the rows that count of  pg + beta kl - c H
//   dz_j = [G (1[j = action] - p_j) + c p_j (log p_j + H_head)] / count
//   G = (-A r where the clip is not binding) + beta (1 - exp(q))
// Every sum is float32; the gradient is rounded once to the logits' type.

#include "ops_common.cuh"

namespace qqt {

struct HeadStat {
  float m, log_s, ent, z_act;
  bool ok;                  // some category is legal and the action is one of them
};

__global__ void k_pl_count(const uint8_t* __restrict__ mask, int64_t rows, float* __restrict__ out) {
  __shared__ float buf[32];
  int64_t n = 0;
  if (mask)
    for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) n += mask[r] != 0;
  const float c = mask ? block_sum((float)n, buf) : (float)rows;
  if (threadIdx.x == 0) out[0] = c > 1.f ? c : 1.f;
}

// What a row adds to the sums, and its gradient's coefficients.
struct RowLoss {
  float pg, kl, clip, g;
};
__device__ __forceinline__ RowLoss row_loss(float logp, float old, float a, float ref, bool has_ref,
                                            float lo, float hi, float beta) {
  RowLoss o;
  const float r = expf(logp - old);
  const float rc = fminf(fmaxf(r, 1.f - lo), 1.f + hi);
  const float u = r * a, v = rc * a;
  o.pg = -(r != r || a != a ? r * a : fminf(u, v));
  o.clip = r < 1.f - lo || r > 1.f + hi ? 1.f : 0.f;
  const bool bound = (a > 0.f && r > 1.f + hi) || (a < 0.f && r < 1.f - lo);
  o.g = bound ? 0.f : -u;
  o.kl = 0.f;
  if (has_ref) {
    const float q = ref - logp, em = expm1f(q);
    o.kl = em - q;
    o.g = fmaf(-beta, em, o.g);
  }
  return o;
}

template <class T>
__global__ void k_pl_rows(QqtPolicyLoss a, const float* __restrict__ count, float* __restrict__ part) {
  __shared__ float buf[32];
  const int64_t r = blockIdx.x;
  const T* z = (const T*)a.logits + r * a.row_stride;
  const uint8_t* legal = a.legal ? a.legal + r * a.legal_stride : nullptr;
  HeadStat hs[QQT_MAX_HEADS];
  float logp = 0.f, ent = 0.f;
  bool ok = true;
  int at = 0;
  for (int h = 0; h < a.n_heads; ++h) {
    const int w = a.width[h];
    const int64_t act = a.actions[r * a.action_stride + h];
    float m = -INFINITY;
    for (int j = threadIdx.x; j < w; j += blockDim.x)
      if (!legal || legal[at + j]) m = max_nan(m, to_f(z[at + j]));
    m = block_max_nan(m, buf);
    float s = 0.f, e = 0.f;
    for (int j = threadIdx.x; j < w; j += blockDim.x) {
      if (legal && !legal[at + j]) continue;
      const float t = to_f(z[at + j]) - m;
      if (t == -INFINITY) continue;
      const float x = expf(t);
      s += x;
      e = fmaf(x, t, e);
    }
    s = block_sum(s, buf);
    e = block_sum(e, buf);
    HeadStat k;
    const bool in = act >= 0 && act < w;
    if (!in && threadIdx.x == 0) flag_error(QQT_DEV_BAD_ACTION);
    k.z_act = in && (!legal || legal[at + act]) ? to_f(z[at + act]) : -INFINITY;
    k.ok = m != -INFINITY && k.z_act != -INFINITY;
    k.m = m;
    k.log_s = logf(s);
    k.ent = m == -INFINITY ? 0.f : k.log_s - e / s;
    logp += k.ok ? k.z_act - m - k.log_s : -INFINITY;
    ent += k.ent;
    ok = ok && k.ok;
    hs[h] = k;
    at += w;
  }
  if (threadIdx.x == 0) {
    if (a.logp) a.logp[r] = logp;
    if (a.entropy) a.entropy[r] = ent;
  }
  if (!a.old_logp) return;
  const bool live = ok && (!a.mask || a.mask[r]);
  RowLoss l{0.f, 0.f, 0.f, 0.f};
  if (live)
    l = row_loss(logp, a.old_logp[r], a.adv[r], a.ref_logp ? a.ref_logp[r] : 0.f,
                 a.ref_logp != nullptr, a.clip_low, a.clip_high, a.kl_coef);
  if (a.stats && threadIdx.x == 0) {
    part[r * 4 + 0] = l.pg;
    part[r * 4 + 1] = l.kl;
    part[r * 4 + 2] = live ? ent : 0.f;
    part[r * 4 + 3] = l.clip;
  }
  if (!a.dlogits) return;
  const float scale = a.grad_scale / count[0] * (a.upstream ? a.upstream[0] : 1.f);
  T* dz = (T*)a.dlogits + r * a.dlogits_stride;
  at = 0;
  for (int h = 0; h < a.n_heads; ++h) {
    const int w = a.width[h];
    const HeadStat k = hs[h];
    const int64_t act = a.actions[r * a.action_stride + h];
    for (int j = threadIdx.x; j < w; j += blockDim.x) {
      float v = 0.f;
      if (live && (!legal || legal[at + j])) {
        // the terms that may cancel are added unscaled, the scale comes last
        const float lp = to_f(z[at + j]) - k.m - k.log_s;
        const float p = expf(lp);
        const float q = lp == -INFINITY ? 0.f : a.entropy_coef * (lp + k.ent);
        v = scale * (j == act ? fmaf(l.g, 1.f - p, p * q) : p * (q - l.g));
      }
      dz[at + j] = from_f<T>(v);
    }
    at += w;
  }
}

__global__ void k_pl_stats(const float* __restrict__ part, int64_t n, const float* __restrict__ count,
                           float beta, float c, float* __restrict__ stats) {
  __shared__ float buf[32];
  double s[4] = {0., 0., 0., 0.};
  for (int64_t r = threadIdx.x; r < n; r += blockDim.x)
    for (int k = 0; k < 4; ++k) s[k] += part[r * 4 + k];
  float v[4];
  for (int k = 0; k < 4; ++k) v[k] = block_sum((float)s[k], buf) / count[0];
  if (threadIdx.x == 0) {
    stats[0] = v[0] + beta * v[1] - c * v[2];
    for (int k = 0; k < 4; ++k) stats[1 + k] = v[k];
  }
}

}  // namespace qqt

using namespace qqt;

extern "C" uint64_t qqt_policy_loss_work_bytes(int64_t rows) {
  return rows < 0 ? 0 : 16 + (uint64_t)rows * 16;
}

extern "C" int qqt_policy_loss(const QqtPolicyLoss* a, qqt_stream_t stream) {
  if (!a || !dtype_ok(a->dtype) || a->rows < 0 || a->n_heads < 1) return QQT_E_ARG;
  if (a->n_heads > QQT_MAX_HEADS || a->rows > 0x7fffffffll) return QQT_E_LIMIT;
  int64_t v = 0;
  for (int h = 0; h < a->n_heads; ++h) {
    if (a->width[h] < 1) return QQT_E_ARG;
    v += a->width[h];
  }
  if (v > 0x7fffffffll) return QQT_E_LIMIT;
  const bool loss = a->stats || a->dlogits;
  if (loss && !a->work) return QQT_E_ARG;
  if (a->rows > 0 && (!a->logits || !a->actions || (loss && (!a->old_logp || !a->adv))))
    return QQT_E_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  float* count = (float*)a->work;
  float* part = count + 4;
  QqtPolicyLoss args = *a;
  if (!loss) args.old_logp = nullptr;
  if (loss) k_pl_count<<<1, 1024, 0, st>>>(a->mask, a->rows, count);
  if (a->rows > 0)
    with_dtype(a->dtype, [&](auto t) {
      k_pl_rows<decltype(t)><<<(unsigned)a->rows, 256, 0, st>>>(args, count, part);
      return 0;
    });
  if (a->stats)
    k_pl_stats<<<1, 1024, 0, st>>>(part, a->rows, count, a->kl_coef, a->entropy_coef, a->stats);
  return launch_status();
}
