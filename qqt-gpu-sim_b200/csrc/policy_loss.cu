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
//
// By the number of logits V of a row:
//  * up to kPlSmall: a thread per row, rows staged in shared memory so that
//    loads and stores stay contiguous (the policy's 5 + 2 logits);
//  * else a warp or a block per row: one pass keeps a running maximum and the
//    two sums, rescaled when the maximum grows; a second pass, whose reads
//    come from L2, writes the gradient.  Bound by the exponentials (two per
//    logit on the special-function unit, 16 lanes a cycle and SM) and by
//    memory at much the same time; the other arithmetic runs in pairs
//    (f32x2).  A row may begin at any address: vectors are put together from
//    two aligned ones, so the element a thread works on, and with it every
//    sum, does not depend on alignment.

#include "ops_common.cuh"

namespace qqt {

#ifndef PL_W
#define PL_W 256
#endif
constexpr int kPlThreads = 512;      // largest block on a row
constexpr int kPlSmall = 32;         // logits of a row that one thread handles
constexpr int kPlSmallRows = 256;    // rows of such a block
constexpr int kPlCounts = 64;        // blocks that count the mask's rows
constexpr int kPlFold = 8192;        // rows up to which such a block counts them itself
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -1.0e4f;    // z - m below it is as good as minus infinity

struct HeadStat {
  float m, inv_s, log_s, ent;
  int act;                  // the action, -1 where it adds nothing
  float z_act;
};

// Rows of the mask, at least 1; `counts`: the counting blocks' results.
__device__ __forceinline__ float rows_counted(const QqtPolicyLoss& a, const int* counts) {
  if (!a.mask) return fmaxf((float)a.rows, 1.f);
  const int l = lane_id();
  const int n = warp_sum(counts[l] + counts[l + 32]);
  return fmaxf((float)n, 1.f);
}

__device__ __forceinline__ int count_bytes(const uint8_t* mask, int64_t first, int64_t step,
                                           int64_t rows) {
  int n = 0;
  const bool whole = ((uintptr_t)mask & 15) == 0;
  for (int64_t r = first * 16; r < rows; r += step * 16) {
    if (whole && r + 16 <= rows) {
      const uint4 v = *reinterpret_cast<const uint4*>(mask + r);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)      // bytes that are not 0
        n += __popc(__vcmpne4(w[k], 0u) & 0x01010101u);
    } else {
      for (int64_t q = r; q < r + 16 && q < rows; ++q) n += mask[q] != 0;
    }
  }
  return n;
}

__global__ void __launch_bounds__(512) k_pl_count(const uint8_t* __restrict__ mask, int64_t rows,
                                                  int* __restrict__ counts) {
  __shared__ int buf[16];
  int n = count_bytes(mask, (int64_t)blockIdx.x * 512 + threadIdx.x, (int64_t)gridDim.x * 512, rows);
  n = warp_sum(n);
  if (lane_id() == 0) buf[warp_id()] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    for (int k = 0; k < 16; ++k) n += buf[k];
    counts[blockIdx.x] = n;
  }
}

// What a row adds to the sums, and its gradient's coefficient.
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


__device__ __forceinline__ RowLoss loss_of(const QqtPolicyLoss& a, int64_t r, float logp, bool live) {
  if (!live) return RowLoss{0.f, 0.f, 0.f, 0.f};
  return row_loss(logp, a.old_logp[r], a.adv[r], a.ref_logp ? a.ref_logp[r] : 0.f,
                  a.ref_logp != nullptr, a.clip_low, a.clip_high, a.kl_coef);
}

// log p of the head's action from its sums, and what the second pass needs.
__device__ __forceinline__ float finish_head(HeadStat& k, float m, float s, float e, float z_act,
                                             bool act_ok) {
  const bool any = m != -INFINITY;
  k.m = m;
  k.inv_s = any ? 1.f / s : 0.f;
  k.log_s = logf(s);
  k.ent = any ? k.log_s - e * k.inv_s : 0.f;
  k.z_act = z_act;
  return any && act_ok && z_act != -INFINITY ? z_act - m - k.log_s : -INFINITY;
}

// The gradient at a logit t = z - m that is not the action's: with p = e / S,
// scale (p (c (log p + H) - G)); the terms that may cancel are added before
// the scale.  At the action's: scale (G (1 - p) + c p (log p + H)).
struct HeadGrad {
  float c_s, k_s, scale;               // e (c_s t + k_s) scale
};
__device__ __forceinline__ HeadGrad head_grad(const HeadStat& k, float g, float c, float scale) {
  return HeadGrad{c * k.inv_s, (c * (k.ent - k.log_s) - g) * k.inv_s, scale};
}
__device__ __forceinline__ float action_grad(const HeadStat& k, float g, float c, float scale) {
  const float lp = k.z_act - k.m - k.log_s, p = expf(lp);
  return scale * fmaf(g, 1.f - p, p * (c * (lp + k.ent)));
}

// ---------------------------------------------------- few logits: thread per row

template <class T>
__global__ void __launch_bounds__(kPlSmallRows)
    k_pl_small(QqtPolicyLoss a, int V, const int* __restrict__ counts, float* __restrict__ part,
               int one_block) {
  extern __shared__ float zs[];          // [rows][pitch]
  __shared__ float buf[32];
  __shared__ int n_mask;
  const int pitch = V | 1;               // odd: threads on rows hit different banks
  const int64_t r0 = (int64_t)blockIdx.x * kPlSmallRows;
  const int n = a.rows - r0 < kPlSmallRows ? (int)(a.rows - r0) : kPlSmallRows;
  const bool loss = a.old_logp != nullptr;
  const bool fold = loss && a.mask && !counts;
  int mine = 0;
  if (fold) {
    if (threadIdx.x == 0) n_mask = 0;
    mine = warp_sum(count_bytes(a.mask, threadIdx.x, kPlSmallRows, a.rows));
  }
  {
    int row = threadIdx.x / V, col = threadIdx.x % V;
    const int dr = kPlSmallRows / V, dc = kPlSmallRows % V;
#pragma unroll 4
    for (int i = threadIdx.x; i < n * V; i += kPlSmallRows) {
      float z = to_f(((const T*)a.logits)[(r0 + row) * a.row_stride + col]);
      if (a.legal && !a.legal[(r0 + row) * a.legal_stride + col]) z = -INFINITY;
      zs[row * pitch + col] = z;
      row += dr;
      col += dc;
      if (col >= V) {
        col -= V;
        ++row;
      }
    }
  }
  __syncthreads();
  if (fold && lane_id() == 0 && mine) atomicAdd(&n_mask, mine);   // whole numbers: any order
  const bool on = threadIdx.x < n;
  const int64_t r = r0 + threadIdx.x;
  float* z = zs + threadIdx.x * pitch;
  HeadStat hs[QQT_MAX_HEADS];
  float logp = 0.f, ent = 0.f;
  if (on) {
    int at = 0;
#pragma unroll 1
    for (int h = 0; h < a.n_heads; ++h) {
      const int w = a.width[h];
      const int64_t act = a.actions[r * a.action_stride + h];
      const bool in = act >= 0 && act < w;
      if (!in) flag_error(QQT_DEV_BAD_ACTION);
      float m = -INFINITY, s = 0.f, e = 0.f;
      for (int j = 0; j < w; ++j) m = max_nan(m, z[at + j]);
      for (int j = 0; j < w; ++j) {
        const float t = max_nan(z[at + j] - m, kFloor), x = expf(t);
        s += x;
        e = fmaf(x, t, e);
      }
      HeadStat k;
      k.act = in ? at + (int)act : -1;
      logp += finish_head(k, m, s, e, in ? z[at + act] : -INFINITY, in);
      ent += k.ent;
      hs[h] = k;
      at += w;
    }
    if (a.logp) a.logp[r] = logp;
    if (a.entropy) a.entropy[r] = ent;
  }
  if (!loss) return;
  if (fold) __syncthreads();
  const float count = fold ? fmaxf((float)n_mask, 1.f) : rows_counted(a, counts);
  const bool live = on && logp != -INFINITY && (!a.mask || a.mask[r]);
  const RowLoss l = loss_of(a, r, logp, live);
  if (a.stats) {
    const float v[4] = {l.pg, l.kl, live ? ent : 0.f, l.clip};
    float sum[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = block_sum(v[k], buf);
    if (threadIdx.x == 0) {
      if (one_block) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] /= count;
        a.stats[0] = sum[0] + a.kl_coef * sum[1] - a.entropy_coef * sum[2];
#pragma unroll
        for (int k = 0; k < 4; ++k) a.stats[1 + k] = sum[k];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) part[blockIdx.x * 4 + k] = sum[k];
      }
    }
  }
  if (!a.dlogits) return;
  const float scale = a.grad_scale / count * (a.upstream ? a.upstream[0] : 1.f);
  if (on) {
    int at = 0;
#pragma unroll 1
    for (int h = 0; h < a.n_heads; ++h) {
      const int w = a.width[h];
      const HeadStat k = hs[h];
      const HeadGrad q = head_grad(k, l.g, a.entropy_coef, scale);
      for (int j = 0; j < w; ++j) {
        const float t = max_nan(z[at + j] - k.m, kFloor);
        z[at + j] = live ? expf(t) * fmaf(q.c_s, t, q.k_s) * scale : 0.f;
      }
      if (live) z[k.act] = action_grad(k, l.g, a.entropy_coef, scale);
      at += w;
    }
  }
  __syncthreads();
  {
    int row = threadIdx.x / V, col = threadIdx.x % V;
    const int dr = kPlSmallRows / V, dc = kPlSmallRows % V;
#pragma unroll 4
    for (int i = threadIdx.x; i < n * V; i += kPlSmallRows) {
      ((T*)a.dlogits)[(r0 + row) * a.dlogits_stride + col] = from_f<T>(zs[row * pitch + col]);
      row += dr;
      col += dc;
      if (col >= V) {
        col -= V;
        ++row;
      }
    }
  }
}

// ------------------------------------------------- many logits: team per row

// Pairs of floats in one instruction each.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The VEC elements from the s-th (0 < s < VEC) of the 2 VEC of a and b.
template <class T, int VEC>
__device__ __forceinline__ uint4 funnel(uint4 a, uint4 b, int s) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const int words = sizeof(T) == 4 ? s : s >> 1;
  if (words & 2) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (words & 1) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (sizeof(T) == 2) {
    const int bits = (s & 1) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Vector j of the w elements from p, minus infinity past them.  sh: elements
// between p and the 16-byte boundary below it.  Reads no element outside.
template <class T, int VEC>
__device__ __forceinline__ Vec<T, VEC> get_logits(const T* p, int sh, int j, int w) {
  const int i = j * VEC;
  uint4 r;
  if (sh == 0 && i + VEC <= w) {
    r = *reinterpret_cast<const uint4*>(p + i);
  } else if (sh && i >= sh && i - sh + 2 * VEC <= w) {
    const uint4* q = reinterpret_cast<const uint4*>(p + i - sh);
    r = funnel<T, VEC>(q[0], q[1], sh);
  } else {
    float f[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) f[v] = i + v < w ? to_f(p[i + v]) : -INFINITY;
    Vec<T, VEC> x;
    x.put(f);
    return x;
  }
  return *reinterpret_cast<const Vec<T, VEC>*>(&r);
}
// Vectors j, j + step, ...  inner: none of the warp's is at an end of the row.
template <class T, int VEC, int U>
__device__ __forceinline__ void get_chunk(const T* p, int sh, int j, int step, int w, bool inner,
                                          Vec<T, VEC>* c) {
  if (inner && sh == 0) {
    const uint4* q = reinterpret_cast<const uint4*>(p) + j;
#pragma unroll
    for (int u = 0; u < U; ++u, q += step) {
      const uint4 r = *q;
      c[u] = *reinterpret_cast<const Vec<T, VEC>*>(&r);
    }
  } else if (inner) {
    const uint4* q = reinterpret_cast<const uint4*>(p - sh) + j;
    uint4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u, q += step) {
      lo[u] = q[0];
      hi[u] = q[1];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint4 r = funnel<T, VEC>(lo[u], hi[u], sh);
      c[u] = *reinterpret_cast<const Vec<T, VEC>*>(&r);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = get_logits<T, VEC>(p, sh, j + u * step, w);
  }
}

// What is done to a vector before it is taken apart into floats: minus
// infinity in illegal places, the maximum, and a finite floor (so that a
// weight of 0 times z - m is 0).
template <class T, int VEC>
struct Logits;
template <int VEC>
struct Logits<float, VEC> {
  static constexpr bool kSafe = false;   // z - m may be minus infinity
  static constexpr float kBound = 0.f;
  __device__ static __forceinline__ void bar(Vec<float, VEC>& x, const uint32_t* legal4) {
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      if (!((legal4[v / 4] >> (v % 4 * 8)) & 0xff)) x.v[v] = -INFINITY;
  }
  __device__ static __forceinline__ float top(float m, const Vec<float, VEC>& x) {
#pragma unroll
    for (int v = 0; v < VEC; v += 2)
      asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(x.v[v]), "f"(x.v[v + 1]));
    return m;
  }
  __device__ static __forceinline__ void lift(Vec<float, VEC>&) {}
};
template <class T>
struct Half2;
template <>
struct Half2<__half> {
  static constexpr uint32_t kNegInf = 0xfc00fc00u, kLowest = 0xfbfffbffu;
  static constexpr float kBound = 3.0e4f;
  __device__ static __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};
template <>
struct Half2<__nv_bfloat16> {
  static constexpr uint32_t kNegInf = 0xff80ff80u, kLowest = 0xff7fff7fu;
  static constexpr float kBound = 1.0e30f;
  __device__ static __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};
template <class T, int VEC>
struct Logits16 {
  // after lift() z - m is finite, and what was minus infinity still adds 0,
  // while |m| is below kBound
  static constexpr bool kSafe = true;
  static constexpr float kBound = Half2<T>::kBound;
  __device__ static __forceinline__ void bar(Vec<T, VEC>& x, const uint32_t* legal4) {
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) {
      const uint32_t on = __vcmpne4(legal4[k], 0u);      // a byte of ones per legal place
      const uint32_t lo = __byte_perm(on, 0, 0x1100), hi = __byte_perm(on, 0, 0x3322);
      x.w[2 * k] = (x.w[2 * k] & lo) | (Half2<T>::kNegInf & ~lo);
      x.w[2 * k + 1] = (x.w[2 * k + 1] & hi) | (Half2<T>::kNegInf & ~hi);
    }
  }
  __device__ static __forceinline__ float top(float m, const Vec<T, VEC>& x) {
    uint32_t t = x.w[0];
#pragma unroll
    for (int k = 1; k < VEC / 2; ++k) t = Half2<T>::max(t, x.w[k]);
    Vec<T, 2> two;
    two.w[0] = t;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(two.get(0)), "f"(two.get(1)));
    return m;
  }
  __device__ static __forceinline__ void lift(Vec<T, VEC>& x) {
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) x.w[k] = Half2<T>::max(x.w[k], Half2<T>::kLowest);
  }
};
template <int VEC>
struct Logits<__half, VEC> : Logits16<__half, VEC> {};
template <int VEC>
struct Logits<__nv_bfloat16, VEC> : Logits16<__nv_bfloat16, VEC> {};

template <class T, int VEC>
__device__ __forceinline__ void bar_illegal(Vec<T, VEC>& x, const uint8_t* legal, int j, int w) {
  const int i = j * VEC;
  const uint8_t* l = legal + i;
  uint32_t b[VEC / 4];
  if (i + VEC <= w && ((uintptr_t)l & (VEC - 1)) == 0) {
    if constexpr (VEC == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(l);
      b[0] = v.x;
      b[1] = v.y;
    } else {
      b[0] = *reinterpret_cast<const uint32_t*>(l);
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) {
      b[k] = 0;
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (i + 4 * k + v < w && l[4 * k + v]) b[k] |= 0xffu << (8 * v);
    }
  }
  Logits<T, VEC>::bar(x, b);
}

// z - m of a pair of places, as floats of at least kFloor where SAFE is not given.
template <bool SAFE>
__device__ __forceinline__ uint64_t below_top(float z0, float z1, uint64_t nm) {
  const uint64_t t = add2(pair(z0, z1), nm);
  if (SAFE) return t;
  float t0, t1;
  unpair(t, t0, t1);
  return pair(max_nan(t0, kFloor), max_nan(t1, kFloor));
}
__device__ __forceinline__ uint64_t exp2_pair(uint64_t t) {
  float x0, x1;
  unpair(mul2(t, pair(kLog2e, kLog2e)), x0, x1);
  return pair(ex2_approx(x0), ex2_approx(x1));
}
template <class T, int VEC, int U, bool SAFE>
__device__ __forceinline__ void add_exps(const Vec<T, VEC>* c, float m, uint64_t& s2, uint64_t& e2) {
  const uint64_t nm = pair(-m, -m);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int v = 0; v < VEC; v += 2) {
      const uint64_t t = below_top<SAFE>(c[u].get(v), c[u].get(v + 1), nm);
      const uint64_t x = exp2_pair(t);
      s2 = add2(s2, x);
      e2 = fma2(x, t, e2);
    }
}

// Stores vector j of the w elements from p; every lane of the warp calls it,
// and lane l of a team of G has vector j0 + l.  on: the vector exists.  Where p
// is not on a 16-byte boundary each lane stores the aligned word that its
// vector's first elements and the lane below's last ones make up.
template <class T, int VEC, int G>
__device__ __forceinline__ void put_grads(T* p, int sh, int j, int w, bool on, const float* f) {
  Vec<T, VEC> x;
  x.put(f);
  const int i = j * VEC;
  if (sh == 0) {
    if (on && i + VEC <= w) {
      st_vec(p + i, x);
    } else if (on) {
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (i + v < w) p[i + v] = from_f<T>(f[v]);
    }
  }
  // (teams of a warp are on rows of their own alignment)
  if (G == 32 ? sh == 0 : __all_sync(QQT_FULL, sh == 0)) return;
  const int l = lane_id() % G;
  const uint4 own = *reinterpret_cast<const uint4*>(&x);
  uint4 under;
  under.x = __shfl_up_sync(QQT_FULL, own.x, 1);
  under.y = __shfl_up_sync(QQT_FULL, own.y, 1);
  under.z = __shfl_up_sync(QQT_FULL, own.z, 1);
  under.w = __shfl_up_sync(QQT_FULL, own.w, 1);
  const bool over = __shfl_down_sync(QQT_FULL, (int)on, 1) && l < G - 1;
  if (!on || sh == 0) return;
  const int first = VEC - sh;            // elements of this vector in the word it shares
  const bool joined = l > 0 && i + first <= w;
  if (joined) *reinterpret_cast<uint4*>(p + i - sh) = funnel<T, VEC>(under, own, first);
  if (joined && over) return;
  // what no joined word takes: first elements without a lane below, last ones
  // without a lane above ...
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    if (i + v < w && ((v < first && !joined) || (v >= first && !over)))
      p[i + v] = from_f<T>(f[v]);
  // ... and the last ones of the lane below a vector that ends before it can join
  if (l > 0 && !joined) {
    const Vec<T, VEC> b = *reinterpret_cast<const Vec<T, VEC>*>(&under);
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      if (v >= first) p[i - VEC + v] = from_f<T>(b.get(v));
  }
}

template <class T>
__device__ __forceinline__ int misfit(const T* p) {
  return (int)(((uintptr_t)p & 15) / sizeof(T));
}

// Maximum and sums over a team of G lanes, or a block (G = 0).
template <int G>
__device__ __forceinline__ float team_max(float v, float* buf) {
  if (G == 0) return block_max_nan(v, buf);
#pragma unroll
  for (int o = (G ? G : 32) / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(QQT_FULL, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float team_add(float v, float* buf) {
  if (G == 0) return block_sum(v, buf);
#pragma unroll
  for (int o = (G ? G : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(QQT_FULL, v, o);
  return v;
}

template <class T, int G, bool LEGAL>
__global__ void __launch_bounds__(kPlThreads, kPlThreads == 512 ? 2 : 1)
    k_pl_rows(QqtPolicyLoss a, const int* __restrict__ counts, float* __restrict__ part) {
  constexpr int VEC = 16 / sizeof(T), U = 4, LANES = G ? G : 32;
  using L = Logits<T, VEC>;
  __shared__ float buf[32];
  // this thread's first vector, the warp's first, and the step between vectors
  const int tl = G ? lane_id() % LANES : (int)threadIdx.x;
  const int wj = G ? 0 : (int)threadIdx.x - lane_id(), step = G ? G : (int)blockDim.x;
  int64_t r = G ? (int64_t)blockIdx.x * (blockDim.x / LANES) + threadIdx.x / LANES
                : (int64_t)blockIdx.x;
  const bool exists = r < a.rows;
  if (G && !exists) r = a.rows - 1;
  const bool lead = tl == 0 && exists;
  const T* z = (const T*)a.logits + r * a.row_stride;
  const uint8_t* legal = LEGAL ? a.legal + r * a.legal_stride : nullptr;
  HeadStat hs[QQT_MAX_HEADS];
  float logp = 0.f, ent = 0.f;
  int at = 0;
#pragma unroll 1
  for (int h = 0; h < a.n_heads; ++h) {
    const int w = a.width[h], nv = (w + VEC - 1) / VEC;
    const T* p = z + at;
    const int sh = misfit(p);
    float m = -INFINITY;
    uint64_t s2 = pair(0.f, 0.f), e2 = s2;
#pragma unroll 1
    for (int jb = 0; jb + wj < nv; jb += step * U) {
      Vec<T, VEC> c[U];
      const int j = jb + tl;
      const bool inner = jb + wj > 0 && (jb + wj + (U - 1) * step + LANES + 1) * VEC <= w;
      get_chunk<T, VEC, U>(p, sh, j, step, w, inner, c);
      if (LEGAL)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (j + u * step < nv) bar_illegal<T, VEC>(c[u], legal + at, j + u * step, w);
      float mx = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mx = L::top(mx, c[u]);
      if (mx == -INFINITY) continue;       // nothing legal so far
      if (mx != m) {                       // rescale: e^(z - m) (z - m) moves with m too
        const float dm = max_nan(m - mx, kFloor), sc = ex2_approx(dm * kLog2e);
        const uint64_t sc2 = pair(sc, sc);
        e2 = mul2(fma2(pair(dm, dm), s2, e2), sc2);
        s2 = mul2(s2, sc2);
        m = mx;
      }
      if (L::kSafe && fabsf(m) < L::kBound) {
#pragma unroll
        for (int u = 0; u < U; ++u) L::lift(c[u]);
        add_exps<T, VEC, U, L::kSafe>(c, m, s2, e2);
      } else {
        add_exps<T, VEC, U, false>(c, m, s2, e2);
      }
    }
    float s, e, hi;
    unpair(s2, s, hi);
    s += hi;
    unpair(e2, e, hi);
    e += hi;
    const float top = team_max<G>(m, buf);
    const float dm = m == -INFINITY ? kFloor : max_nan(m - top, kFloor);
    const float sc = m == -INFINITY ? 0.f : ex2_approx(dm * kLog2e);
    e = team_add<G>(sc * fmaf(dm, s, e), buf);
    s = team_add<G>(sc * s, buf);
    const int64_t act = a.actions[r * a.action_stride + h];
    const bool in = act >= 0 && act < w;
    if (!in && lead) flag_error(QQT_DEV_BAD_ACTION);
    HeadStat k;
    k.act = in ? (int)act : -1;
    logp += finish_head(k, top, s, e, in && !(LEGAL && !legal[at + act]) ? to_f(p[act]) : -INFINITY,
                        in);
    ent += k.ent;
    hs[h] = k;
    at += w;
  }
  if (lead) {
    if (a.logp) a.logp[r] = logp;
    if (a.entropy) a.entropy[r] = ent;
  }
  if (!a.old_logp) return;
  const bool live = logp != -INFINITY && (!a.mask || a.mask[r]);
  const RowLoss l = loss_of(a, r, logp, live);
  if (a.stats && lead)
    *reinterpret_cast<float4*>(part + r * 4) =
        make_float4(l.pg, l.kl, live ? ent : 0.f, l.clip);
  if (!a.dlogits) return;
  const float scale =
      a.grad_scale / rows_counted(a, counts) * (a.upstream ? a.upstream[0] : 1.f);
  T* dz = (T*)a.dlogits + r * a.dlogits_stride;
  at = 0;
#pragma unroll 1
  for (int h = 0; h < a.n_heads; ++h) {
    const int w = a.width[h], nv = (w + VEC - 1) / VEC;
    const HeadStat k = hs[h];
    const T* p = z + at;
    T* q = dz + at;
    const int sh = misfit(p), qsh = misfit(q);
    const HeadGrad g = head_grad(k, l.g, a.entropy_coef, scale);
    const float ga = live ? action_grad(k, l.g, a.entropy_coef, scale) : 0.f;
    const int ja = k.act >= 0 ? k.act / VEC : -1;
    const bool safe = L::kSafe && fabsf(k.m) < L::kBound;
    const uint64_t nm = pair(-k.m, -k.m), cs = pair(g.c_s, g.c_s), ks = pair(g.k_s, g.k_s),
                   sc = pair(g.scale, g.scale);
    constexpr int U2 = 2;
#pragma unroll 1
    for (int jb = 0; jb + wj < nv; jb += step * U2) {
      Vec<T, VEC> c[U2];
      const int j0 = jb + tl;
      const bool inner = jb + wj > 0 && (jb + wj + (U2 - 1) * step + LANES + 1) * VEC <= w;
      if (live) get_chunk<T, VEC, U2>(p, sh, j0, step, w, inner, c);
#pragma unroll
      for (int u = 0; u < U2; ++u) {
        const int j = j0 + u * step;
        float f[VEC];
        if (live) {
          if (LEGAL && j < nv) bar_illegal<T, VEC>(c[u], legal + at, j, w);
          if (safe) L::lift(c[u]);
#pragma unroll
          for (int v = 0; v < VEC; v += 2) {
            const float z0 = c[u].get(v), z1 = c[u].get(v + 1);
            const uint64_t t = safe ? below_top<L::kSafe>(z0, z1, nm) : below_top<false>(z0, z1, nm);
            unpair(mul2(mul2(exp2_pair(t), fma2(cs, t, ks)), sc), f[v], f[v + 1]);
          }
          if (j == ja) {
#pragma unroll
            for (int v = 0; v < VEC; ++v)
              if (j * VEC + v == k.act) f[v] = ga;
          }
        } else {
#pragma unroll
          for (int v = 0; v < VEC; ++v) f[v] = 0.f;
        }
        put_grads<T, VEC, LANES>(q, qsh, j, w, j < nv && exists, f);
      }
    }
    at += w;
  }
}

// Means over the counted rows from n partial sums, in a fixed order.
__global__ void __launch_bounds__(1024)
    k_pl_stats(QqtPolicyLoss a, const float* __restrict__ part, int64_t n,
               const int* __restrict__ counts) {
  __shared__ float buf[32];
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < n; r += 1024) {
    const float4 v = *reinterpret_cast<const float4*>(part + r * 4);
    s[0] += v.x;
    s[1] += v.y;
    s[2] += v.z;
    s[3] += v.w;
  }
  const float count = rows_counted(a, counts);
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = block_sum(s[k], buf) / count;
  if (threadIdx.x == 0) {
    a.stats[0] = s[0] + a.kl_coef * s[1] - a.entropy_coef * s[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) a.stats[1 + k] = s[k];
  }
}

}  // namespace qqt

using namespace qqt;

// 64 counts, then four partial sums a row (or a block of rows).
extern "C" uint64_t qqt_policy_loss_work_bytes(int64_t rows) {
  return rows < 0 ? 0 : kPlCounts * 4 + (uint64_t)rows * 16;
}

extern "C" int qqt_policy_loss(const QqtPolicyLoss* a, qqt_stream_t stream) {
  if (!a || !dtype_ok(a->dtype) || a->rows < 0 || a->n_heads < 1) return QQT_E_ARG;
  if (a->n_heads > QQT_MAX_HEADS || a->rows > 0x7fffffffll) return QQT_E_LIMIT;
  int64_t v = 0;
  for (int h = 0; h < a->n_heads; ++h) {
    if (a->width[h] < 1) return QQT_E_ARG;
    v += a->width[h];
  }
  if (v > 0x3fffffffll) return QQT_E_LIMIT;
  const bool loss = a->stats || a->dlogits;
  if (loss && !a->work) return QQT_E_ARG;
  if (a->rows > 0 && (!a->logits || !a->actions || (loss && (!a->old_logp || !a->adv))))
    return QQT_E_ARG;
  if (!aligned_to(a->work, 16)) return QQT_E_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  QqtPolicyLoss args = *a;
  if (!loss) args.old_logp = nullptr;
  const bool small = v <= kPlSmall;
  const int64_t blocks = (a->rows + kPlSmallRows - 1) / kPlSmallRows;
  const bool one = small && blocks == 1;
  int* counts = (int*)a->work;
  float* part = loss ? (float*)(counts + kPlCounts) : nullptr;
  if (loss && a->mask && !(small && a->rows <= kPlFold && blocks > 0 && (one || !a->stats)))
    k_pl_count<<<kPlCounts, 512, 0, st>>>(a->mask, a->rows, counts);
  else
    counts = nullptr;
  if (a->rows > 0)
    with_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      if (small) {
        const size_t smem = (size_t)kPlSmallRows * (v | 1) * 4;
        k_pl_small<T><<<(unsigned)blocks, kPlSmallRows, smem, st>>>(args, (int)v, counts, part, one);
        return 0;
      }
      // a team of 8 lanes holds rows of up to 32 vectors in one step, a warp
      // rows of up to 256 in two, blocks the rest: 256 threads, 512 where a
      // row is so long that the blocks of all SMs would read past L2
      const int64_t bytes = v * (int64_t)sizeof(T);
      const int g = bytes <= 32 * 16 ? 8 : bytes <= PL_W * 16 ? 32 : 0;
      const int threads = g || bytes <= 128 * 1024 ? 256 : kPlThreads;
      const int per = g ? threads / g : 1;
      const unsigned n = (unsigned)((a->rows + per - 1) / per);
      auto run = [&](auto gg) {
        constexpr int G = decltype(gg)::value;
        if (a->legal)
          k_pl_rows<T, G, true><<<n, threads, 0, st>>>(args, counts, part);
        else
          k_pl_rows<T, G, false><<<n, threads, 0, st>>>(args, counts, part);
      };
      if (g == 8)
        run(std::integral_constant<int, 8>{});
      else if (g == 32)
        run(std::integral_constant<int, 32>{});
      else
        run(std::integral_constant<int, 0>{});
      return 0;
    });
  if (a->stats && !one)
    k_pl_stats<<<1, 1024, 0, st>>>(args, part, small ? blocks : a->rows, counts);
  return launch_status();
}
