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
//  * else 8 lanes, a warp or a block per row: one pass keeps a running maximum
//    and the two sums, rescaled when the maximum grows; a second pass, whose
//    reads come from L2, writes the gradient.  Bound by the exponentials (two
//    per logit on the special-function unit, 16 lanes a cycle and SM) and by
//    memory at much the same time; the other arithmetic runs in pairs
//    (f32x2).  A row may begin at any address: vectors are put together from
//    two aligned ones, so the element a thread works on, and with it every
//    sum, does not depend on alignment.
//
// Measured on a B200 (copy bandwidth 6.55 TB/s):
//   8192 x 32000 bf16     loss and gradient 225 us, 4.7 TB/s (two values a
//                         logit); scores 113 us, 4.6 TB/s
//   2047 x 100003 f16     loss and gradient 290 us, 2.8 TB/s; scores 107 us, 3.8
//                         TB/s (rows at any alignment)
//   4096 x 32000 f32      loss and gradient 209 us, 5.0 TB/s; scores 101 us, 5.2
//   1048576 x 64 f32      loss and gradient 441 us, 163 of them k_pl_stats, one
//                         block that adds a partial sum per row; scores 134 us
//   1048576 rows of 5 + 2 f32 logits, masked: 39 us, 2.6 TB/s; 86 % of the
//                         issue slots (900 instructions a row: logarithms,
//                         exponentials and quotients of both heads and of the
//                         loss)
// The vocabulary rows execute about 9 instructions a logit and pass, 64 % of
// the issue slots, 57 % of the special-function unit and 70 % of the memory
// bandwidth at once; no one of them is full.

#include "ops_common.cuh"

namespace qqt {

constexpr int kPlThreads = 512;      // largest block on a row
constexpr int kPlSmall = 32;         // logits of a row that one thread handles
constexpr int kPlSmallRows = 256;    // rows of such a block
constexpr int kPlCounts = 64;        // blocks that count the mask's rows
constexpr int kPlFold = 8192;        // rows up to which such a block counts them itself
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -1.0e4f;    // z - m below it is as good as minus infinity
constexpr float kRefMost = 1048576.f;   // largest |maximum| that the one-step exponents take

// A head's sums: log p = t - log_s and p = e^t inv_s for t = z less the
// reference that they were taken against.
struct HeadStat {
  float inv_s, log_s, ent;
  float t_act;              // the action's t
  int act;                  // the action, -1 where it is none of the head's
};

// Rows of the mask, at least 1; `counts`: the counting blocks' results.
__device__ __forceinline__ float rows_counted(const QqtPolicyLoss& a, const int* counts) {
  if (!a.mask) return fmaxf((float)a.rows, 1.f);
  const int l = lane_id();
  const int n = __reduce_add_sync(QQT_FULL, counts[l] + counts[l + 32]);
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
  let_next_start();
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
  // (an advantage of 0 weighs any ratio away, one beyond float32 too)
  const float u = a == 0.f && r == INFINITY ? 0.f : r * a, v = rc * a;
  o.pg = -(u != u ? u : fminf(u, v));
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


struct RowIn {
  float old, adv, ref;
  bool counts;
};
__device__ __forceinline__ RowLoss loss_of(const QqtPolicyLoss& a, const RowIn& in, float logp,
                                           bool live) {
  if (!live) return RowLoss{0.f, 0.f, 0.f, 0.f};
  return row_loss(logp, in.old, in.adv, in.ref, a.ref_logp != nullptr, a.clip_low, a.clip_high,
                  a.kl_coef);
}

// log p of the head's action.  any: some category is legal.
__device__ __forceinline__ float finish_head(HeadStat& k, bool any, float s, float log_s, float e,
                                             float t_act, bool act_ok) {
  k.inv_s = any ? rcp_approx(s) : 0.f;      // s >= 1 or NaN
  k.log_s = log_s;
  k.ent = any ? log_s - e * k.inv_s : 0.f;
  k.t_act = t_act;
  return any && act_ok ? t_act - log_s : -INFINITY;
}

// The heads' sum, in which a head without a value (-inf) stays: added to
// another's NaN it would be NaN, and the row would count as live.
__device__ __forceinline__ float add_logp(float sum, float head) {
  return sum == -INFINITY || head == -INFINITY ? -INFINITY : sum + head;
}

// The gradient at a logit that is not the action's, with p = e / S:
// scale (p (c (log p + H) - G)) = scale e (c_s t + k_s); the terms that may
// cancel are added before the scale.  At the action's:
// scale (G (1 - p) + c p (log p + H)).
__device__ __forceinline__ float head_c(const HeadStat& k, float c) { return c * k.inv_s; }
__device__ __forceinline__ float head_k(const HeadStat& k, float g, float c) {
  return (c * (k.ent - k.log_s) - g) * k.inv_s;
}
__device__ __forceinline__ float action_grad(const HeadStat& k, float g, float c, float scale) {
  const float lp = k.t_act - k.log_s, p = expf(lp);
  return scale * fmaf(g, 1.f - p, c * (p * (lp + k.ent)));   // (p = 0 first: c lp may overflow)
}

// ---------------------------------------------------- few logits: thread per row

// Copies n elements from p to floats, minus infinity where legal (optional) is
// 0, or floats to p, by 16-byte vectors; p and legal on 16 bytes.  Rows of V
// elements are V floats apart, V + 1 where 4 divides V; a vector then lies in
// one row.
template <class T>
__device__ __forceinline__ bool run_fits(int V) {
  return (V & 3) != 0 || V % (16 / (int)sizeof(T)) == 0;
}
template <class T>
__device__ __forceinline__ void stage_in(const T* p, const uint8_t* legal, int n, int V, float* to) {
  constexpr int VEC = 16 / sizeof(T);
  const bool padded = (V & 3) == 0;
  for (int i = threadIdx.x * VEC; i + VEC <= n; i += kPlSmallRows * VEC) {
    const Vec<T, VEC> x = ld_vec<T, VEC>(p + i);
    float f[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) f[v] = x.get(v);
    if (legal) {
#pragma unroll
      for (int v = 0; v < VEC; v += 4) {
        const uchar4 l = *reinterpret_cast<const uchar4*>(legal + i + v);
        f[v] = l.x ? f[v] : -INFINITY;
        f[v + 1] = l.y ? f[v + 1] : -INFINITY;
        f[v + 2] = l.z ? f[v + 2] : -INFINITY;
        f[v + 3] = l.w ? f[v + 3] : -INFINITY;
      }
    }
    if (padded) {
      float* q = to + i + i / V;
#pragma unroll
      for (int v = 0; v < VEC; ++v) q[v] = f[v];
    } else {
#pragma unroll
      for (int v = 0; v < VEC; v += 4)
        *reinterpret_cast<float4*>(to + i + v) = make_float4(f[v], f[v + 1], f[v + 2], f[v + 3]);
    }
  }
  const int i = n / VEC * VEC + threadIdx.x;      // (none where a vector lies in one row)
  if (i < n) to[i] = legal && !legal[i] ? -INFINITY : to_f(p[i]);
}
template <class T>
__device__ __forceinline__ void stage_out(T* p, int n, int V, const float* from) {
  constexpr int VEC = 16 / sizeof(T);
  const bool padded = (V & 3) == 0;
  for (int i = threadIdx.x * VEC; i + VEC <= n; i += kPlSmallRows * VEC) {
    float f[VEC];
    if (padded) {
      const float* q = from + i + i / V;
#pragma unroll
      for (int v = 0; v < VEC; ++v) f[v] = q[v];
    } else {
#pragma unroll
      for (int v = 0; v < VEC; v += 4)
        *reinterpret_cast<float4*>(f + v) = *reinterpret_cast<const float4*>(from + i + v);
    }
    Vec<T, VEC> x;
    x.put(f);
    st_vec(p + i, x);
  }
  const int i = n / VEC * VEC + threadIdx.x;
  if (i < n) p[i] = from_f<T>(from[i]);
}

// The warp's sums of v[0] .. v[3], of v[l & 3] in lane l: two exchanges leave
// a value a lane, three more add the lanes that hold the same one.
__device__ __forceinline__ float warp_sum4(const float* v) {
  const int l = lane_id();
  const bool odd = l & 1, hi = l & 2;
  const float a = (odd ? v[1] : v[0]) + __shfl_xor_sync(QQT_FULL, odd ? v[0] : v[1], 1);
  const float b = (odd ? v[3] : v[2]) + __shfl_xor_sync(QQT_FULL, odd ? v[2] : v[3], 1);
  float x = (hi ? b : a) + __shfl_xor_sync(QQT_FULL, hi ? a : b, 2);
#pragma unroll
  for (int o = 4; o < 32; o *= 2) x += __shfl_xor_sync(QQT_FULL, x, o);
  return x;
}

// Rows are V floats apart in shared memory, V + 1 where 4 divides V: at most
// two threads on rows hit the same bank.  Where the rows lie one after the
// other, the block's rows are one run of memory; it is copied by vectors, as it
// is or, where 4 divides V, each vector to its row (1048576 rows of 6: 31 us,
// 46 by elements).  Bound by the issue of instructions, so eight blocks an SM
// and 32 registers are better than six and 40 (36.4 against 39.5 us for rows
// of 5 + 2).
// NH: the number of heads where it is 1 or 2 (what is kept per head then stays
// in registers), QQT_MAX_HEADS for any.
template <class T, int NH>
__global__ void __launch_bounds__(kPlSmallRows, 8)
    k_pl_small(QqtPolicyLoss a, int V, const int* __restrict__ counts, float* __restrict__ part,
               int one_block) {
  extern __shared__ __align__(16) float zs[];
  __shared__ float buf[4][32];
  __shared__ int n_mask;
  const int pitch = V & 3 ? V : V + 1;
  const int64_t r0 = (int64_t)blockIdx.x * kPlSmallRows;
  const int n = a.rows - r0 < kPlSmallRows ? (int)(a.rows - r0) : kPlSmallRows;
  const bool loss = a.old_logp != nullptr;
  const bool fold = loss && a.mask && !counts;
  const bool on = threadIdx.x < n;
  const int64_t r = r0 + threadIdx.x;
  RowIn row{0.f, 0.f, 0.f, true};
  if (loss && on) {
    row.old = a.old_logp[r];
    row.adv = a.adv[r];
    if (a.ref_logp) row.ref = a.ref_logp[r];
    if (a.mask) row.counts = a.mask[r] != 0;
  }
  int mine = 0;
  if (fold) {
    if (threadIdx.x == 0) n_mask = 0;
    mine = warp_sum(count_bytes(a.mask, threadIdx.x, kPlSmallRows, a.rows));
  }
  const T* zp = (const T*)a.logits + r0 * a.row_stride;
  const uint8_t* lp = a.legal ? a.legal + r0 * a.legal_stride : nullptr;
  if (a.row_stride == V && (!lp || a.legal_stride == V) && run_fits<T>(V) &&
      (((uintptr_t)zp | (uintptr_t)lp) & 15) == 0) {
    stage_in(zp, lp, n * V, V, zs);
  } else {
    int q = threadIdx.x / V, col = threadIdx.x % V;
    const int dr = kPlSmallRows / V, dc = kPlSmallRows % V;
#pragma unroll 4
    for (int i = threadIdx.x; i < n * V; i += kPlSmallRows) {
      zs[q * pitch + col] = lp && !lp[q * a.legal_stride + col]
                                ? -INFINITY
                                : to_f(zp[q * a.row_stride + col]);
      q += dr;
      col += dc;
      if (col >= V) {
        col -= V;
        ++q;
      }
    }
  }
  __syncthreads();
  if (fold && lane_id() == 0 && mine) atomicAdd(&n_mask, mine);   // whole numbers: any order
  float* z = zs + threadIdx.x * pitch;
  HeadStat hs[NH];
  float ms[NH];
  float logp = 0.f, ent = 0.f;
  if (on) {
    int at = 0;
#pragma unroll(NH <= 2 ? NH : 1)
    for (int h = 0; h < (NH <= 2 ? NH : a.n_heads); ++h) {
      const int w = a.width[h];
      const int64_t act = a.actions[r * a.action_stride + h];
      const bool in = act >= 0 && act < w;
      if (!in && row.counts) flag_error(QQT_DEV_BAD_ACTION);
      float m = -INFINITY, s = 0.f, e = 0.f;
#pragma unroll 4
      for (int j = at; j < at + w; ++j) m = max_nan(m, z[j]);
#pragma unroll 4
      for (int j = at; j < at + w; ++j) {
        const float t = max_nan(z[j] - m, kFloor), x = ex2_approx(t * kLog2e);
        s += x;
        e = fmaf(x, t, e);
      }
      HeadStat k;
      k.act = in ? at + (int)act : -1;
      const float za = in ? z[at + act] : -INFINITY;
      const float lh = finish_head(k, m != -INFINITY, s, logf(s), e, za - m, za != -INFINITY);
      logp = add_logp(logp, lh);
      k.t_act = za == -INFINITY ? 0.f : za - m;
      ms[h] = m;
      ent += k.ent;
      hs[h] = k;
      at += w;
    }
    if (a.logp) a.logp[r] = logp;
    if (a.entropy) a.entropy[r] = ent;
  }
  if (!loss) return;
  if (fold) __syncthreads();
  before_me_done();
  const float count = fold ? fmaxf((float)n_mask, 1.f) : rows_counted(a, counts);
  const bool live = on && logp != -INFINITY && row.counts;
  const RowLoss l = loss_of(a, row, logp, live);
  if (a.stats) {
    const float v[4] = {l.pg, l.kl, live ? ent : 0.f, l.clip};
    const float x = warp_sum4(v);
    if (lane_id() < 4) buf[lane_id()][warp_id()] = x;
    __syncthreads();
    if (warp_id() == 0) {
      float sum[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        sum[k] = warp_sum_f(lane_id() < kPlSmallRows / 32 ? buf[k][lane_id()] : 0.f);
      if (lane_id() == 0) {
        if (one_block) {
#pragma unroll
          for (int k = 0; k < 4; ++k) sum[k] /= count;
          a.stats[0] = sum[0] + a.kl_coef * sum[1] - a.entropy_coef * sum[2];
#pragma unroll
          for (int k = 0; k < 4; ++k) a.stats[1 + k] = sum[k];
        } else {
          *reinterpret_cast<float4*>(part + (int64_t)blockIdx.x * 4) =
              make_float4(sum[0], sum[1], sum[2], sum[3]);
        }
      }
    }
  }
  if (!a.dlogits) return;
  const float scale = a.grad_scale / count * (a.upstream ? a.upstream[0] : 1.f);
  if (on) {
    int at = 0;
#pragma unroll(NH <= 2 ? NH : 1)
    for (int h = 0; h < (NH <= 2 ? NH : a.n_heads); ++h) {
      const int w = a.width[h];
      const HeadStat k = hs[h];
      const float m = ms[h], cs = head_c(k, a.entropy_coef), ks = head_k(k, l.g, a.entropy_coef);
#pragma unroll 4
      for (int j = at; j < at + w; ++j) {
        const float t = max_nan(z[j] - m, kFloor);
        z[j] = live ? ex2_approx(t * kLog2e) * fmaf(cs, t, ks) * scale : 0.f;
      }
      if (live && k.act >= 0) z[k.act] = action_grad(k, l.g, a.entropy_coef, scale);
      at += w;
    }
  }
  __syncthreads();
  T* op = (T*)a.dlogits + r0 * a.dlogits_stride;
  if (a.dlogits_stride == V && run_fits<T>(V) && ((uintptr_t)op & 15) == 0) {
    stage_out(op, n * V, V, zs);
  } else {
    int q = threadIdx.x / V, col = threadIdx.x % V;
    const int dr = kPlSmallRows / V, dc = kPlSmallRows % V;
#pragma unroll 4
    for (int i = threadIdx.x; i < n * V; i += kPlSmallRows) {
      op[q * a.dlogits_stride + col] = from_f<T>(zs[q * pitch + col]);
      q += dr;
      col += dc;
      if (col >= V) {
        col -= V;
        ++q;
      }
    }
  }
}

// ------------------------------------------------- many logits: team per row

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

// Vectors j, j + step, ... of the w elements from p, minus infinity past them.
// sh: elements between p and the 16-byte boundary below it.  inner: none of
// the warp's vectors is at an end of the row.  Else all whole words are asked
// for before the ends are seen to, which go element by element; nothing
// outside the row is read.
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
    return;
  }
  if (inner) {
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
    return;
  }
  const int i0 = j * VEC, di = step * VEC;
  bool ok[U];
  if (sh == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ok[u] = i0 + u * di + VEC <= w;
      uint4 r = make_uint4(0, 0, 0, 0);
      if (ok[u]) r = *reinterpret_cast<const uint4*>(p + (i0 + u * di));
      c[u] = *reinterpret_cast<const Vec<T, VEC>*>(&r);
    }
  } else {
    uint4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * di - sh;
      ok[u] = i >= 0 && i + 2 * VEC <= w;
      lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
      if (ok[u]) {
        const uint4* q = reinterpret_cast<const uint4*>(p + i);
        lo[u] = q[0];
        hi[u] = q[1];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint4 r = funnel<T, VEC>(lo[u], hi[u], sh);
      c[u] = *reinterpret_cast<const Vec<T, VEC>*>(&r);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!ok[u]) {
      const int i = i0 + u * di;
      float f[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) f[v] = -INFINITY;
      if (i < w) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          if (i + v < w) f[v] = to_f(p[i + v]);
      }
      c[u].put(f);
    }
  }
}

// What is done to a vector before it is taken apart into floats: minus
// infinity in illegal places, the maximum, and a finite floor whose e^t is 0
// beside any maximum above -kLow (a weight of 0 times t is then 0).
template <class T, int VEC>
struct Logits;
template <int VEC>
struct Logits<float, VEC> {
  static constexpr float kLow = 1048576.f;
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
  __device__ static __forceinline__ void lift(Vec<float, VEC>& x) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) x.v[v] = max_nan(x.v[v], -1.0e30f);
  }
};
template <class T>
struct Half2;
template <>
struct Half2<__half> {
  static constexpr uint32_t kNegInf = 0xfc00fc00u, kFloor = 0xfbfffbffu;   // -65504
  static constexpr float kLow = 3.0e4f;
  __device__ static __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};
template <>
struct Half2<__nv_bfloat16> {
  static constexpr uint32_t kNegInf = 0xff80ff80u, kFloor = 0xf149f149u;   // about -1e30
  static constexpr float kLow = 1048576.f;
  __device__ static __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
};
template <class T, int VEC>
struct Logits16 {
  static constexpr float kLow = Half2<T>::kLow;
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
    for (int k = 0; k < VEC / 2; ++k) x.w[k] = Half2<T>::max(x.w[k], Half2<T>::kFloor);
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

// Exponents are taken in base 2 against a whole number r near the maximum:
// t = z log2 e - r in one fused step, r without a rounding of its own, and a
// change of r scales the sums by an exact power of 2.
template <class L>
__device__ __forceinline__ float whole_ref(float m) {
  return rintf(fminf(fmaxf(m, -L::kLow), kRefMost) * kLog2e);
}
__device__ __forceinline__ f32x2 exp2_pair(f32x2 t) {
  return pair(ex2_approx(t.x), ex2_approx(t.y));
}
template <class T, int VEC>
__device__ __forceinline__ void add_exps(const Vec<T, VEC>& c, float ref, f32x2& s2, f32x2& e2) {
  const f32x2 nr = pair(-ref, -ref), l2 = pair(kLog2e, kLog2e);
#pragma unroll
  for (int v = 0; v < VEC; v += 2) {
    const f32x2 t = fma2(pair(c.get(v), c.get(v + 1)), l2, nr);
    const f32x2 x = exp2_pair(t);
    s2 = add2(s2, x);
    e2 = fma2(x, t, e2);
  }
}

// Stores vector j of the w elements from p; every lane of the warp calls it,
// and lane l of a team of G has vector j0 + l.  on: the vector exists.  Where p
// is not on a 16-byte boundary each lane stores the aligned word that its
// vector's first elements and the lane below's last ones make up.
template <class T, int VEC, int G>
__device__ __forceinline__ void put_grads(T* p, int sh, int j, int w, bool on,
                                          const Vec<T, VEC>& x) {
  const int i = j * VEC;
  if (sh == 0) {
    if (on && i + VEC <= w) {
      st_vec(p + i, x);
    } else if (on) {
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (i + v < w) p[i + v] = from_f<T>(x.get(v));
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
      p[i + v] = from_f<T>(x.get(v));
  // ... and the last ones of the lane below a vector that ends before it can join
  if (l > 0 && !joined) {
    const Vec<T, VEC> b = *reinterpret_cast<const Vec<T, VEC>*>(&under);
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      if (v >= first) p[i - VEC + v] = from_f<T>(b.get(v));
  }
}

// The same where all of the warp's vectors lie whole in the row and sh > 0.  The
// first lane's part of the word it shares goes out in pieces of 2, 4 and 8
// bytes, and so does the last lane's (2047 x 100003 f16: 290 us, 340 value by
// value).
template <class T, int VEC>
__device__ __forceinline__ void put_inner(T* p, int sh, int j, const Vec<T, VEC>& x) {
  const int l = lane_id(), first = VEC - sh, b = sh * (int)sizeof(T);
  const uint4 own = *reinterpret_cast<const uint4*>(&x);
  uint4 under;
  under.x = __shfl_up_sync(QQT_FULL, own.x, 1);
  under.y = __shfl_up_sync(QQT_FULL, own.y, 1);
  under.z = __shfl_up_sync(QQT_FULL, own.z, 1);
  under.w = __shfl_up_sync(QQT_FULL, own.w, 1);
  char* to = reinterpret_cast<char*>(p + (int64_t)j * VEC - sh);
  const uint4 word = funnel<T, VEC>(under, own, first);
  if (l > 0) {
    *reinterpret_cast<uint4*>(to) = word;
  } else {                               // bytes b to 15 of the word
    if (b & 2)
      *reinterpret_cast<uint16_t*>(to + b) =
          (uint16_t)((b < 4 ? word.x : b < 8 ? word.y : b < 12 ? word.z : word.w) >> 16);
    const int q = (b + 3) & ~3;
    if (q & 4) *reinterpret_cast<uint32_t*>(to + q) = q == 4 ? word.y : word.w;
    if (q <= 8) *reinterpret_cast<uint2*>(to + 8) = make_uint2(word.z, word.w);
  }
  if (l == 31) {                         // bytes 0 to b - 1 of the next word
    const uint4 rest = funnel<T, VEC>(own, own, first);
    if (b & 8) *reinterpret_cast<uint2*>(to + 16) = make_uint2(rest.x, rest.y);
    if (b & 4) *reinterpret_cast<uint32_t*>(to + 16 + (b & 8)) = b & 8 ? rest.z : rest.x;
    if (b & 2)
      *reinterpret_cast<uint16_t*>(to + 16 + (b & 12)) =
          (uint16_t)((b & 12) == 0 ? rest.x : (b & 12) == 4 ? rest.y : (b & 12) == 8 ? rest.z : rest.w);
  }
}

template <class T>
__device__ __forceinline__ int misfit(const T* p) {
  return (int)(((uintptr_t)p & 15) / sizeof(T));
}

// Joins maximum, reference and sums over a team of G lanes, or a block (G =
// 0): each side's sums are brought to the largest reference.
struct Sums {
  float m, r, s, e;
};
__device__ __forceinline__ void move_ref(Sums& q, float r) {
  const float d = q.r - r, sc = ex2_approx(d);
  q.e = sc * fmaf(d, q.s, q.e);
  q.s = sc * q.s;
  q.r = r;
}
template <int G>
__device__ __forceinline__ void join_lanes(Sums& q) {
  float r = q.r;
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    q.m = max_nan(q.m, __shfl_xor_sync(QQT_FULL, q.m, o));
    r = fmaxf(r, __shfl_xor_sync(QQT_FULL, r, o));
  }
  move_ref(q, r);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    q.s += __shfl_xor_sync(QQT_FULL, q.s, o);
    q.e += __shfl_xor_sync(QQT_FULL, q.e, o);
  }
}
template <int G>
__device__ __forceinline__ void join(Sums& q, float4* buf) {
  join_lanes<G ? G : 32>(q);
  if (G == 0) {
    const int l = lane_id(), nw = blockDim.x >> 5;
    if (l == 0) buf[warp_id()] = make_float4(q.m, q.r, q.s, q.e);
    __syncthreads();
    const bool one = l % 16 < nw;          // (both halves of the warp do the same)
    const float4 v = buf[one ? l % 16 : 0];
    q = Sums{v.x, v.y, one ? v.z : 0.f, one ? v.w : 0.f};
    join_lanes<16>(q);
  }
}

// The same sums against the maximum itself, element by element: for maxima
// that the one-step exponents do not take, NaN among them.
template <class T>
__device__ __forceinline__ float plain_t(const T* p, const uint8_t* legal, int i, float m) {
  const float z = legal && !legal[i] ? -INFINITY : to_f(p[i]);
  return max_nan(z - m, kFloor);
}
template <class T, int G>
__device__ __noinline__ void plain_sums(const T* p, const uint8_t* legal, int w, int tl, int step,
                                        Sums& q, float* buf) {
  float s = 0.f, e = 0.f;
  for (int i = tl; i < w; i += step) {
    const float t = plain_t(p, legal, i, q.m), x = expf(t);
    s += x;
    e = fmaf(x, t, e);
  }
#pragma unroll
  for (int o = (G ? G : 32) / 2; o > 0; o >>= 1) {
    s += __shfl_xor_sync(QQT_FULL, s, o);
    e += __shfl_xor_sync(QQT_FULL, e, o);
  }
  if (G == 0) {
    s = block_sum(lane_id() == 0 ? s : 0.f, buf);
    e = block_sum(lane_id() == 0 ? e : 0.f, buf);
  }
  q.s = s;
  q.e = e;
}

template <class T, int G, bool LEGAL>
__global__ void __launch_bounds__(kPlThreads, kPlThreads == 512 ? 2 : 1)
    k_pl_rows(QqtPolicyLoss a, const int* __restrict__ counts, float* __restrict__ part) {
  constexpr int VEC = 16 / sizeof(T), U = 4, LANES = G ? G : 32;
  using L = Logits<T, VEC>;
  __shared__ float4 buf[2][16];          // two heads in turn
  __shared__ float plain_buf[32];
  // this thread's first vector, the warp's first, and the step between vectors
  const int tl = G ? lane_id() % LANES : (int)threadIdx.x;
  const int wj = G ? 0 : (int)threadIdx.x - lane_id(), step = G ? G : (int)blockDim.x;
  int64_t r = G ? (int64_t)blockIdx.x * (blockDim.x / LANES) + threadIdx.x / LANES
                : (int64_t)blockIdx.x;
  const bool exists = r < a.rows;
  if (G && !exists) r = a.rows - 1;
  const bool lead = tl == 0 && exists;
  // what the row's end needs is asked for at its start
  RowIn in{0.f, 0.f, 0.f, true};
  int n_counted = 0;
  if (a.old_logp) {
    before_me_done();
    if (a.mask) n_counted = counts[lane_id()] + counts[lane_id() + 32];
    in.old = a.old_logp[r];
    in.adv = a.adv[r];
    if (a.ref_logp) in.ref = a.ref_logp[r];
    if (a.mask) in.counts = a.mask[r] != 0;
  }
  const T* z = (const T*)a.logits + r * a.row_stride;
  const uint8_t* legal = LEGAL ? a.legal + r * a.legal_stride : nullptr;
  HeadStat hs[QQT_MAX_HEADS];
  float refs[QQT_MAX_HEADS];
  unsigned plain = 0;                    // heads whose sums are against the maximum itself
  float logp = 0.f, ent = 0.f;
  int at = 0;
#pragma unroll 1
  for (int h = 0; h < a.n_heads; ++h) {
    const int w = a.width[h], nv = (w + VEC - 1) / VEC;
    const T* p = z + at;
    const uint8_t* lg = LEGAL ? legal + at : nullptr;
    const int sh = misfit(p);
    const int64_t act = a.actions[r * a.action_stride + h];
    const bool in_head = act >= 0 && act < w;
    const float z_act = in_head && !(LEGAL && !lg[act]) ? to_f(p[act]) : -INFINITY;
    Sums q{-INFINITY, whole_ref<L>(-INFINITY), 0.f, 0.f};
    f32x2 s2 = pair(0.f, 0.f), e2 = s2;
#pragma unroll 1
    for (int jb = 0; jb + wj < nv; jb += step * U) {
      Vec<T, VEC> c[U];
      const int j = jb + tl;
      const bool inner = (sh == 0 || jb + wj > 0) &&
                         (jb + wj + (U - 1) * step + LANES + (sh ? 1 : 0)) * VEC <= w;
      get_chunk<T, VEC, U>(p, sh, j, step, w, G == 8 ? false : inner, c);
      if (LEGAL)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (j + u * step < nv) bar_illegal<T, VEC>(c[u], lg, j + u * step, w);
      float m = q.m;
#pragma unroll
      for (int u = 0; u < U; ++u) m = L::top(m, c[u]);
      if (!(m <= q.m)) {
        q.m = m;
        const float ref = fmaxf(q.r, whole_ref<L>(m));
        const float d = q.r - ref, sc = ex2_approx(d);
        e2 = mul2(fma2(pair(d, d), s2, e2), pair(sc, sc));
        s2 = mul2(s2, pair(sc, sc));
        q.r = ref;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        L::lift(c[u]);
        add_exps<T, VEC>(c[u], q.r, s2, e2);
      }
    }
    q.s = s2.x + s2.y;
    q.e = e2.x + e2.y;
    join<G>(q, buf[h & 1]);
    const bool any = q.m != -INFINITY;
    const bool one_step = q.m >= -L::kLow && q.m <= kRefMost;
    HeadStat k;
    if (!in_head && lead && in.counts) flag_error(QQT_DEV_BAD_ACTION);
    k.act = in_head ? (int)act : -1;
    float lp;
    // (teams of one warp go together: whoever does not need it leaves it unused)
    if (G == 8 ? __any_sync(QQT_FULL, any && !one_step) : any && !one_step) {
      Sums qp = q;
      plain_sums<T, G>(p, lg, w, tl, step, qp, plain_buf);
      if (any && !one_step) q = qp;
    }
    if (any && !one_step) {
      plain |= 1u << h;
      lp = finish_head(k, any, q.s, logf(q.s), q.e, z_act - q.m, z_act != -INFINITY);
      refs[h] = q.m;
    } else {
      // (far below, where the product may overflow, the maximum is no part of it)
      const float ta = z_act < -1.0e30f ? z_act : fmaf(z_act, kLog2e, -q.r) * kLn2;
      lp = finish_head(k, any, q.s, log2f(q.s) * kLn2, q.e * kLn2, ta, z_act != -INFINITY);
      refs[h] = q.r;
    }
    logp = add_logp(logp, lp);
    ent += k.ent;
    hs[h] = k;
    at += w;
  }
  if (lead) {
    if (a.logp) a.logp[r] = logp;
    if (a.entropy) a.entropy[r] = ent;
  }
  if (!a.old_logp) return;
  const bool live = logp != -INFINITY && in.counts;
  const RowLoss l = loss_of(a, in, logp, live);
  if (a.stats && lead)
    *reinterpret_cast<float4*>(part + r * 4) =
        make_float4(l.pg, l.kl, live ? ent : 0.f, l.clip);
  if (!a.dlogits) return;
  const float n_rows = fmaxf((float)(a.mask ? warp_sum(n_counted) : a.rows), 1.f);
  const float scale = a.grad_scale / n_rows * (a.upstream ? a.upstream[0] : 1.f);
  T* dz = (T*)a.dlogits + r * a.dlogits_stride;
  at = 0;
#pragma unroll 1
  for (int h = 0; h < a.n_heads; ++h) {
    const int w = a.width[h], nv = (w + VEC - 1) / VEC;
    const HeadStat k = hs[h];
    const T* p = z + at;
    T* o = dz + at;
    const uint8_t* lg = LEGAL ? legal + at : nullptr;
    const int sh = misfit(p), osh = misfit(o);
    const float cn = head_c(k, a.entropy_coef), kn = head_k(k, l.g, a.entropy_coef);
    if (live && ((plain >> h) & 1)) {    // (G = 8: divergent, no lane needs another)
      if (exists)
        for (int i = tl; i < w; i += step) {
          const float t = plain_t(p, lg, i, refs[h]);
          if (i != k.act) o[i] = from_f<T>(expf(t) * fmaf(cn, t, kn) * scale);
        }
    }
    const bool skip = live && ((plain >> h) & 1);
    const float ref = refs[h];
    const f32x2 nr = pair(-ref, -ref), l2 = pair(kLog2e, kLog2e), cs = pair(cn * kLn2, cn * kLn2),
                ks = pair(kn, kn), sc = pair(scale, scale);
    if (G == 8 || !skip) {
#pragma unroll 1
      for (int jb = 0; jb + wj < nv; jb += step * U) {
        const int j0 = jb + tl;
        const int last = jb + wj + (U - 1) * step + LANES;
        const bool whole = last * VEC <= w && exists && !skip;
        const bool inner = G != 8 && (sh == 0 || jb + wj > 0) && (last + (sh ? 1 : 0)) * VEC <= w;
        Vec<T, VEC> c[U];
        if (live) get_chunk<T, VEC, U>(p, sh, j0, step, w, inner, c);
        if (LEGAL && live)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (j0 + u * step < nv) bar_illegal<T, VEC>(c[u], lg, j0 + u * step, w);
        float f[U][VEC];
        if (live) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            L::lift(c[u]);
#pragma unroll
            for (int v = 0; v < VEC; v += 2) {
              const f32x2 t = fma2(pair(c[u].get(v), c[u].get(v + 1)), l2, nr);
              const f32x2 d = mul2(mul2(exp2_pair(t), fma2(cs, t, ks)), sc);
              f[u][v] = d.x;
              f[u][v + 1] = d.y;
            }
            c[u].put(f[u]);
          }
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) c[u] = vec_zero<T, VEC>();
        }
        if (G != 8 && whole && osh == 0) {
          uint4* q = reinterpret_cast<uint4*>(o) + j0;
#pragma unroll
          for (int u = 0; u < U; ++u, q += step) *q = *reinterpret_cast<const uint4*>(&c[u]);
        } else if (G != 8 && whole) {
#pragma unroll
          for (int u = 0; u < U; ++u) put_inner<T, VEC>(o, osh, j0 + u * step, c[u]);
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int j = j0 + u * step;
            put_grads<T, VEC, LANES>(o, osh, j, w, j < nv && exists && !skip, c[u]);
          }
        }
      }
    }
    // the action's own value, over what its vector's lane or the one above wrote
    __syncwarp();
    if (live && exists && k.act >= 0 && k.act / VEC % step == tl)
      o[k.act] = from_f<T>(action_grad(k, l.g, a.entropy_coef, scale));
    at += w;
  }
}

// Means over the counted rows from n partial sums, in a fixed order.
__global__ void __launch_bounds__(1024)
    k_pl_stats(QqtPolicyLoss a, const float* __restrict__ part, int64_t n,
               const int* __restrict__ counts) {
  __shared__ float buf[4][32];
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  before_me_done();
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < n; r += 1024) {
    const float4 v = *reinterpret_cast<const float4*>(part + r * 4);
    s[0] += v.x;
    s[1] += v.y;
    s[2] += v.z;
    s[3] += v.w;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    s[k] = warp_sum_f(s[k]);
    if (lane_id() == 0) buf[k][warp_id()] = s[k];
  }
  __syncthreads();
  if (warp_id() > 0) return;
  const float count = rows_counted(a, counts);
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = warp_sum_f(buf[k][lane_id()]) / count;
  if (lane_id() == 0) {
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
        const size_t smem = (size_t)kPlSmallRows * (v & 3 ? v : v + 1) * 4;
        auto run = [&](auto nh) {
          launch_early(k_pl_small<T, decltype(nh)::value>, dim3(blocks), dim3(kPlSmallRows), smem, st,
                    counts != nullptr, args, (int)v, counts, part, (int)one);
        };
        if (a->n_heads == 1)
          run(std::integral_constant<int, 1>{});
        else if (a->n_heads == 2)
          run(std::integral_constant<int, 2>{});
        else
          run(std::integral_constant<int, QQT_MAX_HEADS>{});
        return 0;
      }
      // a team of 8 lanes holds rows of up to 32 vectors in one step, a warp
      // walks over rows of up to 1024 (16384 rows x 8192 bf16: 148 us, 195 by
      // blocks), blocks take the rest, larger ones for long rows, whose second
      // reading then still finds them in L2 (8192 x 32000 bf16: 233 us with
      // 256 threads, 292 with 512; 4096 x 32000 f32: 249 and 220).  The choice
      // does not depend on what is asked for, so neither do a row's sums.
      const int64_t bytes = v * (int64_t)sizeof(T);
      const int g = bytes <= 32 * 16 ? 8 : bytes <= 1024 * 16 ? 32 : 0;
      const int threads = g || bytes <= 80 * 1024 ? 256 : kPlThreads;
      const int per = g ? threads / g : 1;
      const unsigned n = (unsigned)((a->rows + per - 1) / per);
      auto run = [&](auto gg) {
        constexpr int G = decltype(gg)::value;
        if (a->legal)
          launch_early(k_pl_rows<T, G, true>, dim3(n), dim3(threads), 0, st, counts != nullptr, args, counts, part);
        else
          launch_early(k_pl_rows<T, G, false>, dim3(n), dim3(threads), 0, st, counts != nullptr, args, counts, part);
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
    launch_early(k_pl_stats, dim3(1), dim3(1024), 0, st, a->rows > 0, args, part, small ? blocks : a->rows, counts);
  return launch_status();
}
