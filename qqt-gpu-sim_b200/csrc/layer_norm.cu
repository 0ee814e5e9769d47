// Layer norm over the last d values of each row, forward and backward
// (the norms of the MLP and CNN policies, train/model.py:77-101, 140-153, and
// of the memory policy).
//   y  = (x - mean) rstd w + b,   rstd = 1 / sqrt(var + eps)
//   dx = rstd (q - mean(q) - xh mean(q xh)),  q = dy w,  xh = (x - mean) rstd
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// All statistics and sums are float32; the mean comes first and the variance
// is taken around it (no cancellation for rows far from zero); outputs are
// rounded once.
//
// Memory bound: 2 values moved per element forward, 3 backward (one read of x
// and dy serves dx and the weight's gradient).  A row stays in the registers
// of its team -- 8 to 32 lanes, or a block, by the row's number of 16-byte
// vectors -- between the passes over it.  The backward teams walk over rows
// and keep their columns' sums of dy xh and dy in registers; each block writes
// one partial row and a second kernel adds the partials in a fixed order, so
// there are no atomics and results repeat.  Rows that are not made of whole
// vectors go value by value; rows too long for a block's registers are read
// again for every pass.
//
// Measured on a B200 (its copy bandwidth is 6.55 TB/s):
//   1048576 x 128 f32    forward 172 us, 6.2 TB/s; backward 253 us, 6.4 TB/s
//   5632 x 10816 f16     forward 57 us, 4.3 TB/s; backward 102 us, 3.6 TB/s
//   11267 x 2704 bf16    forward 30 us, 4.0 TB/s; backward 56 us, 3.3 TB/s
//   40000 x 512 f32      forward 32 us, 5.1 TB/s; backward 48 us, 5.1 TB/s
//   20000 x 1351 bf16    forward 57 us, 1.9 TB/s; backward 111 us, 1.5 TB/s
// Short rows are bound by memory.  Rows of a block, 16-bit ones above all, are
// bound by what each row costs its block beside the memory: two exchanges
// across the warps forward and one of two sums backward, with 24 warps an SM
// in all (the backward pass holds 32 sums and 16 weights a thread).  Rows read
// value by value are bound by their loads: one of 2 bytes a lane in place of
// one of 16, and one row ahead at most.

#include "ops_common.cuh"

namespace qqt {

constexpr int kLnWarpThreads = 256;   // block of the teams inside a warp
// Blocks of an SM that walk over rows.  Forward more than are resident (rows
// are short, the last blocks even out: 180 against 187 us with 8 at 1048576 x
// 128 f32); backward as many as are resident, since every block ends in a
// partial row: 3 with 80 registers (250 us, 294 with 4 that do not all fit), 2
// with 128 where a lane holds 16 values (40000 x 512 f32: 48 us, 78 with 3 and
// sums that spill).
constexpr int kLnFwdBlocks = 16;
__host__ __device__ constexpr int ln_bwd_blocks(int e) { return e >= 16 ? 2 : 3; }
// Threads of an SM in blocks that take a row each, 16 or 32 elements a thread.
constexpr int kLnRowThreads16 = 768, kLnRowThreads32 = 512;

// Largest block that walks rows with e elements a thread: the backward pass
// keeps 2 e sums besides its operands.
__host__ __device__ constexpr int ln_max_threads(int e) { return e == 16 ? 768 : 512; }
// That of rows read value by value with their weights in registers, backward
// (3000 x 7001 f16: 105 us, 136 with 768 threads of 80 registers).
constexpr int kLnSpreadThreads = 512;

// 1 / sqrt(v) of the unit with one Newton step: float32 accuracy.  Where v or r
// is infinite the step is 0 x inf, and r is the value already.
__device__ __forceinline__ float ln_rstd(float v) {
  const float r = rsqrtf(v);
  return r == INFINITY || r == 0.f ? r : r * fmaf(-0.5f * v * r, r, 1.5f);
}

// Sums of N values over a team of G lanes (G <= 32), or over the block (G =
// 0; buf holds 2 x N x 32 floats, used in turn so that one barrier is enough).
template <int G, int N>
__device__ __forceinline__ void team_sum(float* v, float (*buf)[N][32], int& turn) {
#pragma unroll
  for (int o = (G ? G : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(QQT_FULL, v[k], o);
  if (G == 0) {
    const int nw = blockDim.x >> 5;
    float(*b)[32] = buf[turn];
    turn ^= 1;
    if (lane_id() == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) b[k][warp_id()] = v[k];
    __syncthreads();
    const int l = nw <= 8 ? lane_id() & 7 : lane_id();
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = l < nw ? b[k][l] : 0.f;
    if (nw <= 8) {
#pragma unroll
      for (int o = 4; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(QQT_FULL, v[k], o);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = warp_sum_f(v[k]);
    }
  }
}

// What a thread holds: vectors j, j + step, ... of its team's row, of nv.
struct LnTeam {
  int64_t row, rows_step;
  int j, step;
};
template <int G>
__device__ __forceinline__ LnTeam ln_team() {
  LnTeam t;
  if (G) {
    constexpr int per = kLnWarpThreads / (G ? G : 1);
    t.row = (int64_t)blockIdx.x * per + threadIdx.x / (G ? G : 1);
    t.rows_step = (int64_t)gridDim.x * per;
    t.j = threadIdx.x % (G ? G : 1);
    t.step = G;
  } else {
    t.row = blockIdx.x;
    t.rows_step = gridDim.x;
    t.j = threadIdx.x;
    t.step = blockDim.x;
  }
  return t;
}

// How a row of d values lies in its team's registers.  WHOLE: vectors of VEC
// values, each one access.  SINGLE: the same vectors value by value, where some
// address is not on 16 bytes; the sums are WHOLE's.  SPREAD: where d is not
// made of vectors, the values j, j + step, ... of lane j, so that the lanes of
// an access lie side by side (3000 x 7001 f16, forward: 56 us, 93 by runs of 8
// values a lane; 20000 x 1351 bf16: 55 and 100).  Values past the row's end are 0.
enum LnMode { SINGLE, WHOLE, SPREAD };
template <int VEC, LnMode M>
__device__ __forceinline__ int ln_col(int j, int v, int step) {      // of value v of vector j
  return M == SPREAD ? j + v * step : j * VEC + v;
}
// The next vector's j, and the end of j.
template <int VEC, LnMode M>
__device__ __forceinline__ int ln_next(int step) {
  return M == SPREAD ? VEC * step : step;
}
template <int VEC, LnMode M>
__device__ __forceinline__ int ln_end(int d) {
  return M == SPREAD ? d : (d + VEC - 1) / VEC;
}
template <class T, int VEC, LnMode M>
__device__ __forceinline__ Vec<T, VEC> ln_get(const T* p, int j, int step, int d) {
  if constexpr (M == WHOLE) {
    return ld_vec<T, VEC>(p + (int64_t)j * VEC);
  } else {
    Vec<T, VEC> r;
    T e[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const int c = ln_col<VEC, M>(j, v, step);
      e[v] = M == SINGLE || c < d ? p[c] : from_f<T>(0.f);
    }
    if constexpr (sizeof(T) == 4) {
      r.put(e);
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
      for (int v = 0; v < VEC; v += 2)
        w[v / 2] = __byte_perm(*reinterpret_cast<const unsigned short*>(&e[v]),
                               *reinterpret_cast<const unsigned short*>(&e[v + 1]), 0x5410);
    }
    return r;
  }
}
template <class T, int VEC, LnMode M>
__device__ __forceinline__ void ln_put(T* p, int j, int step, int d, const float* f) {
  if constexpr (M == WHOLE) {
    Vec<T, VEC> r;
    r.put(f);
    st_vec(p + (int64_t)j * VEC, r);
  } else {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const int c = ln_col<VEC, M>(j, v, step);
      if (M == SINGLE || c < d) p[c] = from_f<T>(f[v]);
    }
  }
}
template <int VEC, LnMode M>
__device__ __forceinline__ Vec<float, VEC> ln_param(const float* p, int j, int step, int d) {
  if constexpr (M == WHOLE && VEC == 8) {
    Vec<float, VEC> r;
    const float4 lo = *reinterpret_cast<const float4*>(p + j * 8);
    const float4 hi = *reinterpret_cast<const float4*>(p + j * 8 + 4);
    const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    r.put(f);
    return r;
  } else {
    return ln_get<float, VEC, M>(p, j, step, d);
  }
}
template <class T, int VEC, int K, LnMode M>
__device__ __forceinline__ void ln_load(const T* p, const LnTeam& t, int d, bool on,
                                        Vec<T, VEC>* out) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = t.j + k * ln_next<VEC, M>(t.step);
    out[k] = on && j < ln_end<VEC, M>(d) ? ln_get<T, VEC, M>(p, j, t.step, d) : vec_zero<T, VEC>();
  }
}
// The parameters of a thread's columns where they stay in registers (KEEP).
template <int VEC, int K, LnMode M, bool KEEP>
struct LnParams {
  Vec<float, VEC> r[KEEP ? K : 1];
  __device__ __forceinline__ void read(const float* p, const LnTeam& t, int d) {
    if constexpr (KEEP) ln_load<float, VEC, K, M>(p, t, d, p != nullptr, r);
  }
  __device__ __forceinline__ Vec<float, VEC> get(const float* p, int k, int j, int step, int d) const {
    if constexpr (KEEP) return r[k];
    return ln_param<VEC, M>(p, j, step, d);
  }
};
// The steps of both passes on one vector, two values at a time.
// Sums f, and its square once it is centred.
template <int VEC>
__device__ __forceinline__ void ln_sum(const float* f, f32x2& s) {
#pragma unroll
  for (int v = 0; v < VEC; v += 2) s = add2(s, pair(f[v], f[v + 1]));
}
template <int VEC>
__device__ __forceinline__ void ln_centre(float* f, float mu, f32x2& s) {
  const f32x2 m = pair(-mu, -mu);
#pragma unroll
  for (int v = 0; v < VEC; v += 2) {
    const f32x2 c = add2(pair(f[v], f[v + 1]), m);
    f[v] = c.x;
    f[v + 1] = c.y;
    s = fma2(c, c, s);
  }
}
// The scaled and shifted row.
template <int VEC>
__device__ __forceinline__ void ln_scale(const float* c, float rs, const Vec<float, VEC>& w,
                                         bool has_b, const Vec<float, VEC>& b, float* o) {
  const f32x2 r = pair(rs, rs);
#pragma unroll
  for (int v = 0; v < VEC; v += 2) {
    const f32x2 x = mul2(pair(c[v], c[v + 1]), r), wv = pair(w.get(v), w.get(v + 1));
    const f32x2 y = has_b ? fma2(x, wv, pair(b.get(v), b.get(v + 1))) : mul2(x, wv);
    o[v] = y.x;
    o[v + 1] = y.y;
  }
}
// Backward, first half: the sums of dy xh and dy (columns), of q and q xh (row).
template <int VEC, class C>
__device__ __forceinline__ void ln_gather(const C& cx, const C& cy,
                                          const float* w, float mu, float rs, float* aw, float* ab,
                                          f32x2& s1, f32x2& s2) {
  const f32x2 m = pair(-mu, -mu), r = pair(rs, rs);
#pragma unroll
  for (int v = 0; v < VEC; v += 2) {
    const f32x2 g = pair(cy.get(v), cy.get(v + 1));
    const f32x2 xh = mul2(add2(pair(cx.get(v), cx.get(v + 1)), m), r);
    const f32x2 q = mul2(g, pair(w[v], w[v + 1]));
    const f32x2 nb = add2(pair(ab[v], ab[v + 1]), g), nw = fma2(g, xh, pair(aw[v], aw[v + 1]));
    ab[v] = nb.x;
    ab[v + 1] = nb.y;
    aw[v] = nw.x;
    aw[v + 1] = nw.y;
    s1 = add2(s1, q);
    s2 = fma2(q, xh, s2);
  }
}
// Second half: dx = rs q - rs m1 - (x - mu) rs^2 m2, m1 and m2 the row's means.
template <int VEC, class C>
__device__ __forceinline__ void ln_spread(const C& cx, const C& cy,
                                          const float* w, float mu, float rs, float m1, float m2,
                                          float* o) {
  const f32x2 m = pair(-mu, -mu), r = pair(rs, rs);
  const float a = -rs * m1, b = -rs * rs * m2;
  const f32x2 c1 = pair(a, a), c2 = pair(b, b);
#pragma unroll
  for (int v = 0; v < VEC; v += 2) {
    const f32x2 q = mul2(pair(cy.get(v), cy.get(v + 1)), pair(w[v], w[v + 1]));
    const f32x2 x = add2(pair(cx.get(v), cx.get(v + 1)), m);
    const f32x2 y = fma2(q, r, fma2(x, c2, c1));
    o[v] = y.x;
    o[v + 1] = y.y;
  }
}

template <class T, int VEC, int K, int G, LnMode M>
__global__ void __launch_bounds__(G ? kLnWarpThreads : ln_max_threads(VEC * K))
    k_ln_fwd(const T* __restrict__ x, int64_t xs, int64_t rows, int d, const float* __restrict__ w,
             const float* __restrict__ b, float eps, T* __restrict__ y, float* __restrict__ mean,
             float* __restrict__ rstd) {
  __shared__ float buf[2][1][32];
  int turn = 0;
  const int nv = ln_end<VEC, M>(d);
  const float inv_d = 1.f / (float)d;
  LnTeam t = ln_team<G>();
  // (a team's lanes shuffle together with the rest of their warp, so a warp
  // goes on until its last team is done)
  const int64_t lead = G && G < 32 ? t.row - (threadIdx.x % 32) / (G ? G : 1) : t.row;
  LnParams<VEC, K, M, M != WHOLE && VEC * K <= 16> pw, pb;
  pw.read(w, t, d);
  pb.read(b, t, d);
  Vec<T, VEC> c[K];
  ln_load<T, VEC, K, M>(x + t.row * xs, t, d, t.row < rows, c);
  for (int64_t lr = lead; lr < rows; lr += t.rows_step) {
    const bool on = t.row < rows;
    float f[K][VEC];
    f32x2 s2 = pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) f[k][v] = c[k].get(v);
      ln_sum<VEC>(f[k], s2);
    }
    float s[1] = {s2.x + s2.y};
    // the next row's values are on their way meanwhile
    const int64_t next = t.row + t.rows_step;
    ln_load<T, VEC, K, M>(x + next * xs, t, d, next < rows, c);
    team_sum<G, 1>(s, buf, turn);
    const float mu = s[0] * inv_d;
    s2 = pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = t.j + k * ln_next<VEC, M>(t.step);
      if (j < nv) {
        if (M == SPREAD && ln_col<VEC, M>(j, VEC - 1, t.step) >= d)   // no values: they add nothing
#pragma unroll
          for (int v = 0; v < VEC; ++v)
            if (ln_col<VEC, M>(j, v, t.step) >= d) f[k][v] = mu;
        ln_centre<VEC>(f[k], mu, s2);
      }
    }
    s[0] = s2.x + s2.y;
    team_sum<G, 1>(s, buf, turn);
    const float rs = ln_rstd(s[0] * inv_d + eps);
    if (on) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int j = t.j + k * ln_next<VEC, M>(t.step);
        if (j < nv) {
          const Vec<float, VEC> wv = pw.get(w, k, j, t.step, d);
          const Vec<float, VEC> bv = b ? pb.get(b, k, j, t.step, d) : wv;
          float o[VEC];
          ln_scale<VEC>(f[k], rs, wv, b != nullptr, bv, o);
          ln_put<T, VEC, M>(y + t.row * d, j, t.step, d, o);
        }
      }
      if (t.j == 0 && mean) {
        mean[t.row] = mu;
        rstd[t.row] = rs;
      }
    }
    t.row = next;
  }
}

// dx of the team's rows, and the block's partial sums of dy xh and dy.
template <class T, int VEC, int K, int G, LnMode M>
__global__ void __launch_bounds__(G ? kLnWarpThreads : M == SPREAD ? kLnSpreadThreads : ln_max_threads(VEC * K),
                  G ? ln_bwd_blocks(VEC * K) : 1)
    k_ln_bwd(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
             int64_t rows, int d, const float* __restrict__ mean, const float* __restrict__ rstd,
             const float* __restrict__ w, T* __restrict__ dx, float* __restrict__ part) {
  __shared__ float buf[2][2][32];
  extern __shared__ float sums[];          // teams inside a warp: [teams][2 d]
  int turn = 0;
  const int nv = ln_end<VEC, M>(d);
  const float inv_d = 1.f / (float)d;
  LnTeam t = ln_team<G>();
  const int64_t lead = G && G < 32 ? t.row - (threadIdx.x % 32) / (G ? G : 1) : t.row;
  // Columns read value by value keep their weights in registers where the sums
  // leave room (60000 x 200 bf16 rows of stride 201: 42 us, 63 without; 30011 x
  // 517 bf16: 77 and 87).
  LnParams<VEC, K, M, (M != WHOLE && G != 0) || (M == SPREAD && VEC * K <= 16)> pr;
  pr.read(w, t, d);
  float aw[K][VEC], ab[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int v = 0; v < VEC; ++v) aw[k][v] = ab[k][v] = 0.f;
  // Where registers allow it the next row is loaded while this one is finished
  // (80000 x 384 f16: 51 us, 55 without).
  constexpr bool AHEAD =
      VEC * K <= 8 || (sizeof(T) == 2 && VEC * K <= 16 && (G != 0 || M == SPREAD));
  Vec<T, VEC> cx[K], cy[K];
  ln_load<T, VEC, K, M>(x + t.row * xs, t, d, t.row < rows, cx);
  ln_load<T, VEC, K, M>(dy + t.row * dys, t, d, t.row < rows, cy);
  float mu = t.row < rows ? mean[t.row] : 0.f, rs = t.row < rows ? rstd[t.row] : 0.f;
  for (int64_t lr = lead; lr < rows; lr += t.rows_step) {
    const bool on = t.row < rows;
    const float m0 = mu, r0 = rs;
    f32x2 s1 = pair(0.f, 0.f), s2 = s1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = t.j + k * ln_next<VEC, M>(t.step);
      if (j < nv) {
        const Vec<float, VEC> wv = pr.get(w, k, j, t.step, d);
        ln_gather<VEC>(cx[k], cy[k], wv.v, m0, r0, aw[k], ab[k], s1, s2);
      }
    }
    float s[2] = {s1.x + s1.y, s2.x + s2.y};
    Vec<T, VEC> px[K], py[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      px[k] = cx[k];
      py[k] = cy[k];
    }
    const int64_t next = t.row + t.rows_step;
    auto load_next = [&] {
      ln_load<T, VEC, K, M>(x + next * xs, t, d, next < rows, cx);
      ln_load<T, VEC, K, M>(dy + next * dys, t, d, next < rows, cy);
      if (next < rows) {
        mu = mean[next];
        rs = rstd[next];
      }
    };
    if (AHEAD || !dx) load_next();
    if (dx) {
      team_sum<G, 2>(s, buf, turn);
      const float m1 = s[0] * inv_d, m2 = s[1] * inv_d;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int j = t.j + k * ln_next<VEC, M>(t.step);
        if (on && j < nv) {
          float o[VEC];
          const Vec<float, VEC> wv = pr.get(w, k, j, t.step, d);
          ln_spread<VEC>(px[k], py[k], wv.v, m0, r0, m1, m2, o);
          ln_put<T, VEC, M>(dx + t.row * d, j, t.step, d, o);
        }
      }
      if (!AHEAD) load_next();
    }
    t.row = next;
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * d;
  if (G == 0) {                            // a block's threads own their columns
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = t.j + k * ln_next<VEC, M>(t.step);
      if (j < nv)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const int c = ln_col<VEC, M>(j, v, t.step);
          if (M != SPREAD || c < d) {
            pw[c] = aw[k][v];
            pw[d + c] = ab[k][v];
          }
        }
    }
    return;
  }
  constexpr int teams = kLnWarpThreads / (G ? G : 1);
  float* mine = sums + (int64_t)(threadIdx.x / (G ? G : 1)) * 2 * d;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = t.j + k * ln_next<VEC, M>(t.step);
    if (j < nv)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const int c = ln_col<VEC, M>(j, v, t.step);
        if (M != SPREAD || c < d) {
          mine[c] = aw[k][v];
          mine[d + c] = ab[k][v];
        }
      }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * d; c += kLnWarpThreads) {
    float a = 0.f;
#pragma unroll 8
    for (int q = 0; q < teams; ++q) a += sums[q * 2 * d + c];
    pw[c] = a;
  }
}

// ------------------------------------------- a block per row, rows staged
//
// Rows of whole 16-byte vectors beyond a warp's reach: a block walks over rows,
// bulk copies bring the next ones into a ring of stages in shared memory
// meanwhile, and the block's threads hold K vectors each.  A register holds
// one row's values at most, the ring the 2 to 8 rows that keep the memory
// system busy across the block's barriers.

constexpr int kLnStages = 8;
struct LnRing {
  int stages;
  uint32_t stage_bytes, row_bytes;
  uint32_t test_wait;      // polls of the failure-path check, 0 without it
};

// The last row that a block still fetches and waits for once its wait for `row`
// has run out: what is in flight is waited for, row by row, and nothing more
// is copied, so that nothing arrives after the block has given up its shared
// memory.
__device__ __forceinline__ int64_t ln_last(int64_t last, int64_t row, const LnRing& ring) {
  return min(last, row + (int64_t)(ring.stages - 1) * gridDim.x);
}

template <class T, int VEC, int K>
__global__ void __launch_bounds__(ln_max_threads(VEC* K))
    k_ln_row_fwd(const T* __restrict__ x, int64_t xs, int64_t rows, int d,
                 const float* __restrict__ w, const float* __restrict__ b, float eps,
                 T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, LnRing ring) {
  extern __shared__ __align__(128) unsigned char stage[];
  __shared__ uint64_t bar[kLnStages + 1];   // (the last is the failure-path check's)
  __shared__ float buf[2][1][32];
  int turn = 0;
  const int nv = (d + VEC - 1) / VEC;
  const float inv_d = 1.f / (float)d;
  int64_t last = rows - 1;
  auto fetch = [&](int64_t row, int s) {
    if (row <= last) {
      stage_arm(&bar[s], ring.row_bytes);
      stage_copy(stage + (size_t)s * ring.stage_bytes, x + row * xs, ring.row_bytes, &bar[s]);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s <= kLnStages; ++s) stage_init(&bar[s]);
    stage_init_done();
  }
  __syncthreads();
  if (threadIdx.x == 0)
    for (int s = 0; s < ring.stages; ++s) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
  // a block's columns do not change: weight and bias stay in registers
  Vec<float, VEC> wr[K], br[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = threadIdx.x + k * blockDim.x;
    wr[k] = j < nv ? ln_param<VEC, WHOLE>(w, j, 0, d) : vec_zero<float, VEC>();
    br[k] = j < nv && b ? ln_param<VEC, WHOLE>(b, j, 0, d) : vec_zero<float, VEC>();
  }
  int s = 0;
  uint32_t parity = 0;
  if (ring.test_wait && !stage_wait(&bar[kLnStages], 0, ring.test_wait))
    last = ln_last(last, blockIdx.x, ring);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    if (row <= last && !stage_wait(&bar[s], parity)) last = ln_last(last, row, ring);
    const T* in = (const T*)(stage + (size_t)s * ring.stage_bytes);
    float f[K][VEC];
    f32x2 s2 = pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = threadIdx.x + k * blockDim.x;
      if (j < nv) {
        const Vec<T, VEC> c = ld_vec<T, VEC>(in + j * VEC);
#pragma unroll
        for (int v = 0; v < VEC; ++v) f[k][v] = c.get(v);
        ln_sum<VEC>(f[k], s2);
      }
    }
    float sum[1] = {s2.x + s2.y};
    team_sum<0, 1>(sum, buf, turn);        // (its barrier: everyone has read the stage)
    if (threadIdx.x == 0) fetch(row + (int64_t)ring.stages * gridDim.x, s);
    const float mu = sum[0] * inv_d;
    s2 = pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (threadIdx.x + k * blockDim.x < nv) ln_centre<VEC>(f[k], mu, s2);
    sum[0] = s2.x + s2.y;
    team_sum<0, 1>(sum, buf, turn);
    const float rs = ln_rstd(sum[0] * inv_d + eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = threadIdx.x + k * blockDim.x;
      if (j < nv) {
        float o[VEC];
        ln_scale<VEC>(f[k], rs, wr[k], b != nullptr, br[k], o);
        ln_put<T, VEC, WHOLE>(y + row * d, j, 0, d, o);
      }
    }
    if (threadIdx.x == 0 && mean) {
      mean[row] = mu;
      rstd[row] = rs;
    }
    if (++s == ring.stages) {
      s = 0;
      parity ^= 1;
    }
  }
}

template <class T, int VEC, int K>
__global__ void __launch_bounds__(ln_max_threads(VEC* K))
    k_ln_row_bwd(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                 int64_t rows, int d, const float* __restrict__ mean,
                 const float* __restrict__ rstd, const float* __restrict__ w, T* __restrict__ dx,
                 float* __restrict__ part, LnRing ring) {
  extern __shared__ __align__(128) unsigned char stage[];
  __shared__ uint64_t bar[kLnStages + 1];   // (the last is the failure-path check's)
  __shared__ float buf[2][2][32];
  int turn = 0;
  const int nv = (d + VEC - 1) / VEC;
  const float inv_d = 1.f / (float)d;
  constexpr bool WREG = VEC * K <= 16;     // the weights fit beside the sums
  int64_t last = rows - 1;
  auto fetch = [&](int64_t row, int s) {
    if (row <= last) {
      unsigned char* to = stage + (size_t)s * ring.stage_bytes;
      stage_arm(&bar[s], 2 * ring.row_bytes);
      stage_copy(to, x + row * xs, ring.row_bytes, &bar[s]);
      stage_copy(to + ring.stage_bytes / 2, dy + row * dys, ring.row_bytes, &bar[s]);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s <= kLnStages; ++s) stage_init(&bar[s]);
    stage_init_done();
  }
  __syncthreads();
  if (threadIdx.x == 0)
    for (int s = 0; s < ring.stages; ++s) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
  float aw[K][VEC], ab[K][VEC], wr[WREG ? K : 1][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = threadIdx.x + k * blockDim.x;
    Vec<float, VEC> wv = vec_zero<float, VEC>();
    if (WREG && j < nv) wv = ln_param<VEC, WHOLE>(w, j, 0, d);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      aw[k][v] = ab[k][v] = 0.f;
      if (WREG) wr[WREG ? k : 0][v] = wv.get(v);
    }
  }
  int s = 0, before = -1;                  // before: the stage of the row before
  uint32_t parity = 0;
  float mu = 0.f, rs = 0.f;
  if (blockIdx.x < rows) {
    mu = mean[blockIdx.x];
    rs = rstd[blockIdx.x];
  }
  if (ring.test_wait && !stage_wait(&bar[kLnStages], 0, ring.test_wait))
    last = ln_last(last, blockIdx.x, ring);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float m0 = mu, r0 = rs;
    const int64_t next = row + gridDim.x;
    if (next < rows) {
      mu = mean[next];
      rs = rstd[next];
    }
    if (row <= last && !stage_wait(&bar[s], parity)) last = ln_last(last, row, ring);
    const T* ix = (const T*)(stage + (size_t)s * ring.stage_bytes);
    const T* iy = (const T*)((const unsigned char*)ix + ring.stage_bytes / 2);
    f32x2 s1 = pair(0.f, 0.f), s2 = s1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = threadIdx.x + k * blockDim.x;
      if (j < nv) {
        Vec<float, VEC> wv;
        if (!WREG) wv = ln_param<VEC, WHOLE>(w, j, 0, d);
        ln_gather<VEC>(ld_vec<T, VEC>(ix + j * VEC), ld_vec<T, VEC>(iy + j * VEC),
                          WREG ? wr[WREG ? k : 0] : wv.v, m0, r0, aw[k], ab[k], s1, s2);
      }
    }
    float sum[2] = {s1.x + s1.y, s2.x + s2.y};
    if (dx)
      team_sum<0, 2>(sum, buf, turn);      // (its barrier: the row before is done with)
    else
      __syncthreads();
    if (threadIdx.x == 0 && before >= 0)
      fetch(row + (int64_t)(ring.stages - 1) * gridDim.x, before);
    if (dx) {
      const float m1 = sum[0] * inv_d, m2 = sum[1] * inv_d;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int j = threadIdx.x + k * blockDim.x;
        if (j < nv) {
          Vec<float, VEC> wv;
          if (!WREG) wv = ln_param<VEC, WHOLE>(w, j, 0, d);
          float o[VEC];
          ln_spread<VEC>(ld_vec<T, VEC>(ix + j * VEC), ld_vec<T, VEC>(iy + j * VEC),
                            WREG ? wr[WREG ? k : 0] : wv.v, m0, r0, m1, m2, o);
          ln_put<T, VEC, WHOLE>(dx + row * d, j, 0, d, o);
        }
      }
    }
    before = s;
    if (++s == ring.stages) {
      s = 0;
      parity ^= 1;
    }
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = threadIdx.x + k * blockDim.x;
    if (j < nv)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        pw[j * VEC + v] = aw[k][v];
        pw[d + j * VEC + v] = ab[k][v];
      }
  }
}

// Adds the partial rows: a block takes 32 columns, each of its 32 warps every
// 32nd row.
__global__ void __launch_bounds__(1024) k_ln_add(const float* __restrict__ part, int n_part,
                                                 int64_t d, float* __restrict__ dw,
                                                 float* __restrict__ db) {
  __shared__ float buf[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + lane_id();
  const float* p = part + (int64_t)warp_id() * 2 * d + c;
  float s = 0.f;
  before_me_done();
  if (c < 2 * d) {
#pragma unroll 16
    for (int r = warp_id(); r < n_part; r += 32, p += 64 * d) s += *p;
  }
  buf[warp_id()][lane_id()] = s;
  __syncthreads();
  // column w of the 32 is warp w's to add
  s = warp_sum_f(buf[lane_id()][warp_id()]);
  const int64_t col = (int64_t)blockIdx.x * 32 + warp_id();
  if (lane_id() == 0 && col < 2 * d) {
    float* out = col < d ? dw : db;
    if (out) out[col < d ? col : col - d] = s;
  }
}

// ------------------------------------- rows longer than a block's registers

template <class T>
__global__ void k_ln_long_fwd(const T* __restrict__ x, int64_t xs, int64_t d, const float* __restrict__ w,
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
__global__ void k_ln_long_dx(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
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

template <class T>
__global__ void k_ln_long_part(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x,
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

// How rows are handed out: k vectors a thread, teams of g lanes (0: a block of
// `threads`), `blocks` blocks that walk over rows (0: rows too long for them).
// It does not depend on alignment, so neither do results.
struct LnPlan {
  int k, g, threads;
  int64_t blocks;
  LnRing ring;
};
static LnPlan ln_plan(int64_t rows, int64_t d, int vec, bool bwd) {
  LnPlan p{0, 0, kLnWarpThreads, 0, {0, 0, 0, 0}};
  const int64_t nv = (d + vec - 1) / vec;
  const int sms = sm_count();
  if (nv <= (vec == 8 ? 64 : 128)) {       // a team inside a warp
    const bool one = vec == 8 || nv <= 8;
    p.k = one ? 1 : 2;
    p.g = nv <= 8 * p.k ? 8 : nv <= 16 * p.k ? 16 : 32;
    if (nv > 32 * p.k) p.k *= 2;
    const int64_t per_block = kLnWarpThreads / p.g, need = (rows + per_block - 1) / per_block;
    const int64_t room = (int64_t)sms * (bwd ? ln_bwd_blocks(p.k * vec) : kLnFwdBlocks);
    p.blocks = need < room ? need : room;
    return p;
  }
  // a block: 16 elements a thread, 32 where that takes too many threads
  p.k = 16 / vec;
  const bool few = bwd && d % vec;          // SPREAD's backward pass
  if (nv > (int64_t)p.k * (few ? kLnSpreadThreads : ln_max_threads(16))) p.k *= 2;
  const int64_t th = (nv + p.k - 1) / p.k;
  if (th > ln_max_threads(p.k * vec)) return p;         // too long
  p.threads = (int)((th + 31) / 32 * 32);
  // blocks of an SM by the threads that the registers allow, and stages by the
  // shared memory that leaves each
  const int room = p.k * vec == 16 && !few ? kLnRowThreads16 : kLnRowThreads32;
  int per_sm = room / p.threads;
  per_sm = per_sm < 1 ? 1 : per_sm > 16 ? 16 : per_sm;
  const int64_t row = d * (16 / vec), stage = (row + 127) / 128 * 128 * (bwd ? 2 : 1);
  int64_t n = 220 * 1024 / per_sm / stage;
  while (n < 3 && per_sm > 1) n = 220 * 1024 / --per_sm / stage;
  if (n < 2) return p;                                  // too long for two stages
  p.ring = {(int)(n > kLnStages ? kLnStages : n), (uint32_t)stage, (uint32_t)row,
            g_test_wait_polls.load(std::memory_order_relaxed)};
  p.blocks = rows < (int64_t)sms * per_sm ? rows : (int64_t)sms * per_sm;
  return p;
}
static int64_t ln_parts(int64_t rows, int64_t d, int vec) {
  const LnPlan p = ln_plan(rows, d, vec, true);
  if (p.blocks > 0) return p.blocks;
  return rows < 512 ? (rows > 0 ? rows : 1) : 512;
}
// Whether rows of these strides and addresses are made of whole 16-byte vectors.
static bool ln_whole(int64_t es, int64_t d, int64_t s1, int64_t s2, const void* p1, const void* p2,
                     const void* p3, const void* w, const void* b) {
  const int64_t v = 16 / es;
  return d % v == 0 && s1 % v == 0 && s2 % v == 0 && aligned_to(p1, 16) && aligned_to(p2, 16) &&
         aligned_to(p3, 16) && aligned_to(w, 16) && aligned_to(b, 16);
}

static bool ln_allow_smem(const void* kernel, size_t bytes) {
  return bytes <= 48 * 1024 ||
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) ==
             cudaSuccess;
}
template <int VEC, class F>
static void ln_shapes(const LnPlan& p, F f) {
  using std::integral_constant;
#define QQT_LN(KK, GG) \
  if (p.k == KK && p.g == GG) return f(integral_constant<int, KK>{}, integral_constant<int, GG>{})
  QQT_LN(1, 8);
  QQT_LN(2, 32);
  QQT_LN(4, 0);
  if constexpr (VEC == 8) {
    QQT_LN(1, 16);
    QQT_LN(1, 32);
    QQT_LN(2, 0);
  } else {
    QQT_LN(2, 8);
    QQT_LN(2, 16);
    QQT_LN(4, 32);
    QQT_LN(8, 0);
  }
#undef QQT_LN
}

}  // namespace qqt

using namespace qqt;

extern "C" uint64_t qqt_layernorm_work_bytes(int64_t rows, int64_t d) {
  if (rows < 0 || d <= 0) return 0;
  const int64_t p4 = ln_parts(rows, d, 4), p8 = ln_parts(rows, d, 8);
  const int64_t parts = p4 > p8 ? p4 : p8;
  return (uint64_t)parts * 2 * (uint64_t)d * sizeof(float);
}

extern "C" int qqt_layernorm_forward(const void* x, int32_t dtype, int64_t rows, int64_t d,
                                     int64_t x_stride, const float* w, const float* b, float eps,
                                     void* y, float* mean, float* rstd, qqt_stream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || d <= 0 || x_stride < 0 || !(eps >= 0.f)) return QQT_E_ARG;
  if (rows > 0x7fffffffll || d > 0x3fffffffll) return QQT_E_LIMIT;
  if (rows == 0) return QQT_OK;
  if (!x || !w || !y || !mean != !rstd) return QQT_E_ARG;
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    constexpr int V = 16 / sizeof(T);
    cudaStream_t st = (cudaStream_t)stream;
    const bool whole = ln_whole(sizeof(T), d, x_stride, 0, x, y, nullptr, w, b);
    const LnPlan p = ln_plan(rows, d, V, false);
    const T* xp = (const T*)x;
    T* yp = (T*)y;
    const unsigned blocks = (unsigned)p.blocks;
    if (p.blocks == 0) {
      k_ln_long_fwd<T><<<(unsigned)rows, 1024, 0, st>>>(xp, x_stride, d, w, b, eps, yp, mean, rstd);
      return launch_status();
    }
    ln_shapes<V>(p, [&](auto kk, auto gg) {
      constexpr int K = decltype(kk)::value, G = decltype(gg)::value;
      auto run = [&](auto m) {
        k_ln_fwd<T, V, K, G, decltype(m)::value><<<blocks, p.threads, 0, st>>>(
            xp, x_stride, rows, (int)d, w, b, eps, yp, mean, rstd);
      };
      if (d % V) {
        run(std::integral_constant<LnMode, SPREAD>{});
      } else if (!whole) {
        run(std::integral_constant<LnMode, SINGLE>{});
      } else if constexpr (G == 0) {
        const size_t smem = (size_t)p.ring.stages * p.ring.stage_bytes;
        if (ln_allow_smem((const void*)k_ln_row_fwd<T, V, K>, smem))
          k_ln_row_fwd<T, V, K><<<blocks, p.threads, smem, st>>>(xp, x_stride, rows, (int)d, w, b, eps,
                                                                 yp, mean, rstd, p.ring);
      } else {
        run(std::integral_constant<LnMode, WHOLE>{});
      }
    });
    return launch_status();
  });
}

extern "C" int qqt_layernorm_backward(const void* dy, int64_t dy_stride, const void* x,
                                      int64_t x_stride, int32_t dtype, int64_t rows, int64_t d,
                                      const float* mean, const float* rstd, const float* w,
                                      void* dx, float* dw, float* db, void* work,
                                      qqt_stream_t stream) {
  if (!dtype_ok(dtype) || rows < 0 || d <= 0 || x_stride < 0 || dy_stride < 0) return QQT_E_ARG;
  if (rows > 0x7fffffffll || d > 0x3fffffffll) return QQT_E_LIMIT;
  if (rows > 0 && (!dy || !x || !mean || !rstd || !w)) return QQT_E_ARG;
  const bool sums = dw || db;
  if (sums && !work) return QQT_E_ARG;
  if (sums && !aligned_to(work, 16)) return QQT_E_ALIGN;
  return with_dtype(dtype, [&](auto e) {
    using T = decltype(e);
    constexpr int V = 16 / sizeof(T);
    cudaStream_t st = (cudaStream_t)stream;
    float* part = sums ? (float*)work : nullptr;
    const bool whole = ln_whole(sizeof(T), d, x_stride, dy_stride, x, dy, dx, w, nullptr);
    const LnPlan p = ln_plan(rows, d, V, true);
    const T *xp = (const T*)x, *yp = (const T*)dy;
    T* gp = (T*)dx;
    const unsigned blocks = (unsigned)p.blocks;
    const int64_t parts = rows > 0 ? ln_parts(rows, d, V) : 0;
    if (rows > 0 && p.blocks == 0) {
      if (dx)
        k_ln_long_dx<T><<<(unsigned)rows, 1024, 0, st>>>(yp, dy_stride, xp, x_stride, d, mean, rstd, w,
                                                         gp);
      if (sums)
        k_ln_long_part<T><<<dim3((unsigned)((d + 127) / 128), (unsigned)parts), 128, 0, st>>>(
            yp, dy_stride, xp, x_stride, rows, d, mean, rstd, part);
    } else if (rows > 0 && (dx || sums)) {
      ln_shapes<V>(p, [&](auto kk, auto gg) {
        constexpr int K = decltype(kk)::value, G = decltype(gg)::value;
        size_t smem = G ? (size_t)(kLnWarpThreads / (G ? G : 1)) * 2 * d * 4 : 0;
        auto run = [&](auto m) {
          k_ln_bwd<T, V, K, G, decltype(m)::value><<<blocks, p.threads, smem, st>>>(
              yp, dy_stride, xp, x_stride, rows, (int)d, mean, rstd, w, gp, part);
        };
        if (d % V) {
          run(std::integral_constant<LnMode, SPREAD>{});
        } else if (!whole) {
          run(std::integral_constant<LnMode, SINGLE>{});
        } else if constexpr (G == 0) {
          smem = (size_t)p.ring.stages * p.ring.stage_bytes;
          if (ln_allow_smem((const void*)k_ln_row_bwd<T, V, K>, smem))
            k_ln_row_bwd<T, V, K><<<blocks, p.threads, smem, st>>>(
                yp, dy_stride, xp, x_stride, rows, (int)d, mean, rstd, w, gp, part, p.ring);
        } else {
          run(std::integral_constant<LnMode, WHOLE>{});
        }
      });
    }
    if (sums)
      launch_early(k_ln_add, dim3((unsigned)((2 * d + 31) / 32)), dim3(1024), 0, st, rows > 0, part,
                   (int)parts, d, dw, db);
    return launch_status();
  });
}
