// Gated linear recurrence over T ticks of N sequences of width D, with resets
// at episode ends (the memory of a policy over its rollout).
//   f = sigmoid(gate_t),  k = 0 where reset_t else 1
//   h_t = f k h_{t-1} + (1 - f) x_t
// and its gradient, with e_t = dL/dh_t summed over every later use:
//   e_t = dh_t + f_{t+1} k_{t+1} e_{t+1}      (+ dh_last at the last tick)
//   dx_t = (1 - f) e_t,   dgate_t = f (1 - f) e_t (k h_{t-1} - x_t)
//   dh0 = f_1 k_1 e_1
// States are float32 whatever the type of the sequence.  The forward pass
// saves the state entering every kRecU ticks in float32 (half a byte per
// element and tick); the backward pass starts from it and rebuilds the kRecU
// states in registers, so rounded outputs are not read back.
//
// A thread walks its VEC channels ((n, d) pairs) along time, the loads of the
// tick kRecU later issued as soon as a tick is consumed.  Where the channels
// do not fill the GPU, time is cut into segments, and a thread walks one of
// them: a stretch of ticks acts on the state as h -> A h + B, and on the
// gradient that passes down through it as g -> A g + G, with the same A.  A
// first kernel finds each segment's pair (k_rec_sum), a second what enters
// each segment, one after the other (k_rec_join), and then every segment is
// walked from there: inputs are read twice, no block waits for another, and
// the order of all sums is fixed by the sizes.  A stretch that holds a reset
// has A = -0 (products of gates are +0 or more): what enters it is dropped by
// a select, whatever it is.
//
// Measured on a B200 (copy bandwidth 6.55 TB/s), bytes of the sequences alone:
//   128 ticks x 5632 x 128   f32: forward 183 us, 6.05 TB/s, backward 288 us,
//                            6.4 TB/s; bf16: 105 us, 5.3 TB/s, and 210 us, 4.4
//   65536 x 1024 bf16        forward 110 us (segment sums 40, join 8, walk 62),
//                            backward 174 us
//   10007 x 3 x 517 f32      forward 67 us, backward 97 us, 4-byte loads
// 32-bit sequences are bound by memory.  The 16-bit backward walk is bound by
// the loads it has in flight: 128 registers leave 16 warps an SM, each with 24
// 4-byte loads a lane (100 M warp instructions at an IPC of 0.45).

#include "ops_common.cuh"

namespace qqt {

constexpr int kRecU = 8;                     // ticks a thread holds, and between saved states
constexpr int kSeqThreads = 128;             // most threads of a block
// Blocks of an SM that the registers are cut for.  16-bit forward walks take 4
// channels a thread, backward ones 2: 8 ticks of 4 channels' states and
// operands do not fit 128 registers (213 against 340 us measured at 128 ticks
// x 5632 x 128).
constexpr int kFwdBlocks = 6, kBwdBlocks = 4;
// Segments are cut so that all walks run at once forward, in two rounds
// backward, where a second round fills the SMs that are done (16384 x 4 x 512:
// f32 forward 96 us against 105 in two rounds and 107 in three; bf16 backward
// 96 in two, 102 in one, 103 in three).
constexpr int kFwdRounds = 1, kBwdRounds = 2;
constexpr int64_t kRecMostSegs = 32768;      // (a grid's second dimension ends at 65535)

// f = sigmoid(g) and i = 1 - f = sigmoid(-g), each to a few units of its own
// last place: e = exp(-g), f = 1 / (1 + e), i = e f.  e = 2^(-g log2 e) carries
// the rounding of that product, |g| 2^-25 of itself; 32-bit sequences add the
// product's lost part back.  The exponent stops at 125, where f is 2^-125 and
// i is 1; a NaN passes.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <class T>
__device__ __forceinline__ void gates(f32x2 gate, f32x2& f, f32x2& i) {
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  f32x2 e;
  if constexpr (sizeof(T) == 4) {
    const f32x2 g = pair(max_nan(min_nan(gate.x, 120.f), -86.f), max_nan(min_nan(gate.y, 120.f), -86.f));
    const f32x2 l2 = pair(-kLog2e, -kLog2e);
    const f32x2 p = mul2(g, l2);
    // the product's rounding and log2 e's own tail
    const f32x2 lost = fma2(g, pair(-1.9259629911e-8f, -1.9259629911e-8f),
                            fma2(g, l2, pair(-p.x, -p.y)));
    e = pair(ex2_approx(p.x), ex2_approx(p.y));
    e = fma2(e, mul2(lost, pair(kLn2, kLn2)), e);
  } else {
    const f32x2 p = mul2(gate, pair(-kLog2e, -kLog2e));
    e = pair(ex2_approx(min_nan(p.x, 125.f)), ex2_approx(min_nan(p.y, 125.f)));
  }
  const f32x2 d = add2(e, pair(1.f, 1.f));
  f = pair(rcp_approx(d.x), rcp_approx(d.y));
  i = mul2(e, f);
}
// Values v and v + 1 of a vector (the second of a single one is a copy, never used).
template <class T, int VEC>
__device__ __forceinline__ f32x2 two(const Vec<T, VEC>& x, int v) {
  const float a = x.get(v);
  return pair(a, VEC > 1 ? x.get(v + 1) : a);
}
template <int VEC>
__device__ __forceinline__ f32x2 two(const float* x, int v) {
  return pair(x[v], VEC > 1 ? x[v + 1] : x[v]);
}
template <int VEC>
__device__ __forceinline__ void set_two(float* x, int v, f32x2 q) {
  x[v] = q.x;
  if (VEC > 1) x[v + 1] = q.y;
}
// A walk's tick: s = f s + i x.
template <class T, int VEC>
__device__ __forceinline__ void tick(const Vec<T, VEC>& x, const Vec<T, VEC>& g, float* s) {
#pragma unroll
  for (int v = 0; v < VEC; v += 2) {
    f32x2 f, i;
    gates<T>(two(g, v), f, i);
    set_two<VEC>(s, v, fma2(f, two<VEC>(s, v), mul2(i, two(x, v))));
  }
}

__device__ __forceinline__ bool drops(float a) { return __float_as_int(a) < 0; }
__device__ __forceinline__ float through(float a, float b, float s) {
  return drops(a) ? b : fmaf(a, s, b);
}

struct RecSeq {            // one (T, N, D) sequence: element strides of t and n
  const void* p;
  int64_t ts, ns;
};

struct RecArgs {
  RecSeq x, g, reset, h;           // h: output (forward), dh (backward)
  RecSeq dx, dg;
  const float* s0;                 // h0 or dh_last
  float* s_end;                    // h_last or dh0
  float* carry;                    // [ticks / kRecU rounded up][channels] states
  int64_t nT;
  uint32_t nC, nD;                 // channels (N D) and D
  int64_t seg;                     // ticks of a segment, a multiple of kRecU
  float2* pair;                    // [segments][channels] (A, B or G)
  float* enters;                   // [segments][channels] what enters each; null with one segment
};

// One tick for every channel: what acting does.
template <class T, int VEC>
__global__ void k_rec_step(RecArgs a) {
  const uint32_t c = (blockIdx.x * blockDim.x + threadIdx.x) * VEC;
  if (c >= a.nC) return;
  const int64_t n = c / a.nD, d = c - (uint32_t)n * a.nD;
  const auto x = ld_vec<T, VEC>((const T*)a.x.p + n * a.x.ns + d);
  const auto g = ld_vec<T, VEC>((const T*)a.g.p + n * a.g.ns + d);
  Vec<float, VEC> s;
  if (a.s0 && !(a.reset.p && ((const uint8_t*)a.reset.p)[n * a.reset.ns])) {
    s = ld_vec<float, VEC>(a.s0 + c);
  } else {
#pragma unroll
    for (int v = 0; v < VEC; ++v) s.v[v] = 0.f;
  }
  Vec<T, VEC> o;
  tick<T, VEC>(x, g, s.v);
  o.put(s.v);
  st_vec((T*)a.h.p + n * a.h.ns + d, o);
  if (a.s_end) st_vec(a.s_end + c, s);
}

// Where a thread's VEC channels are: of sequence n from d on.  A thread past
// the last channel reads the last ones and stores nothing.
struct RecPlace {
  uint32_t c;
  int64_t n, d;
  bool on, one_n;                  // one_n: the whole warp follows one sequence
};
template <int VEC>
__device__ __forceinline__ RecPlace rec_place(const RecArgs& a, uint32_t c) {
  RecPlace p;
  p.on = c < a.nC;
  p.c = p.on ? c : a.nC - VEC;
  const uint32_t n = p.c / a.nD;
  p.n = n;
  p.d = p.c - n * a.nD;
  p.one_n = __shfl_sync(QQT_FULL, n, 0) == __shfl_sync(QQT_FULL, n, 31);
  return p;
}
template <class T>
__device__ __forceinline__ T* at(const RecSeq& s, const RecPlace& p, int64_t t) {
  return (T*)s.p + p.n * s.ns + p.d + t * s.ts;
}

// The resets of kRecU ticks from t0 as a bit mask per lane.
__device__ __forceinline__ unsigned load_resets(const RecArgs& a, const RecPlace& p, int64_t t0) {
  if (!a.reset.p) return 0;
  const uint8_t* r = (const uint8_t*)a.reset.p + p.n * a.reset.ns;
  if (p.one_n) {
    const int64_t t = t0 + lane_id();
    return __ballot_sync(QQT_FULL, lane_id() < kRecU && t < a.nT && r[t * a.reset.ts]);
  }
  unsigned m = 0;
#pragma unroll
  for (int u = 0; u < kRecU; ++u)
    if (t0 + u < a.nT && r[(t0 + u) * a.reset.ts]) m |= 1u << u;
  return m;
}

template <class T, int VEC>
__device__ __forceinline__ void load_ticks(const T* p, int64_t ts, int n, Vec<T, VEC>* out) {
#pragma unroll
  for (int u = 0; u < kRecU; ++u, p += ts)
    if (u < n) out[u] = ld_vec<T, VEC>(p);
}

// ------------------------------------------------------ walking along time

template <class T, int VEC>
__global__ void __launch_bounds__(kSeqThreads, kFwdBlocks) k_rec_seq_fwd(RecArgs a) {
  const RecPlace p = rec_place<VEC>(a, (blockIdx.x * blockDim.x + threadIdx.x) * VEC);
  const int64_t first = blockIdx.y * a.seg;
  const int64_t ticks = a.nT - first < a.seg ? a.nT - first : a.seg;
  const T *xp = at<T>(a.x, p, first), *gp = at<T>(a.g, p, first);
  T* hp = at<T>(a.h, p, first);
  if (a.enters) before_me_done();
  const float* from = a.enters ? a.enters + (int64_t)blockIdx.y * a.nC : a.s0;
  Vec<float, VEC> s = from ? ld_vec<float, VEC>(from + p.c) : vec_zero<float, VEC>();
  float* cp = a.carry ? a.carry + first / kRecU * a.nC + p.c : nullptr;
  const int64_t full = ticks / kRecU;
  const int rem = (int)(ticks % kRecU);
  Vec<T, VEC> x[kRecU], g[kRecU];
  if (full > 0) {
    load_ticks<T, VEC>(xp, a.x.ts, kRecU, x);
    load_ticks<T, VEC>(gp, a.g.ts, kRecU, g);
  }
  unsigned rst = load_resets(a, p, first);
  for (int64_t b = 0; b < full; ++b) {
    const bool more = b + 1 < full;
    const unsigned rst_next = load_resets(a, p, first + (b + 1) * kRecU);
    if (cp) {
      if (p.on) st_vec(cp, s);
      cp += a.nC;
    }
    xp += kRecU * a.x.ts;
    gp += kRecU * a.g.ts;
    const T *xn = xp, *gn = gp;
#pragma unroll
    for (int u = 0; u < kRecU; ++u) {
      if ((rst >> u) & 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) s.v[v] = 0.f;
      }
      Vec<T, VEC> o;
      tick<T, VEC>(x[u], g[u], s.v);
      o.put(s.v);
      if (more) {
        x[u] = ld_vec<T, VEC>(xn);
        g[u] = ld_vec<T, VEC>(gn);
      }
      xn += a.x.ts;
      gn += a.g.ts;
      if (p.on) st_vec(hp, o);
      hp += a.h.ts;
    }
    rst = rst_next;
  }
  if (rem) {
    if (cp && p.on) st_vec(cp, s);
    load_ticks<T, VEC>(xp, a.x.ts, rem, x);
    load_ticks<T, VEC>(gp, a.g.ts, rem, g);
#pragma unroll
    for (int u = 0; u < kRecU; ++u) {
      if (u >= rem) break;
      if ((rst >> u) & 1) s = vec_zero<float, VEC>();
      Vec<T, VEC> o;
      tick<T, VEC>(x[u], g[u], s.v);
      o.put(s.v);
      if (p.on) st_vec(hp, o);
      hp += a.h.ts;
    }
  }
  if (a.s_end && p.on && first + ticks == a.nT) st_vec(a.s_end + p.c, s);
}

// Gradients of n ticks from the state entering them; acc: what enters from
// the later ticks, then what leaves below.  A first walk up finds the state
// before every tick, a second one down the gradients; the gates are computed
// again there, which costs less than the registers to hold them.  emit(u, dx,
// dgate) takes tick u's and may load what comes next into its operands.
// CLEAN: no lane has a reset.
template <class T, int VEC, bool CLEAN, class F>
__device__ __forceinline__ void backward_ticks(const Vec<T, VEC>* x, const Vec<T, VEC>* g,
                                               const Vec<T, VEC>* dh, unsigned rst, int n,
                                               Vec<float, VEC> s, Vec<float, VEC>& acc, F emit) {
  float prev[kRecU][VEC];
#pragma unroll
  for (int u = 0; u < kRecU; ++u) {
    if (u < n) {
      if (!CLEAN && ((rst >> u) & 1)) s = vec_zero<float, VEC>();
#pragma unroll
      for (int v = 0; v < VEC; ++v) prev[u][v] = s.v[v];
      if (u + 1 < kRecU) tick<T, VEC>(x[u], g[u], s.v);
    }
  }
#pragma unroll
  for (int u = kRecU - 1; u >= 0; --u) {
    if (u < n) {
      Vec<T, VEC> dx, dg;
      float fx[VEC], fg[VEC];
#pragma unroll
      for (int v = 0; v < VEC; v += 2) {
        f32x2 f, i;
        gates<T>(two(g[u], v), f, i);
        const f32x2 e = add2(two(dh[u], v), two<VEC>(acc.v, v));
        const f32x2 fe = mul2(f, e), px = two<VEC>(prev[u], v), xx = two(x[u], v);
        set_two<VEC>(fx, v, mul2(i, e));
        set_two<VEC>(fg, v, mul2(mul2(i, fe), add2(px, pair(-xx.x, -xx.y))));
        set_two<VEC>(acc.v, v, fe);
      }
      if (!CLEAN && ((rst >> u) & 1)) acc = vec_zero<float, VEC>();
      dx.put(fx);
      dg.put(fg);
      emit(u, dx, dg);
    }
  }
}

template <class T, int VEC>
__global__ void __launch_bounds__(kSeqThreads, kBwdBlocks) k_rec_seq_bwd(RecArgs a) {
  const RecPlace p = rec_place<VEC>(a, (blockIdx.x * blockDim.x + threadIdx.x) * VEC);
  const int64_t first = blockIdx.y * a.seg;
  const int64_t end = first + a.seg < a.nT ? first + a.seg : a.nT;
  const int64_t full = end / kRecU;    // (batches are counted from tick 0)
  const int rem = (int)(end % kRecU);
  const bool has_dh = a.h.p != nullptr;
  if (a.enters) before_me_done();
  const float* from = a.enters ? a.enters + (int64_t)blockIdx.y * a.nC : a.s0;
  Vec<float, VEC> acc = from ? ld_vec<float, VEC>(from + p.c) : vec_zero<float, VEC>();
  Vec<T, VEC> x[kRecU], g[kRecU], dh[kRecU];
#pragma unroll
  for (int u = 0; u < kRecU; ++u) dh[u] = vec_zero<T, VEC>();
  if (rem) {                         // the last, short stretch first
    const int64_t t0 = full * kRecU;
    load_ticks<T, VEC>(at<T>(a.x, p, t0), a.x.ts, rem, x);
    load_ticks<T, VEC>(at<T>(a.g, p, t0), a.g.ts, rem, g);
    if (has_dh) load_ticks<T, VEC>(at<T>(a.h, p, t0), a.h.ts, rem, dh);
    T *xo = at<T>(a.dx, p, t0), *go = at<T>(a.dg, p, t0);
    const Vec<float, VEC> s = ld_vec<float, VEC>(a.carry + full * a.nC + p.c);
    backward_ticks<T, VEC, false>(
        x, g, dh, load_resets(a, p, t0), rem, s, acc,
        [&](int u, const Vec<T, VEC>& dx, const Vec<T, VEC>& dg) {
          if (p.on) {
            st_vec(xo + u * a.dx.ts, dx);
            st_vec(go + u * a.dg.ts, dg);
          }
        });
  }
  const int64_t b0 = first / kRecU;
  if (full > b0) {
    int64_t b = full - 1;
    const T *xp = at<T>(a.x, p, b * kRecU), *gp = at<T>(a.g, p, b * kRecU);
    const T* hp = has_dh ? at<T>(a.h, p, b * kRecU) : nullptr;
    T *xo = at<T>(a.dx, p, full * kRecU), *go = at<T>(a.dg, p, full * kRecU);
    load_ticks<T, VEC>(gp, a.g.ts, kRecU, g);
    load_ticks<T, VEC>(xp, a.x.ts, kRecU, x);
    if (has_dh) load_ticks<T, VEC>(hp, a.h.ts, kRecU, dh);
    Vec<float, VEC> s = ld_vec<float, VEC>(a.carry + b * a.nC + p.c);
    unsigned rst = load_resets(a, p, b * kRecU);
    for (; b >= b0; --b) {
      const bool more = b > b0;
      Vec<float, VEC> s_next = s;
      unsigned rst_next = 0;
      // (the tick before the first is the last of the batch to come)
      const T *xn = xp - a.x.ts, *gn = gp - a.g.ts, *hn = hp - a.h.ts;
      if (more) {
        s_next = ld_vec<float, VEC>(a.carry + (b - 1) * a.nC + p.c);
        rst_next = load_resets(a, p, (b - 1) * kRecU);
      }
      auto emit = [&](int u, const Vec<T, VEC>& dx, const Vec<T, VEC>& dg) {
        if (more) {
          x[u] = ld_vec<T, VEC>(xn);
          g[u] = ld_vec<T, VEC>(gn);
          if (has_dh) dh[u] = ld_vec<T, VEC>(hn);
        }
        xn -= a.x.ts;
        gn -= a.g.ts;
        hn -= a.h.ts;
        xo -= a.dx.ts;
        go -= a.dg.ts;
        if (p.on) {
          st_vec(xo, dx);
          st_vec(go, dg);
        }
      };
      if (__all_sync(QQT_FULL, rst == 0))
        backward_ticks<T, VEC, true>(x, g, dh, rst, kRecU, s, acc, emit);
      else
        backward_ticks<T, VEC, false>(x, g, dh, rst, kRecU, s, acc, emit);
      gp -= kRecU * a.g.ts;
      xp -= kRecU * a.x.ts;
      hp -= kRecU * a.h.ts;
      s = s_next;
      rst = rst_next;
    }
  }
  if (a.s_end && p.on && first == 0) st_vec(a.s_end + p.c, acc);
}

// ------------------------------------------------------------- segments

// The pair of a segment of VEC channels: (A, B) of the state, or, with BWD,
// (A, G) of the gradient.  The segment is gone through against the direction
// of the walk that follows, which then finds what was read last -- the ticks
// it begins with -- still in L2.  P is the product of the gates between the
// tick and the segment's exit, so B = sum P' i x over the ticks, P' before the
// tick's own gate, and G = sum P dh with it.  What lies beyond a reset never
// comes through: P is -0 from there on, and nothing more is added.
// CLEAN: no lane has met a reset.
template <class T, int VEC, bool BWD, bool CLEAN>
__device__ __forceinline__ void pair_tick(const Vec<T, VEC>& x, const Vec<T, VEC>& g, bool r,
                                          float* A, float* B) {
#pragma unroll
  for (int v = 0; v < VEC; v += 2) {
    f32x2 f, i;
    gates<T>(two(g, v), f, i);
    const f32x2 P = two<VEC>(A, v), S = two<VEC>(B, v);
    f32x2 nA = mul2(P, f);
    if (!CLEAN) {
      nA.x = r || drops(P.x) ? -0.f : nA.x;
      nA.y = r || drops(P.y) ? -0.f : nA.y;
    }
    f32x2 nB = BWD ? fma2(nA, two(x, v), S) : fma2(P, mul2(i, two(x, v)), S);
    if (!CLEAN) {
      nB.x = drops(BWD ? nA.x : P.x) ? S.x : nB.x;
      nB.y = drops(BWD ? nA.y : P.y) ? S.y : nB.y;
    }
    set_two<VEC>(A, v, nA);
    set_two<VEC>(B, v, nB);
  }
}

template <class T, int VEC, bool BWD>
__global__ void __launch_bounds__(kSeqThreads, kFwdBlocks) k_rec_sum(RecArgs a) {
  const RecPlace p = rec_place<VEC>(a, (blockIdx.x * blockDim.x + threadIdx.x) * VEC);
  // the segments that some other one follows in the scan's direction
  const int64_t first = (blockIdx.y + (BWD ? 1 : 0)) * a.seg;
  const int64_t end = first + a.seg < a.nT ? first + a.seg : a.nT;
  const RecSeq& in = BWD ? a.h : a.x;
  const bool has_in = in.p != nullptr;
  float A[VEC], B[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    A[v] = 1.f;
    B[v] = 0.f;
  }
  Vec<T, VEC> x[kRecU], g[kRecU];
#pragma unroll
  for (int u = 0; u < kRecU; ++u) x[u] = vec_zero<T, VEC>();
  const int64_t full = end / kRecU, b0 = first / kRecU;   // batches counted from tick 0
  const int rem = (int)(end % kRecU);                      // (only in the last segment: BWD)
  bool done = false;
  if (full > b0) {
    const int64_t dir = BWD ? 1 : -1;
    int64_t b = BWD ? b0 : full - 1;
    const T* gp = at<T>(a.g, p, b * kRecU);
    const T* xp = has_in ? at<T>(in, p, b * kRecU) : nullptr;
    load_ticks<T, VEC>(gp, a.g.ts, kRecU, g);
    if (has_in) load_ticks<T, VEC>(xp, in.ts, kRecU, x);
    unsigned rst = load_resets(a, p, b * kRecU);
    // from here on the pointers are at the first tick of the next batch
    const int64_t gs = dir * a.g.ts, xs = dir * in.ts;
    const T* gn = BWD ? gp + kRecU * a.g.ts : gp - a.g.ts;
    const T* xn = BWD ? xp + kRecU * in.ts : xp - in.ts;
    for (int64_t left = full - b0; left > 0; --left) {
      const bool more = left > 1;
      b += dir;
      const unsigned rst_next = more ? load_resets(a, p, b * kRecU) : 0;
      auto batch = [&](auto clean) {
#pragma unroll
        for (int j = 0; j < kRecU; ++j) {
          const int u = BWD ? j : kRecU - 1 - j;
          pair_tick<T, VEC, BWD, decltype(clean)::value>(x[u], g[u], (rst >> u) & 1, A, B);
          if (more) {
            g[u] = ld_vec<T, VEC>(gn);
            if (has_in) x[u] = ld_vec<T, VEC>(xn);
          }
          gn += gs;
          xn += xs;
        }
      };
      if (__all_sync(QQT_FULL, rst == 0 && !drops(A[0])))
        batch(std::true_type{});
      else
        batch(std::false_type{});
      if (__all_sync(QQT_FULL, drops(A[0]))) {   // nothing more comes through
        done = true;
        break;
      }
      rst = rst_next;
    }
  }
  if (BWD && rem && !done) {
    load_ticks<T, VEC>(at<T>(a.g, p, full * kRecU), a.g.ts, rem, g);
    if (has_in) load_ticks<T, VEC>(at<T>(in, p, full * kRecU), in.ts, rem, x);
    const unsigned rst = load_resets(a, p, full * kRecU);
#pragma unroll
    for (int u = 0; u < kRecU; ++u)
      if (u < rem) pair_tick<T, VEC, BWD, false>(x[u], g[u], (rst >> u) & 1, A, B);
  }
  if (!p.on) return;
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    a.pair[(int64_t)blockIdx.y * a.nC + p.c + v] = make_float2(A[v], B[v]);
}

// What enters each segment.  Pair j is the j-th row that k_rec_sum wrote; with
// BWD the scan begins at the last.  A block takes 32 channels; each of its 32
// warps composes its share of the segments, one warp joins the shares, and
// then each walks its own: two short walks in place of one of all segments.
template <bool BWD>
__global__ void __launch_bounds__(1024) k_rec_join(RecArgs a, int segs) {
  __shared__ float sA[32][33], sB[32][33];
  const int l = lane_id(), w = warp_id();
  before_me_done();
  const uint32_t c0 = blockIdx.x * 32 + l;
  const bool on = c0 < a.nC;
  const uint32_t c = on ? c0 : a.nC - 1;
  const int per = (segs + 31) / 32;
  const int k0 = w * per, k1 = k0 + per < segs ? k0 + per : segs;
  constexpr int Q = 16;              // of a share's pairs, the last ones read stay in registers
  float2 v[Q];
  auto read = [&](int k) {           // those of the segments from the k-th along the scan
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (k + q < k1 && k + q + 1 < segs)
        v[q] = a.pair[(int64_t)(BWD ? segs - 2 - (k + q) : k + q) * a.nC + c];
  };
  float A = 1.f, B = 0.f;
  for (int k = k0; k < k1; k += Q) {
    read(k);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (k + q < k1 && k + q + 1 < segs) {
        B = through(v[q].x, v[q].y, B);
        A = drops(A) || drops(v[q].x) ? -0.f : A * v[q].x;
      }
    }
  }
  sA[w][l] = A;
  sB[w][l] = B;
  __syncthreads();
  if (w == 0) {
    float s = a.s0 ? a.s0[c] : 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) {
      const float nA = sA[q][l], nB = sB[q][l];
      sB[q][l] = s;
      s = through(nA, nB, s);
    }
  }
  __syncthreads();
  float s = sB[w][l];
  for (int k = k0; k < k1; k += Q) {
    if (per > Q) read(k);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (k + q < k1) {
        if (on) a.enters[(int64_t)(BWD ? segs - 1 - (k + q) : k + q) * a.nC + c] = s;
        if (k + q + 1 < segs) s = through(v[q].x, v[q].y, s);
      }
    }
  }
}

// How time is cut: segments of at least 4 kRecU ticks (8 measured 17 against
// 12 us at 512 ticks x 8 x 256), one where fewer than three would come of it
// (the inputs are read twice then).  It goes by the sizes and the type, not by
// alignment, and so does the order of the sums.
struct RecCut {
  int64_t seg;
  int segs, threads;
};
static RecCut rec_cut(int64_t T, int64_t C, int64_t D, int es, bool bwd) {
  const int v = D % 2 ? 1 : D % 4 == 0 && es == 2 && !bwd ? 4 : 2;
  const int64_t walks = C / v;
  const int threads = walks < kSeqThreads ? (int)(walks + 31) / 32 * 32 : kSeqThreads;
  const int64_t row = (walks + threads - 1) / threads;
  const int at_once = (bwd ? kBwdBlocks * kBwdRounds : kFwdBlocks * kFwdRounds) *
                      (kSeqThreads / threads);
  int64_t want = (int64_t)sm_count() * at_once / row;
  if (want > kRecMostSegs) want = kRecMostSegs;
  int64_t seg = want > 1 ? (T + want - 1) / want : T;
  if (seg < 4 * kRecU) seg = 4 * kRecU;
  seg = (seg + kRecU - 1) / kRecU * kRecU;
  const int64_t segs = (T + seg - 1) / seg;
  if (segs < 3) return {(T + kRecU - 1) / kRecU * kRecU, 1, threads};
  return {seg, (int)segs, threads};
}

static bool rec_sizes_ok(int64_t T, int64_t N, int64_t D) {
  return T >= 0 && N >= 0 && D > 0;
}
static bool rec_fits(int64_t T, int64_t N, int64_t D) {
  return T <= 0x7fffffffll && N <= 0x7fffffffll && D <= 0x7fffffffll && N * D <= 0x7fffff00ll;
}
static bool seq_vec(const RecSeq& s, int64_t bytes, int64_t es) {
  return !s.p || (aligned_to(s.p, bytes) && (s.ts * es) % bytes == 0 && (s.ns * es) % bytes == 0);
}
// Whether a step that writes `bytes` bytes from `out` on would write over what
// another thread has yet to read: n rows of `width` bytes from p, `stride` bytes
// apart, share memory with them, and not value by value (in_place).
static bool rec_clash(const void* out, int64_t bytes, const void* p, int64_t n, int64_t stride,
                      int64_t width, bool in_place) {
  const int64_t lo = (int64_t)(uintptr_t)out, hi = lo + bytes;
  int64_t at = (int64_t)(uintptr_t)p;
  if (at == 0 || (in_place && at == lo)) return false;
  if (stride < 0) {
    at += (n - 1) * stride;
    stride = -stride;
  }
  // the first row that ends beyond out's beginning
  const int64_t row = at + width > lo ? 0 : stride ? (lo - at - width) / stride + 1 : n;
  return row < n && at + row * stride < hi;
}
static RecSeq rec_seq(const QqtSeq* s) {
  return s ? RecSeq{s->p, s->t_stride, s->n_stride} : RecSeq{nullptr, 0, 0};
}

template <class T, int VEC, bool BWD>
static int rec_walk(RecArgs a, void* work, cudaStream_t st) {
  const RecCut cut = rec_cut(a.nT, a.nC, a.nD, sizeof(T), BWD);
  const dim3 threads(cut.threads);
  const unsigned blocks = (a.nC / VEC + cut.threads - 1) / cut.threads;
  a.seg = cut.seg;
  if (cut.segs > 1) {
    if (!work) return QQT_E_ARG;
    a.pair = (float2*)work;
    a.enters = (float*)(a.pair + (int64_t)(cut.segs - 1) * a.nC);
    k_rec_sum<T, VEC, BWD><<<dim3(blocks, cut.segs - 1), threads, 0, st>>>(a);
    launch_early(k_rec_join<BWD>, dim3((a.nC + 31) / 32), dim3(1024), 0, st, true, a, cut.segs);
  }
  const bool early = cut.segs > 1;
  if (BWD)
    launch_early(k_rec_seq_bwd<T, VEC>, dim3(blocks, cut.segs), threads, 0, st, early, a);
  else
    launch_early(k_rec_seq_fwd<T, VEC>, dim3(blocks, cut.segs), threads, 0, st, early, a);
  return launch_status();
}

// Channels that one access may cover: 4, 2 or 1.
static int rec_vec(const RecArgs& a, int64_t es) {
  for (int v = 4; v > 1; v /= 2)
    if (a.nD % v == 0 && seq_vec(a.x, v * es, es) && seq_vec(a.g, v * es, es) &&
        seq_vec(a.h, v * es, es) && seq_vec(a.dx, v * es, es) && seq_vec(a.dg, v * es, es) &&
        aligned_to(a.s0, 4 * v) && aligned_to(a.s_end, 4 * v) && aligned_to(a.carry, 4 * v))
      return v;
  return 1;
}

template <class T, bool BWD>
static int rec_run(const RecArgs& a, void* work, cudaStream_t st) {
  const int vec = rec_vec(a, sizeof(T));
  if constexpr (sizeof(T) == 2 && !BWD) {
    if (vec == 4) return rec_walk<T, 4, BWD>(a, work, st);
  }
  return vec >= 2 ? rec_walk<T, 2, BWD>(a, work, st) : rec_walk<T, 1, BWD>(a, work, st);
}

}  // namespace qqt

using namespace qqt;

extern "C" int64_t qqt_recurrence_chunks(int64_t T) {
  return T <= 0 ? 0 : (T + kRecU - 1) / kRecU;
}

extern "C" uint64_t qqt_recurrence_work_bytes(int64_t T, int64_t N, int64_t D) {
  if (!rec_sizes_ok(T, N, D) || !rec_fits(T, N, D) || T == 0 || N == 0) return 0;
  int segs = 1;
  for (int k = 0; k < 4; ++k) {          // of either direction and any type
    const RecCut c = rec_cut(T, N * D, D, k & 1 ? 2 : 4, k >> 1);
    if (c.segs > segs) segs = c.segs;
  }
  return segs > 1 ? (uint64_t)(segs - 1) * N * D * 8 + (uint64_t)segs * N * D * 4 : 0;
}

extern "C" int qqt_recurrence_forward(const QqtSeq* x, const QqtSeq* gate, const QqtSeq* reset,
                                      const float* h0, int32_t dtype, int64_t T, int64_t N,
                                      int64_t D, const QqtSeq* h, float* h_last, float* carry,
                                      void* work, qqt_stream_t stream) {
  if (!x || !gate || !h || !dtype_ok(dtype) || !rec_sizes_ok(T, N, D)) return QQT_E_ARG;
  if (!rec_fits(T, N, D)) return QQT_E_LIMIT;
  if (!aligned_to(work, 16)) return QQT_E_ALIGN;
  const int64_t C = N * D;
  if (C == 0) return QQT_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (T == 0) {                     // the state passes through
    if (!h_last) return QQT_OK;
    const cudaError_t e =
        h0 ? cudaMemcpyAsync(h_last, h0, (size_t)C * 4, cudaMemcpyDeviceToDevice, st)
           : cudaMemsetAsync(h_last, 0, (size_t)C * 4, st);
    return e == cudaSuccess ? QQT_OK : QQT_E_LAUNCH;
  }
  if (!x->p || !gate->p || !h->p) return QQT_E_ARG;
  RecArgs a{};
  a.x = rec_seq(x);
  a.g = rec_seq(gate);
  a.reset = rec_seq(reset);
  a.h = rec_seq(h);
  a.s0 = h0;
  a.s_end = h_last;
  a.carry = carry;
  a.nT = T;
  a.nC = (uint32_t)C;
  a.nD = (uint32_t)D;
  return with_dtype(dtype, [&](auto t) { return rec_run<decltype(t), false>(a, work, st); });
}

extern "C" int qqt_recurrence_step(const void* x, int64_t x_stride, const void* gate,
                                   int64_t gate_stride, const uint8_t* reset, int64_t reset_stride,
                                   const float* state, int32_t dtype, int64_t N, int64_t D, void* h,
                                   float* state_out, qqt_stream_t stream) {
  if (!dtype_ok(dtype) || !rec_sizes_ok(1, N, D)) return QQT_E_ARG;
  if (!rec_fits(1, N, D)) return QQT_E_LIMIT;
  if (N == 0) return QQT_OK;
  if (!x || !gate || !state || !h || !state_out) return QQT_E_ARG;
  const int64_t es = dtype == QQT_F32 ? 4 : 2, out = N * D * 4;
  if (rec_clash(state_out, out, state, N, D * 4, D * 4, true) ||
      rec_clash(state_out, out, x, N, x_stride * es, D * es,
                es == 4 && (N == 1 || x_stride == D)) ||
      rec_clash(state_out, out, gate, N, gate_stride * es, D * es,
                es == 4 && (N == 1 || gate_stride == D)) ||
      rec_clash(state_out, out, reset, N, reset_stride, 1, false) ||
      rec_clash(state_out, out, h, N, D * es, D * es, false))
    return QQT_E_ARG;
  RecArgs a{};
  a.x = RecSeq{x, 0, x_stride};
  a.g = RecSeq{gate, 0, gate_stride};
  a.reset = RecSeq{reset, 0, reset_stride};
  a.h = RecSeq{h, 0, D};
  a.s0 = state;
  a.s_end = state_out;
  a.nT = 1;
  a.nC = (uint32_t)(N * D);
  a.nD = (uint32_t)D;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    cudaStream_t st = (cudaStream_t)stream;
    if (rec_vec(a, sizeof(T)) == 4)
      k_rec_step<T, 4><<<(a.nC / 4 + 127) / 128, 128, 0, st>>>(a);
    else
      k_rec_step<T, 1><<<(a.nC + 127) / 128, 128, 0, st>>>(a);
    return launch_status();
  });
}

extern "C" int qqt_recurrence_backward(const QqtSeq* dh, const float* dh_last, const QqtSeq* x,
                                       const QqtSeq* gate, const QqtSeq* reset, const float* carry,
                                       int32_t dtype, int64_t T, int64_t N, int64_t D,
                                       const QqtSeq* dx, const QqtSeq* dgate, float* dh0, void* work,
                                       qqt_stream_t stream) {
  if (!x || !gate || !dx || !dgate || !dtype_ok(dtype) || !rec_sizes_ok(T, N, D)) return QQT_E_ARG;
  if (!rec_fits(T, N, D)) return QQT_E_LIMIT;
  if (!aligned_to(work, 16)) return QQT_E_ALIGN;
  const int64_t C = N * D;
  if (C == 0) return QQT_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (T == 0) {
    if (!dh0) return QQT_OK;
    const cudaError_t e =
        dh_last ? cudaMemcpyAsync(dh0, dh_last, (size_t)C * 4, cudaMemcpyDeviceToDevice, st)
                : cudaMemsetAsync(dh0, 0, (size_t)C * 4, st);
    return e == cudaSuccess ? QQT_OK : QQT_E_LAUNCH;
  }
  if (!x->p || !gate->p || !dx->p || !dgate->p || !carry) return QQT_E_ARG;
  RecArgs a{};
  a.x = rec_seq(x);
  a.g = rec_seq(gate);
  a.reset = rec_seq(reset);
  a.h = rec_seq(dh);
  a.dx = rec_seq(dx);
  a.dg = rec_seq(dgate);
  a.s0 = dh_last;
  a.s_end = dh0;
  a.carry = const_cast<float*>(carry);
  a.nT = T;
  a.nC = (uint32_t)C;
  a.nD = (uint32_t)D;
  return with_dtype(dtype, [&](auto t) { return rec_run<decltype(t), true>(a, work, st); });
}
