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
//
// A stretch of ticks acts on the state as h -> A h + B, and on the gradient
// that leaves it downwards as g -> A g + B', with the same A.  A block takes
// a tile of kRecChunk ticks of 32 x VEC channels ((n, d) pairs); each of its
// warps holds U ticks in registers and reduces them to (A, B), one thread per
// channel composes the warps' pairs with the state that enters the tile, and
// the warps then finish from the state that enters theirs.  A stretch that
// holds a reset has A = -0 (products of gates are +0 or more): the state
// entering it is dropped by a select, whatever it is.
//
// Two ways to get a tile's incoming state:
//  * enough channels to fill the GPU: a block walks its channels' tiles along
//    T, the next tile's loads issued before the present one is finished;
//  * few channels, many ticks: one block per tile, in the order of a ticket.
//    Tile k publishes its (A, B) at once; its incoming state is the one that
//    entered its group of kRecGroup tiles, published by the last tile of the
//    group before, composed with the pairs of the group's tiles before k --
//    always in that order, so results do not depend on timing.  A tile waits
//    only on tiles with smaller tickets, and only for kRecPolls polls.

#include "ops_common.cuh"

namespace qqt {

constexpr int kRecChunk = 64;
constexpr int kRecGroup = 32;
constexpr uint32_t kRecPolls = 1u << 22;

// f = sigmoid(g) and i = 1 - f = sigmoid(-g), each to float32 accuracy: with
// e = exp(-|g|) the larger of the two is 1/(1+e) and the smaller e/(1+e).
__device__ __forceinline__ void gates(float g, float& f, float& i) {
  const float e = expf(-fabsf(g));
  const float big = rcp_approx(1.f + e);
  const float small = e * big;
  f = g < 0.f ? small : big;
  i = g < 0.f ? big : small;
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
  float* carry;                    // state entering every kRecChunk ticks
  int64_t nT, nN, nD;
  unsigned long long* agg;         // [tiles][channels] (A, B), all ones before they are known
  unsigned* group_in;              // [groups][channels] state entering a group, ditto
  unsigned* ticket;                // -1 at first
};

// One tick for every channel: what acting does.
template <class T, int VEC>
__global__ void k_rec_step(RecArgs a) {
  const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * VEC;
  if (c >= a.nN * a.nD) return;
  const int64_t n = c / a.nD, d = c % a.nD;
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
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float f, i;
    gates(to_f(g.v[v]), f, i);
    s.v[v] = fmaf(f, s.v[v], i * to_f(x.v[v]));
    o.v[v] = from_f<T>(s.v[v]);
  }
  st_vec((T*)a.h.p + n * a.h.ns + d, o);
  if (a.s_end) st_vec(a.s_end + c, s);
}

// The gates' resets of this thread's U ticks as a bit mask.
template <int U>
__device__ __forceinline__ unsigned load_resets(const RecSeq& r, int64_t n, bool one_n, int64_t t0,
                                                int64_t nT) {
  if (!r.p) return 0;
  const uint8_t* p = (const uint8_t*)r.p + n * r.ns;
  unsigned m = 0;
  if (one_n) {                      // the whole warp follows one sequence
    const int64_t t = t0 + lane_id();
    m = __ballot_sync(QQT_FULL, lane_id() < U && t < nT && p[t * r.ts]);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t0 + u < nT && p[(t0 + u) * r.ts]) m |= 1u << u;
  }
  return m;
}

template <class T, int VEC, int U>
__device__ __forceinline__ void load_ticks(const RecSeq& s, int64_t off, int64_t t0, int64_t nT,
                                           bool on, Vec<T, VEC>* out) {
  const T* p = (const T*)s.p + off + t0 * s.ts;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (on && t0 + u < nT) {
      out[u] = ld_vec<T, VEC>(p);
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) out[u].v[v] = from_f<T>(0.f);
    }
    p += s.ts;
  }
}

__device__ __forceinline__ unsigned long long ld_poll64(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned ld_poll32(const unsigned* p) {
  unsigned v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void st_pub64(unsigned long long* p, unsigned long long v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ void st_pub32(unsigned* p, unsigned v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// The state entering tile k of channel c (tiles counted along the scan's own
// direction), composed in a fixed order from what earlier tiles published.
// Every value carries its own validity: no arithmetic result is all ones (a
// NaN comes out of the units as 0x7fffffff).
__device__ __forceinline__ float state_entering(const RecArgs& a, int64_t k, int64_t c, int64_t nC,
                                                float s0) {
  const int64_t grp = k / kRecGroup;
  const int64_t first = grp * kRecGroup;
  float s = s0;
  bool late = false;
  constexpr int B = 16;
  for (int64_t q = first; q < k; q += B) {
    unsigned long long v[B];
#pragma unroll
    for (int j = 0; j < B; ++j) v[j] = q + j < k ? ld_poll64(a.agg + (q + j) * nC + c) : 0;
    if (q == first && grp > 0) {
      unsigned w = ld_poll32(a.group_in + grp * nC + c);
      for (uint32_t i = 0; w == 0xffffffffu && i < kRecPolls; ++i)
        w = ld_poll32(a.group_in + grp * nC + c);
      late |= w == 0xffffffffu;
      s = __uint_as_float(w);
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (q + j < k) {
        for (uint32_t i = 0; v[j] == ~0ull && i < kRecPolls; ++i)
          v[j] = ld_poll64(a.agg + (q + j) * nC + c);
        late |= v[j] == ~0ull;
        s = through(__uint_as_float((unsigned)(v[j] >> 32)), __uint_as_float((unsigned)v[j]), s);
      }
    }
  }
  if (k == first && grp > 0) {
    unsigned w = ld_poll32(a.group_in + grp * nC + c);
    for (uint32_t i = 0; w == 0xffffffffu && i < kRecPolls; ++i)
      w = ld_poll32(a.group_in + grp * nC + c);
    late |= w == 0xffffffffu;
    s = __uint_as_float(w);
  }
  if (late) flag_error(QQT_DEV_TIMEOUT);
  return s;
}

// Tile (k, channel group) of this block: its ticket in split mode.
__device__ __forceinline__ int64_t take_ticket(unsigned* ticket) {
  __shared__ unsigned mine;
  if (threadIdx.x == 0) mine = atomicAdd(ticket, 1u) + 1u;
  __syncthreads();
  return mine;
}

template <class T, int VEC, int U, bool SPLIT>
__global__ void __launch_bounds__(kRecChunk / U * 32, U == 8 ? 2 : 1) k_rec_fwd(RecArgs a) {
  constexpr int W = kRecChunk / U, CH = 32 * VEC;
  __shared__ float sA[W][CH], sB[W][CH];
  const int warps = blockDim.x >> 5, w = warp_id(), lane = lane_id();
  const int64_t nC = a.nN * a.nD, nG = (nC + CH - 1) / CH;
  const int64_t nK = (a.nT + kRecChunk - 1) / kRecChunk;
  int64_t k = 0, grp = blockIdx.x;
  if (SPLIT) {
    const int64_t tk = take_ticket(a.ticket);
    k = tk / nG;
    grp = tk % nG;
  }
  const int64_t c = grp * CH + lane * VEC;
  const bool on = c < nC;
  const int64_t n = on ? c / a.nD : 0, d = on ? c % a.nD : 0;
  const bool one_n = __shfl_sync(QQT_FULL, (int)n, 0) == __shfl_sync(QQT_FULL, (int)n, 31) &&
                     __all_sync(QQT_FULL, on);
  // thread-per-channel part
  const int64_t cc = grp * CH + threadIdx.x;
  const bool mine = threadIdx.x < CH && cc < nC;
  float s = 0.f;
  // (a block of fewer than CH threads -- few ticks -- strides over its channels)
  Vec<T, VEC> x[U], g[U];
  int64_t t0 = k * kRecChunk + w * U;
  load_ticks<T, VEC, U>(a.x, n * a.x.ns + d, t0, a.nT, on, x);
  load_ticks<T, VEC, U>(a.g, n * a.g.ns + d, t0, a.nT, on, g);
  unsigned rst = load_resets<U>(a.reset, n, one_n, t0, a.nT);
  (void)mine;
  const int64_t k_end = SPLIT ? k + 1 : nK;
  for (; k < k_end; ++k) {
    float cA[U][VEC], lh[U][VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float A = 1.f, B = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f, i;
        gates(to_f(g[u].v[v]), f, i);
        const bool r = (rst >> u) & 1;
        const float na = r ? -0.f : (drops(A) ? A : A * f);
        const float nb = fmaf(f, r ? 0.f : B, i * to_f(x[u].v[v]));
        const bool in = t0 + u < a.nT;
        A = in ? na : A;
        B = in ? nb : B;
        cA[u][v] = A;
        lh[u][v] = B;
      }
      sA[w][lane * VEC + v] = A;
      sB[w][lane * VEC + v] = B;
    }
    const int64_t t_now = t0;
    if (!SPLIT && k + 1 < k_end) {
      t0 += kRecChunk;
      load_ticks<T, VEC, U>(a.x, n * a.x.ns + d, t0, a.nT, on, x);
      load_ticks<T, VEC, U>(a.g, n * a.g.ns + d, t0, a.nT, on, g);
      rst = load_resets<U>(a.reset, n, one_n, t0, a.nT);
    }
    __syncthreads();
    for (int j = threadIdx.x; j < CH; j += blockDim.x) {
      const int64_t ch = grp * CH + j;
      if (ch >= nC) break;
      if (SPLIT) {
        float A = 1.f, B = 0.f;
        for (int q = 0; q < warps; ++q) {
          B = through(sA[q][j], sB[q][j], B);
          A = drops(sA[q][j]) ? sA[q][j] : A * sA[q][j];
        }
        if (k + 1 < nK)
          st_pub64(a.agg + k * nC + ch,
                   ((unsigned long long)__float_as_uint(A) << 32) | __float_as_uint(B));
        s = state_entering(a, k, ch, nC, a.s0 ? a.s0[ch] : 0.f);
        const float out = through(A, B, s);
        if (k + 1 < nK && (k + 1) % kRecGroup == 0)
          st_pub32(a.group_in + (k + 1) / kRecGroup * nC + ch, __float_as_uint(out));
      } else if (k == 0) {
        s = a.s0 ? a.s0[ch] : 0.f;
      }
      if (a.carry) a.carry[k * nC + ch] = s;
      for (int q = 0; q < warps; ++q) {
        const float A = sA[q][j], B = sB[q][j];
        sB[q][j] = s;
        s = through(A, B, s);
      }
      if (k + 1 == nK && a.s_end) a.s_end[ch] = s;
    }
    __syncthreads();
    if (on) {
      T* hp = (T*)a.h.p + n * a.h.ns + d + t_now * a.h.ts;
      float in[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) in[v] = sB[w][lane * VEC + v];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t_now + u < a.nT) {
          Vec<T, VEC> o;
#pragma unroll
          for (int v = 0; v < VEC; ++v) o.v[v] = from_f<T>(through(cA[u][v], lh[u][v], in[v]));
          st_vec(hp, o);
        }
        hp += a.h.ts;
      }
    }
    if (!SPLIT) __syncthreads();
  }
}

template <class T, int VEC, int U, bool SPLIT>
__global__ void __launch_bounds__(kRecChunk / U * 32, U == 8 ? 2 : 1) k_rec_bwd(RecArgs a) {
  constexpr int W = kRecChunk / U, CH = 32 * VEC;
  __shared__ float sA[W][CH], sB[W][CH], sG[W][CH];
  const int warps = blockDim.x >> 5, w = warp_id(), lane = lane_id();
  const int64_t nC = a.nN * a.nD, nG = (nC + CH - 1) / CH;
  const int64_t nK = (a.nT + kRecChunk - 1) / kRecChunk;
  int64_t m = 0, grp = blockIdx.x;        // m counts tiles from the last one back
  if (SPLIT) {
    const int64_t tk = take_ticket(a.ticket);
    m = tk / nG;
    grp = tk % nG;
  }
  const int64_t c = grp * CH + lane * VEC;
  const bool on = c < nC;
  const int64_t n = on ? c / a.nD : 0, d = on ? c % a.nD : 0;
  const bool one_n = __shfl_sync(QQT_FULL, (int)n, 0) == __shfl_sync(QQT_FULL, (int)n, 31) &&
                     __all_sync(QQT_FULL, on);
  float e_in = 0.f;
  const int64_t m_end = SPLIT ? m + 1 : nK;
  for (; m < m_end; ++m) {
    const int64_t k = nK - 1 - m;
    const int64_t t0 = k * kRecChunk + w * U;
    Vec<T, VEC> x[U], g[U], dh[U];
    load_ticks<T, VEC, U>(a.x, n * a.x.ns + d, t0, a.nT, on, x);
    load_ticks<T, VEC, U>(a.g, n * a.g.ns + d, t0, a.nT, on, g);
    load_ticks<T, VEC, U>(a.h, n * a.h.ns + d, t0, a.nT, on && a.h.p, dh);
    const unsigned rst = load_resets<U>(a.reset, n, one_n, t0, a.nT);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float A = 1.f, B = 0.f, G = 0.f, f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float i;
        gates(to_f(g[u].v[v]), f[u], i);
        const bool r = (rst >> u) & 1;
        const float na = r ? -0.f : (drops(A) ? A : A * f[u]);
        const float nb = fmaf(f[u], r ? 0.f : B, i * to_f(x[u].v[v]));
        const bool in = t0 + u < a.nT;
        A = in ? na : A;
        B = in ? nb : B;
      }
#pragma unroll
      for (int u = U - 1; u >= 0; --u) {
        const float ng = (rst >> u) & 1 ? 0.f : f[u] * (to_f(dh[u].v[v]) + G);
        G = t0 + u < a.nT ? ng : G;
      }
      sA[w][lane * VEC + v] = A;
      sB[w][lane * VEC + v] = B;
      sG[w][lane * VEC + v] = G;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < CH; j += blockDim.x) {
      const int64_t ch = grp * CH + j;
      if (ch >= nC) break;
      if (SPLIT) {
        float A = 1.f, G = 0.f;
        for (int q = warps - 1; q >= 0; --q) {
          G = through(sA[q][j], sG[q][j], G);
          A = drops(sA[q][j]) ? sA[q][j] : A * sA[q][j];
        }
        if (m + 1 < nK)
          st_pub64(a.agg + m * nC + ch,
                   ((unsigned long long)__float_as_uint(A) << 32) | __float_as_uint(G));
        e_in = state_entering(a, m, ch, nC, a.s0 ? a.s0[ch] : 0.f);
        const float out = through(A, G, e_in);
        if (m + 1 < nK && (m + 1) % kRecGroup == 0)
          st_pub32(a.group_in + (m + 1) / kRecGroup * nC + ch, __float_as_uint(out));
      } else if (m == 0) {
        e_in = a.s0 ? a.s0[ch] : 0.f;
      }
      float s = a.carry[k * nC + ch];
      for (int q = 0; q < warps; ++q) {
        const float B = sB[q][j];
        sB[q][j] = s;
        s = through(sA[q][j], B, s);
      }
      for (int q = warps - 1; q >= 0; --q) {
        const float G = sG[q][j];
        sG[q][j] = e_in;
        e_in = through(sA[q][j], G, e_in);
      }
      if (k == 0 && a.s_end) a.s_end[ch] = e_in;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float f[U], i[U], prev[U];
      float s = sB[w][lane * VEC + v], acc = sG[w][lane * VEC + v];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        gates(to_f(g[u].v[v]), f[u], i[u]);
        prev[u] = (rst >> u) & 1 ? 0.f : s;
        s = fmaf(f[u], prev[u], i[u] * to_f(x[u].v[v]));
      }
#pragma unroll
      for (int u = U - 1; u >= 0; --u) {
        const bool in = t0 + u < a.nT;
        const float e = to_f(dh[u].v[v]) + acc;
        const float ie = i[u] * e;
        const float dg = f[u] * ie * (prev[u] - to_f(x[u].v[v]));
        x[u].v[v] = from_f<T>(ie);
        g[u].v[v] = from_f<T>(dg);
        acc = in ? ((rst >> u) & 1 ? 0.f : f[u] * e) : acc;
      }
    }
    if (on) {
      T* xp = (T*)a.dx.p + n * a.dx.ns + d + t0 * a.dx.ts;
      T* gp = (T*)a.dg.p + n * a.dg.ns + d + t0 * a.dg.ts;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t0 + u < a.nT) {
          st_vec(xp, x[u]);
          st_vec(gp, g[u]);
        }
        xp += a.dx.ts;
        gp += a.dg.ts;
      }
    }
    if (!SPLIT) __syncthreads();
  }
}

// Tiles of few ticks take fewer warps, so a block may have fewer threads than
// channels; the per-channel part strides over them, and only a whole block
// (blockDim >= CH) may walk several tiles with the state in a register.
static int rec_sms() {
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

struct RecWork {
  int64_t agg, group, total;       // byte offsets; the ticket is at 0
};
static RecWork rec_work(int64_t T, int64_t C) {
  const int64_t k = (T + kRecChunk - 1) / kRecChunk;
  RecWork w;
  w.agg = 16;
  w.group = w.agg + k * C * 8;
  w.total = w.group + ((k + kRecGroup - 1) / kRecGroup) * C * 4;
  return w;
}
// Split along time when one block per channel group would leave SMs without
// two blocks each and there is more than one tile to hand out.
static bool rec_split(int64_t T, int64_t C, int vec) {
  return T > kRecChunk && (C + 32 * vec - 1) / (32 * vec) < 2 * rec_sms();
}

static bool rec_sizes_ok(int64_t T, int64_t N, int64_t D) {
  return T >= 0 && N >= 0 && D > 0 && N <= 0x7fffffffll && D <= 0x7fffffffll &&
         (N == 0 || D <= 0x7fffffffll * 32 / N) && T <= 0x7fffffffll;
}
static bool seq_vec(const RecSeq& s, int64_t bytes, int64_t es) {
  return !s.p || (aligned_to(s.p, bytes) && (s.ts * es) % bytes == 0 && (s.ns * es) % bytes == 0);
}
static RecSeq rec_seq(const QqtSeq* s) {
  return s ? RecSeq{s->p, s->t_stride, s->n_stride} : RecSeq{nullptr, 0, 0};
}

template <class T, int VEC, bool BWD>
static int rec_launch(RecArgs a, void* work, cudaStream_t st) {
  constexpr int U = sizeof(T) * VEC == 16 ? 4 : 8, W = kRecChunk / U;
  const int64_t C = a.nN * a.nD, nG = (C + 32 * VEC - 1) / (32 * VEC);
  const int64_t nK = (a.nT + kRecChunk - 1) / kRecChunk;
  const int warps = a.nT >= kRecChunk ? W : (int)((a.nT + U - 1) / U);
  if (rec_split(a.nT, C, VEC)) {
    const RecWork w = rec_work(a.nT, C);
    char* base = (char*)work;
    if (!base) return QQT_E_ARG;
    if (nK * nG > 0x7fffffffll) return QQT_E_LIMIT;
    if (cudaMemsetAsync(base, 0xff, (size_t)w.total, st) != cudaSuccess) return QQT_E_LAUNCH;
    a.ticket = (unsigned*)base;
    a.agg = (unsigned long long*)(base + w.agg);
    a.group_in = (unsigned*)(base + w.group);
    if (BWD)
      k_rec_bwd<T, VEC, U, true><<<(unsigned)(nK * nG), 32 * W, 0, st>>>(a);
    else
      k_rec_fwd<T, VEC, U, true><<<(unsigned)(nK * nG), 32 * W, 0, st>>>(a);
  } else {
    if (BWD)
      k_rec_bwd<T, VEC, U, false><<<(unsigned)nG, 32 * warps, 0, st>>>(a);
    else
      k_rec_fwd<T, VEC, U, false><<<(unsigned)nG, 32 * warps, 0, st>>>(a);
  }
  return launch_status();
}

}  // namespace qqt

using namespace qqt;

extern "C" int64_t qqt_recurrence_chunks(int64_t T) {
  return T <= 0 ? 0 : (T + kRecChunk - 1) / kRecChunk;
}

extern "C" uint64_t qqt_recurrence_work_bytes(int64_t T, int64_t N, int64_t D) {
  if (!rec_sizes_ok(T, N, D) || T == 0 || N == 0) return 0;
  return rec_split(T, N * D, 1) || rec_split(T, N * D, 4) ? (uint64_t)rec_work(T, N * D).total : 0;
}

extern "C" int qqt_recurrence_forward(const QqtSeq* x, const QqtSeq* gate, const QqtSeq* reset,
                                      const float* h0, int32_t dtype, int64_t T, int64_t N,
                                      int64_t D, const QqtSeq* h, float* h_last, float* carry,
                                      void* work, qqt_stream_t stream) {
  if (!x || !gate || !h || !dtype_ok(dtype) || !rec_sizes_ok(T, N, D)) return QQT_E_ARG;
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
  a.nN = N;
  a.nD = D;
  return with_dtype(dtype, [&](auto t) {
    using E = decltype(t);
    const int64_t es = sizeof(E), vb = 4 * es;
    const bool v4 = D % 4 == 0 && seq_vec(a.x, vb, es) && seq_vec(a.g, vb, es) &&
                    seq_vec(a.h, vb, es);
    if (T == 1 && !carry && aligned_to(h0, 16) && aligned_to(h_last, 16)) {
      if (v4)
        k_rec_step<E, 4><<<(unsigned)((C / 4 + 127) / 128), 128, 0, st>>>(a);
      else
        k_rec_step<E, 1><<<(unsigned)((C + 127) / 128), 128, 0, st>>>(a);
      return launch_status();
    }
    return v4 ? rec_launch<E, 4, false>(a, work, st) : rec_launch<E, 1, false>(a, work, st);
  });
}

extern "C" int qqt_recurrence_backward(const QqtSeq* dh, const float* dh_last, const QqtSeq* x,
                                       const QqtSeq* gate, const QqtSeq* reset, const float* carry,
                                       int32_t dtype, int64_t T, int64_t N, int64_t D,
                                       const QqtSeq* dx, const QqtSeq* dgate, float* dh0, void* work,
                                       qqt_stream_t stream) {
  if (!x || !gate || !dx || !dgate || !dtype_ok(dtype) || !rec_sizes_ok(T, N, D)) return QQT_E_ARG;
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
  a.nN = N;
  a.nD = D;
  return with_dtype(dtype, [&](auto t) {
    using E = decltype(t);
    const int64_t es = sizeof(E), vb = 4 * es;
    const bool v4 = D % 4 == 0 && seq_vec(a.x, vb, es) && seq_vec(a.g, vb, es) &&
                    seq_vec(a.h, vb, es) && seq_vec(a.dx, vb, es) && seq_vec(a.dg, vb, es);
    return v4 ? rec_launch<E, 4, true>(a, work, st) : rec_launch<E, 1, true>(a, work, st);
  });
}
