// Gated linear recurrence over (B, T, C), elementwise in the C channels:
//   h_t = e^{g_t} h_{t-1} + b_t x_t,   out_t = h_t,   h_final = h_T,
// its backward pass and its step for one token.  A token with g_t = -inf starts
// anew: h_t = b_t x_t whatever h_{t-1} holds (NaN and infinities included), which
// separates the sequences of a packed batch.
//
// A run of tokens maps the state entering it to the one leaving it by h -> e^L h + H
// with L the sum of its g: two runs compose as (L1 + L2, e^{L2} H1 + H2).  L, not
// e^L, is carried, so that L = -inf says that the run holds a fresh start, and sums of
// small decays lose nothing; the mark stays whatever is added to it (a NaN or +inf in another g
// of the run would undo it, and let through what a fresh start drops).  Everything is held in
// float32.
//
// A thread takes V neighbouring channels (8- or 16-byte accesses) of 16 / V consecutive tokens:
// it composes its run in registers, the runs of a wave are composed by lane shuffles and
// the waves' through LDS, and the thread then walks its tokens again from the state that
// enters them.  The data are read once and the results written once, which bounds all of it.
//
// Short axes: a workgroup walks along the whole axis for its tile of channels, 128 tokens at a
// time, the next ones in flight meanwhile.  Long axes: every step (512 threads, 8192 values)
// has a workgroup of its own and the state is handed on through memory, in one pass over the
// data too.  Tiles are wide where there are channels enough: rows of 32 bytes, a quarter of
// a line, keep the address path busy without moving much (8 x 8192 x 768 bfloat16, walked
// in tiles of 16, 32 and 64 channels, which leave ever more CUs without work: 201, 150, 191 us;
// in steps at once 175, 125, 115).  Copies reach 5.16 TB/s on this card; these reach, forward
// and backward: 8 x 8192 x 768 bfloat16 4.4 and 5.0 TB/s, 2 x 16384 x 2048 bfloat16 4.7 and 5.0,
// 1 x 131072 x 1024 float32 without a gate forward 5.2.
//
// The backward pass needs the state before every token: the forward pass keeps the state
// that enters each step (under 1% of the data), from which the backward forms them again on
// its way from the last step to the first, so that it too reads every input once and never
// reads the outputs.
#include <limits.h>

#include "gdn2.h"
#include "gdn2_common.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;  // of the elementwise kernels
constexpr int kMinTile = 16;   // channels of the narrowest workgroup
constexpr float kLog2e = 1.44269504088896340736f;

// Strides are in elements; channels are contiguous.
struct Rows {
  const void* p;
  long long sb, st;
};
struct ScanArgs {
  Rows x, g, b, dout;
  const float* h0;        // (B, C) or null
  const float* dh_final;  // (B, C) or null
  void *out, *dx, *dg, *db;            // (B, T, C) dense
  float *h_final, *dh0;                // (B, C)
  float* kept;                         // (steps, B, C) or null
  void* ws;
  int B, T, C, nct;                    // nct: channel tiles
  int chunk;                           // work items of one XCD
};

// exp2 of a sum of g in units of log2(e).
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kNegInf = -__builtin_inff();

// e^l h + u, or u alone where l = -inf.
__device__ __forceinline__ float carry_through(float l, float h, float u) {
  return l == kNegInf ? u : fmaf(exp2_(l), h, u);
}
// L of two runs together.
__device__ __forceinline__ float sum_decays(float l0, float l1) {
  return l0 == kNegInf || l1 == kNegInf ? kNegInf : l0 + l1;
}

template <typename T, int V> struct Raw;
template <> struct Raw<float, 4> { using type = f32x4; };
template <> struct Raw<bf16_t, 4> { using type = bf16x4; };
template <> struct Raw<float, 1> { using type = float; };
template <> struct Raw<bf16_t, 1> { using type = bf16_t; };

template <typename T, int V>
__device__ __forceinline__ void widen(const typename Raw<T, V>::type& r, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = (float)r;
  } else {
#pragma unroll
    for (int c = 0; c < V; ++c) f[c] = (float)r[c];
  }
}
template <typename T, int V>
__device__ __forceinline__ void put(T* p, const float (&f)[V]) {
  if constexpr (V == 1) {
    *p = (T)f[0];
  } else {
    typename Raw<T, V>::type r;
#pragma unroll
    for (int c = 0; c < V; ++c) r[c] = (T)f[c];
    *reinterpret_cast<typename Raw<T, V>::type*>(p) = r;
  }
}

// Where a workgroup and a thread work: NT threads, CT channels, V neighbouring ones a
// thread, 16 values of a step for each.
template <int V, int CT, int NT_>
struct Place {
  static constexpr int NT = NT_, NW = NT / 64;       // threads, waves
  static constexpr int BLOCK = 16 * NT / CT;         // tokens of a step
  static constexpr int LPR = CT / V;                 // lanes across the channels
  static constexpr int TLW = 64 / LPR;               // runs of a wave
  static constexpr int S = 16 / V;                   // tokens of a run
  static_assert(LPR <= 64 && TLW * NW * S == BLOCK, "a step is the workgroup's runs");
  int lane, wave, tl, ci, c, b;
  bool on;       // the channels exist
  bool idle;     // the workgroup has no work
  int blocks;    // steps of the axis
  __device__ Place(const ScanArgs& a) {
    // neighbouring channel tiles share cache lines: consecutive items on one XCD
    const int unit = (blockIdx.x & 7) * a.chunk + (blockIdx.x >> 3);
    idle = (int)(blockIdx.x >> 3) >= a.chunk || unit >= a.B * a.nct;
    b = unit / a.nct;
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    tl = lane / LPR;
    ci = (lane % LPR) * V;
    c = (unit - b * a.nct) * CT + ci;
    on = c < a.C;
    if (!on) c = 0;   // loads stay in bounds, nothing is stored
    blocks = (a.T + BLOCK - 1) / BLOCK;
  }
  // first token of the thread's run in step blk
  __device__ int first(int blk) const { return blk * BLOCK + (wave * TLW + tl) * S; }
  __device__ size_t bc(const ScanArgs& a) const { return (size_t)b * a.C + c; }
};

// The rows of a run; tokens past the end repeat the last one and are neutralised later.
template <typename T, int V, int S>
struct Run {
  typename Raw<T, V>::type r[S];
  __device__ __forceinline__ void load(const Rows& m, int b, int c, int t, int T_len) {
    const T* p = (const T*)m.p + (long long)b * m.sb + c;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int ti = t + i < T_len ? t + i : T_len - 1;
      r[i] = *reinterpret_cast<const typename Raw<T, V>::type*>(p + (long long)ti * m.st);
    }
  }
};
struct None {};

// Compose (L, H) of the runs of a wave: on return (L, H) is the composition of the runs
// before this one (identity for the first), (TL, TH) that of all, valid in the last run's
// lanes.  REV: of the runs after this one, all valid in the first run's lanes.
template <int V, int LPR, bool REV>
__device__ __forceinline__ void wave_compose(float (&L)[V], float (&H)[V], float (&TL)[V],
                                             float (&TH)[V], int lane) {
  const int place = REV ? 63 - lane : lane;   // lanes already passed in scan order
#pragma unroll
  for (int m = LPR; m < 64; m *= 2) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float l = REV ? __shfl_down(L[c], m) : __shfl_up(L[c], m);
      const float h = REV ? __shfl_down(H[c], m) : __shfl_up(H[c], m);
      if (place >= m) {
        H[c] = carry_through(L[c], h, H[c]);
        L[c] = sum_decays(L[c], l);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    TL[c] = L[c];
    TH[c] = H[c];
    const float l = REV ? __shfl_down(L[c], LPR) : __shfl_up(L[c], LPR);
    const float h = REV ? __shfl_down(H[c], LPR) : __shfl_up(H[c], LPR);
    L[c] = place >= LPR ? l : 0.f;
    H[c] = place >= LPR ? h : 0.f;
  }
}

// Factors and inputs of a run: a = e^g (negative for a fresh start), u = b x; L and H of
// the run.  Tokens from T on are neutral (a = 1, u = 0).
template <int V, int S>
struct Factors {
  float a[S][V], u[S][V], L[V], H[V];
};
template <typename TX, typename TG, bool GATE, int V, int S, typename RB>
__device__ __forceinline__ void factors(Factors<V, S>& f, const Run<TX, V, S>& x,
                                        const Run<TG, V, S>& g, const RB& b, int t, int T_len) {
#pragma unroll
  for (int c = 0; c < V; ++c) f.L[c] = f.H[c] = 0.f;
  bool started[V] = {};
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const bool real = t + i < T_len;
    float gv[V], xv[V], bv[V];
    widen<TG, V>(g.r[i], gv);
    widen<TX, V>(x.r[i], xv);
    if constexpr (GATE) widen<TX, V>(b.r[i], bv);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float l = real ? gv[c] * kLog2e : 0.f;
      const bool anew = l == kNegInf;
      const float in = GATE ? bv[c] * xv[c] : xv[c];
      f.u[i][c] = real ? in : 0.f;
      f.a[i][c] = anew ? -1.f : exp2_(l);
      f.H[c] = fmaf(f.a[i][c], anew ? 0.f : f.H[c], f.u[i][c]);
      f.L[c] += l;
      started[c] |= anew;
    }
  }
#pragma unroll
  for (int c = 0; c < V; ++c)
    if (started[c]) f.L[c] = kNegInf;
}
// a h + u for one token of a run.
__device__ __forceinline__ float token(float a, float h, float u) {
  return fmaf(a, a < 0.f ? 0.f : h, u);
}

// A wave's composition in LDS: e^L (negative for a fresh start), and H or D.
template <int NW, int CT>
struct Totals {
  float a[2][NW][CT], h[2][NW][CT];   // two buffers: one barrier a step
  template <int V>
  __device__ __forceinline__ void put_(int buf, int wave, int ci, const float (&L)[V],
                                       const float (&H)[V]) {
    float f[V];
#pragma unroll
    for (int c = 0; c < V; ++c) f[c] = L[c] == kNegInf ? -1.f : exp2_(L[c]);
    put<float, V>(&a[buf][wave][ci], f);
    put<float, V>(&h[buf][wave][ci], H);
  }
  // h <- e^L h + H of wave k
  template <int V>
  __device__ __forceinline__ void pass(int buf, int k, int ci, float (&x)[V]) const {
    const auto av = *reinterpret_cast<const typename Raw<float, V>::type*>(&a[buf][k][ci]);
    const auto hv = *reinterpret_cast<const typename Raw<float, V>::type*>(&h[buf][k][ci]);
    float af[V], hf[V];
    widen<float, V>(av, af);
    widen<float, V>(hv, hf);
#pragma unroll
    for (int c = 0; c < V; ++c) x[c] = fmaf(af[c], af[c] < 0.f ? 0.f : x[c], hf[c]);
  }
};

// Forward.
template <typename TX, typename TG, bool GATE, int V, int CT>
__global__ void __launch_bounds__(8 * CT) gscan_fwd(ScanArgs a) {
  using P = Place<V, CT, 8 * CT>;
  constexpr int S = P::S, LPR = P::LPR, NW = P::NW;
  __shared__ __attribute__((aligned(16))) Totals<NW, CT> tot;
  const P w(a);
  if (w.idle) return;
  float h[V];
#pragma unroll
  for (int c = 0; c < V; ++c) h[c] = a.h0 ? a.h0[w.bc(a) + c] : 0.f;
  Run<TX, V, S> x;
  Run<TG, V, S> g;
  std::conditional_t<GATE, Run<TX, V, S>, None> b;
  auto load = [&](int blk) {
    const int t = w.first(blk);
    x.load(a.x, w.b, w.c, t, a.T);
    g.load(a.g, w.b, w.c, t, a.T);
    if constexpr (GATE) b.load(a.b, w.b, w.c, t, a.T);
  };
  load(0);
  for (int blk = 0; blk < w.blocks; ++blk) {
    const int t = w.first(blk);
    Factors<V, S> f;
    factors<TX, TG, GATE, V, S>(f, x, g, b, t, a.T);
    if (blk + 1 < w.blocks) load(blk + 1);
    float L[V], H[V], TL[V], TH[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      L[c] = f.L[c];
      H[c] = f.H[c];
    }
    wave_compose<V, LPR, false>(L, H, TL, TH, w.lane);
    const int buf = blk & 1;
    if (w.lane >= 64 - LPR) tot.template put_<V>(buf, w.wave, w.ci, TL, TH);
    if (a.kept && w.on && w.wave == 0 && w.tl == 0)
      put<float, V>(a.kept + (size_t)blk * a.B * a.C + w.bc(a), h);
    lds_barrier();   // the other buffer is written next: one barrier a step
    float mine[V];
#pragma unroll
    for (int c = 0; c < V; ++c) mine[c] = h[c];
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      if (k == w.wave)
#pragma unroll
        for (int c = 0; c < V; ++c) mine[c] = h[c];
      tot.template pass<V>(buf, k, w.ci, h);
    }
#pragma unroll
    for (int c = 0; c < V; ++c) mine[c] = carry_through(L[c], mine[c], H[c]);
    TX* out = (TX*)a.out + (long long)w.b * a.T * a.C + w.c;
#pragma unroll
    for (int i = 0; i < S; ++i) {
#pragma unroll
      for (int c = 0; c < V; ++c) mine[c] = token(f.a[i][c], mine[c], f.u[i][c]);
      if (w.on && t + i < a.T) put<TX, V>(out + (long long)(t + i) * a.C, mine);
    }
  }
  if (w.on && w.wave == 0 && w.tl == 0) put<float, V>(a.h_final + w.bc(a), h);
}

// Backward.  With e the gradient that reaches the state after token t from later tokens
// (dh_final after the last): dh = dout_t + e, dx = b dh, db = x dh, dg = a h_{t-1} dh,
// and a dh goes on to the token before; a run maps the e entering it from the right to
// e^L e + D.
template <typename TX, typename TG, bool GATE, int V, int CT>
__global__ void __launch_bounds__(8 * CT) gscan_bwd(ScanArgs a) {
  using P = Place<V, CT, 8 * CT>;
  constexpr int S = P::S, LPR = P::LPR, NW = P::NW;
  __shared__ __attribute__((aligned(16))) Totals<NW, CT> fwd, rev;
  const P w(a);
  if (w.idle) return;
  float e[V];
#pragma unroll
  for (int c = 0; c < V; ++c) e[c] = a.dh_final ? a.dh_final[w.bc(a) + c] : 0.f;
  const bool has_dout = a.dout.p != nullptr;
  Run<TX, V, S> x, d;
  Run<TG, V, S> g;
  std::conditional_t<GATE, Run<TX, V, S>, None> b;
  float h[V];
#pragma unroll
  for (int c = 0; c < V; ++c) h[c] = 0.f;
  auto load = [&](int blk) {
    const int t = w.first(blk);
    g.load(a.g, w.b, w.c, t, a.T);
    if (has_dout) d.load(a.dout, w.b, w.c, t, a.T);
    x.load(a.x, w.b, w.c, t, a.T);
    if constexpr (GATE) b.load(a.b, w.b, w.c, t, a.T);
#pragma unroll
    for (int c = 0; c < V; ++c) h[c] = a.kept[(size_t)blk * a.B * a.C + w.bc(a) + c];
  };
  load(w.blocks - 1);
  for (int blk = w.blocks - 1; blk >= 0; --blk) {
    const int t = w.first(blk);
    Factors<V, S> f;
    float xv[S][V], bv[S][V], dv[S][V], hw[V];
    factors<TX, TG, GATE, V, S>(f, x, g, b, t, a.T);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      widen<TX, V>(x.r[i], xv[i]);
      if constexpr (GATE) widen<TX, V>(b.r[i], bv[i]);
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if (has_dout) widen<TX, V>(d.r[i], dv[i]);
#pragma unroll
      for (int c = 0; c < V; ++c)
        if (!has_dout || t + i >= a.T) dv[i][c] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < V; ++c) hw[c] = h[c];
    if (blk > 0) load(blk - 1);
    float L[V], H[V], R[V], D[V], TL[V], TH[V], TD[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      D[c] = 0.f;
#pragma unroll
      for (int i = S - 1; i >= 0; --i)
        D[c] = f.a[i][c] < 0.f ? 0.f : f.a[i][c] * (dv[i][c] + D[c]);
      R[c] = L[c] = f.L[c];
      H[c] = f.H[c];
    }
    const int buf = blk & 1;
    wave_compose<V, LPR, false>(L, H, TL, TH, w.lane);
    if (w.lane >= 64 - LPR) fwd.template put_<V>(buf, w.wave, w.ci, TL, TH);
    wave_compose<V, LPR, true>(R, D, TL, TD, w.lane);
    if (w.lane < LPR) rev.template put_<V>(buf, w.wave, w.ci, TL, TD);
    lds_barrier();
    float mine[V];
#pragma unroll
    for (int c = 0; c < V; ++c) mine[c] = e[c];
#pragma unroll
    for (int k = NW - 1; k >= 0; --k) {
      if (k == w.wave)
#pragma unroll
        for (int c = 0; c < V; ++c) mine[c] = e[c];
      rev.template pass<V>(buf, k, w.ci, e);
    }
#pragma unroll
    for (int k = 0; k < NW - 1; ++k)
      if (k < w.wave) fwd.template pass<V>(buf, k, w.ci, hw);
    float before[S][V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      float hc = carry_through(L[c], hw[c], H[c]);
      mine[c] = carry_through(R[c], mine[c], D[c]);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        before[i][c] = hc;
        hc = token(f.a[i][c], hc, f.u[i][c]);
      }
    }
    const long long o = (long long)w.b * a.T * a.C + w.c;
#pragma unroll
    for (int i = S - 1; i >= 0; --i) {
      float dx[V], dg[V], db[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float dh = dv[i][c] + mine[c], av = f.a[i][c];
        mine[c] = av < 0.f ? 0.f : av * dh;
        dg[c] = av < 0.f ? 0.f : mine[c] * before[i][c];
        dx[c] = GATE ? bv[i][c] * dh : dh;
        db[c] = xv[i][c] * dh;
      }
      if (w.on && t + i < a.T) {
        const long long at = o + (long long)(t + i) * a.C;
        put<TX, V>((TX*)a.dx + at, dx);
        put<TG, V>((TG*)a.dg + at, dg);
        if constexpr (GATE) put<TX, V>((TX*)a.db + at, db);
      }
    }
  }
  if (w.on && w.wave == 0 && w.tl == 0 && a.dh0) put<float, V>(a.dh0 + w.bc(a), e);
}

// ---- The axis cut into its steps, all in one launch --------------------------------
// (The published single-pass scan with decoupled look-back, Merrill and Garland 2016, its
// order of service by tickets.)
// A workgroup takes 128 tokens of 64 channels (or 256 of 32, 512 of 16).  It publishes its
// composition as soon as it has it, finds the state that enters it from the steps before,
// and publishes the one that leaves it.  Steps are dealt by a ticket, the earliest of all
// tiles first (or, each tile with tickets of its own, the earliest of the tile): a workgroup
// waits only for ones with smaller tickets, which have started and which in their turn never
// wait for it, so every wait ends whatever else the GPU runs.
// The entering state is always the same sequence of operations -- the nearest published
// state, carried through the published compositions after it, each rounded the same wherever
// it is done -- so results do not depend on what was found first.
//
// What a step has published is 64 bits, written at once: first {e^L, H} (e^L = -1 for a fresh
// start), then {kState, state}; before, the clearing kernel's kNone.
constexpr unsigned long long kNone = ~0ull;
constexpr float kState = -2.f;
// Steps looked back over at a time: 8 where the registers allow (1 x 131072 x 1024 float32
// forward 313 us, with 4 345); the backward has none to spare (8 x 8192 x 768 bfloat16 250 us,
// with 4 194).  Even so its gated forms do not fit the 128 registers of two workgroups a CU and
// keep 8 to 36 bytes a lane in scratch memory (12 there: 37 MB read and 31 written beyond the
// operands' 503 and 403), as do gated bfloat16 forwards with one channel a thread (12 to 20).
template <bool REV> constexpr int kWindow = REV ? 4 : 8;
constexpr int kTicketStride = 16; // tickets of different tiles on cache lines of their own
struct Chain {
  unsigned long long* slot;       // (steps, B, C)
  unsigned* ticket;               // (B tiles) kTicketStride; counted from -1, as cleared
  int own;                        // each tile draws from its own
};

__device__ __forceinline__ unsigned long long pack(float hi, float lo) {
  return ((unsigned long long)__float_as_uint(hi) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ float upper(unsigned long long v) {
  return __uint_as_float((unsigned)(v >> 32));
}
__device__ __forceinline__ float lower(unsigned long long v) { return __uint_as_float((unsigned)v); }
__device__ __forceinline__ void publish(unsigned long long* p, float hi, float lo) {
  __hip_atomic_store(p, pack(hi, lo), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// h through a composition (a = e^L, negative for a fresh start)
__device__ __forceinline__ float through(float a, float h, float u) {
  return fmaf(a, a < 0.f ? 0.f : h, u);
}

// The state that enters step blk (REV: from the right), not the first, for one channel a lane.
// at: the channel's place; on: it exists.  The first step publishes no composition, only its
// state, so nothing beyond it is ever looked for, and it alone reads h0 (REV: dh_final), which
// the last step may overwrite as soon as it has found a state.
template <bool REV>
__device__ __forceinline__ float entering(const Chain& ch, size_t n, size_t at, bool on, int blk,
                                          int blocks) {
  while (true) {
    unsigned long long v[kWindow<REV>];
#pragma unroll
    for (int d = 0; d < kWindow<REV>; ++d) {
      const int j = REV ? blk + 1 + d : blk - 1 - d;
      const bool in = REV ? j < blocks : j >= 0;
      v[d] = __hip_atomic_load(ch.slot + (size_t)(in ? j : blk) * n + at, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
      if (!in || !on) v[d] = pack(kState, 0.f);
    }
    int found = -1;   // the nearest state with nothing missing before it
#pragma unroll
    for (int d = 0; d < kWindow<REV>; ++d)
      if (found == -1) found = upper(v[d]) == kState ? d : v[d] == kNone ? -2 : -1;
    if (__all(found >= 0)) {
      float h = 0.f;
#pragma unroll
      for (int d = kWindow<REV> - 1; d >= 0; --d)
        if (d <= found) h = d == found ? lower(v[d]) : through(upper(v[d]), h, lower(v[d]));
      return h;
    }
    __builtin_amdgcn_s_sleep(2);
  }
}

// One wave, a channel a lane: publish the workgroup's composition, find the entering state
// (start's, or zero, for the first step), publish the leaving one.  Returns both.
template <bool REV, int NW, int CT>
__device__ __forceinline__ void link(const Chain& ch, const Totals<NW, CT>& tot, size_t n,
                                     size_t at, bool on, int blk, int blocks, const float* start,
                                     int lane, float& in, float& out) {
  float A = 1.f, H = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int k = REV ? NW - 1 - i : i;
    const float ak = tot.a[0][k][lane % CT], hk = tot.h[0][k][lane % CT];
    H = through(ak, H, hk);
    A = ak < 0.f || A < 0.f ? -1.f : A * ak;
  }
  if (A != A) A = __uint_as_float(0x7fc00000u);   // any NaN but kNone's
  // the steps after this one, if any, read these
  const bool first = REV ? blk == blocks - 1 : blk == 0, last = REV ? blk == 0 : blk == blocks - 1;
  unsigned long long* slot = ch.slot + (size_t)blk * n + at;
  if (!last && !first && on) publish(slot, A, H);
  in = !first ? entering<REV>(ch, n, at, on, blk, blocks) : start && on ? start[at] : 0.f;
  out = through(A, in, H);
  if (!last && on) publish(slot, kState, out);
}

// A workgroup's tile and step, by the ticket that its first thread draws.
__device__ __forceinline__ int draw(const ScanArgs& a, const Chain& ch, int* shared) {
  if (threadIdx.x == 0) {
    const int units = a.B * a.nct;
    if (ch.own) {
      const int unit = (int)(blockIdx.x % (unsigned)units);
      *shared = (int)(atomicAdd(ch.ticket + unit * kTicketStride, 1u) + 1u) * units + unit;
    } else {
      *shared = (int)(atomicAdd(ch.ticket, 1u) + 1u);
    }
  }
  __syncthreads();
  return *shared;
}
template <int V, int CT>
struct Step : Place<V, CT, 512> {
  int unit, blk;
  __device__ Step(const ScanArgs& a, int item, bool rev) : Place<V, CT, 512>(a) {
    const int units = a.B * a.nct;
    blk = item / units;
    unit = item - blk * units;
    if (rev) blk = this->blocks - 1 - blk;
    this->b = unit / a.nct;
    this->c = (unit - this->b * a.nct) * CT + this->ci;
    this->on = this->c < a.C;
    if (!this->on) this->c = 0;
  }
  // The channel of a lane of the wave that links, and C where the tile is narrower.
  __device__ int lane_channel(const ScanArgs& a) const {
    return this->lane < CT ? unit % a.nct * CT + this->lane : a.C;
  }
};

__global__ void __launch_bounds__(kThreads) chain_clear(uint4* p, size_t n) {
  const size_t stride = (size_t)gridDim.x * kThreads;
  for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += stride)
    p[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

template <typename TX, typename TG, bool GATE, int V, int CT>
__global__ void __launch_bounds__(512, 4) chain_fwd(ScanArgs a, Chain ch) {
  using P = Place<V, CT, 512>;
  constexpr int S = P::S, LPR = P::LPR, NW = P::NW;
  __shared__ __attribute__((aligned(16))) Totals<NW, CT> tot;
  __shared__ __attribute__((aligned(16))) float s_in[CT];
  __shared__ int s_ticket;
  const Step<V, CT> w(a, draw(a, ch, &s_ticket), false);
  Run<TX, V, S> x;
  Run<TG, V, S> g;
  std::conditional_t<GATE, Run<TX, V, S>, None> b;
  const int t = w.first(w.blk);
  g.load(a.g, w.b, w.c, t, a.T);
  x.load(a.x, w.b, w.c, t, a.T);
  if constexpr (GATE) b.load(a.b, w.b, w.c, t, a.T);
  Factors<V, S> f;
  factors<TX, TG, GATE, V, S>(f, x, g, b, t, a.T);
  float L[V], H[V], TL[V], TH[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    L[c] = f.L[c];
    H[c] = f.H[c];
  }
  wave_compose<V, LPR, false>(L, H, TL, TH, w.lane);
  if (w.lane >= 64 - LPR) tot.template put_<V>(0, w.wave, w.ci, TL, TH);
  lds_barrier();
  if (w.wave == 0) {
    // lane = channel of the tile
    const int unit_c = w.lane_channel(a);
    const bool on = unit_c < a.C;
    const size_t n = (size_t)a.B * a.C, at = (size_t)w.b * a.C + (on ? unit_c : 0);
    float in, out;
    link<false, NW, CT>(ch, tot, n, at, on, w.blk, w.blocks, a.h0, w.lane, in, out);
    if (w.lane < CT) s_in[w.lane] = in;
    if (on && a.kept) a.kept[(size_t)w.blk * n + at] = in;
    if (on && w.blk == w.blocks - 1) a.h_final[at] = out;
  }
  lds_barrier();
  float mine[V];
#pragma unroll
  for (int c = 0; c < V; ++c) mine[c] = s_in[w.ci + c];
#pragma unroll
  for (int k = 0; k < NW - 1; ++k)
    if (k < w.wave) tot.template pass<V>(0, k, w.ci, mine);
#pragma unroll
  for (int c = 0; c < V; ++c) mine[c] = carry_through(L[c], mine[c], H[c]);
  TX* out = (TX*)a.out + (long long)w.b * a.T * a.C + w.c;
#pragma unroll
  for (int i = 0; i < S; ++i) {
#pragma unroll
    for (int c = 0; c < V; ++c) mine[c] = token(f.a[i][c], mine[c], f.u[i][c]);
    if (w.on && t + i < a.T) put<TX, V>(out + (long long)(t + i) * a.C, mine);
  }
}

template <typename TX, typename TG, bool GATE, int V, int CT>
__global__ void __launch_bounds__(512, 4) chain_bwd(ScanArgs a, Chain ch) {
  using P = Place<V, CT, 512>;
  constexpr int S = P::S, LPR = P::LPR, NW = P::NW;
  __shared__ __attribute__((aligned(16))) Totals<NW, CT> fwd, rev;
  __shared__ __attribute__((aligned(16))) float s_in[CT];
  __shared__ int s_ticket;
  const Step<V, CT> w(a, draw(a, ch, &s_ticket), true);
  const bool has_dout = a.dout.p != nullptr;
  Run<TX, V, S> x, d;
  Run<TG, V, S> g;
  std::conditional_t<GATE, Run<TX, V, S>, None> b;
  const int t = w.first(w.blk);
  g.load(a.g, w.b, w.c, t, a.T);
  if (has_dout) d.load(a.dout, w.b, w.c, t, a.T);
  x.load(a.x, w.b, w.c, t, a.T);
  if constexpr (GATE) b.load(a.b, w.b, w.c, t, a.T);
  float hw[V];
#pragma unroll
  for (int c = 0; c < V; ++c) hw[c] = a.kept[(size_t)w.blk * a.B * a.C + w.bc(a) + c];
  Factors<V, S> f;
  factors<TX, TG, GATE, V, S>(f, x, g, b, t, a.T);
  float dv[S][V];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    if (has_dout) widen<TX, V>(d.r[i], dv[i]);
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (!has_dout || t + i >= a.T) dv[i][c] = 0.f;
  }
  float L[V], H[V], R[V], D[V], TL[V], TH[V], TD[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    D[c] = 0.f;
#pragma unroll
    for (int i = S - 1; i >= 0; --i)
      D[c] = f.a[i][c] < 0.f ? 0.f : f.a[i][c] * (dv[i][c] + D[c]);
    R[c] = L[c] = f.L[c];
    H[c] = f.H[c];
  }
  wave_compose<V, LPR, true>(R, D, TL, TD, w.lane);
  if (w.lane < LPR) rev.template put_<V>(0, w.wave, w.ci, TL, TD);
  wave_compose<V, LPR, false>(L, H, TL, TH, w.lane);
  if (w.lane >= 64 - LPR) fwd.template put_<V>(0, w.wave, w.ci, TL, TH);
  lds_barrier();
  if (w.wave == 0) {
    const int unit_c = w.lane_channel(a);
    const bool on = unit_c < a.C;
    const size_t n = (size_t)a.B * a.C, at = (size_t)w.b * a.C + (on ? unit_c : 0);
    float in, out;
    link<true, NW, CT>(ch, rev, n, at, on, w.blk, w.blocks, a.dh_final, w.lane, in, out);
    if (w.lane < CT) s_in[w.lane] = in;
    if (on && w.blk == 0 && a.dh0) a.dh0[at] = out;
  }
  // meanwhile the other waves form the states before their tokens
  float before[S][V];
#pragma unroll
  for (int k = 0; k < NW - 1; ++k)
    if (k < w.wave) fwd.template pass<V>(0, k, w.ci, hw);
#pragma unroll
  for (int c = 0; c < V; ++c) hw[c] = carry_through(L[c], hw[c], H[c]);
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float xv[V], bv[V];   // b x once more: kept, it would not fit the registers
    widen<TX, V>(x.r[i], xv);
    if constexpr (GATE) widen<TX, V>(b.r[i], bv);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      before[i][c] = hw[c];
      hw[c] = token(f.a[i][c], hw[c], GATE ? bv[c] * xv[c] : xv[c]);
    }
  }
  lds_barrier();
  float mine[V];
#pragma unroll
  for (int c = 0; c < V; ++c) mine[c] = s_in[w.ci + c];
#pragma unroll
  for (int k = NW - 1; k > 0; --k)
    if (k > w.wave) rev.template pass<V>(0, k, w.ci, mine);
#pragma unroll
  for (int c = 0; c < V; ++c) mine[c] = carry_through(R[c], mine[c], D[c]);
  const long long o = (long long)w.b * a.T * a.C + w.c;
#pragma unroll
  for (int i = S - 1; i >= 0; --i) {
    float dx[V], dg[V], db[V], xv[V], bv[V];
    widen<TX, V>(x.r[i], xv);
    if constexpr (GATE) widen<TX, V>(b.r[i], bv);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float dh = dv[i][c] + mine[c], av = f.a[i][c];
      mine[c] = av < 0.f ? 0.f : av * dh;
      dg[c] = av < 0.f ? 0.f : mine[c] * before[i][c];
      dx[c] = GATE ? bv[c] * dh : dh;
      db[c] = xv[c] * dh;
    }
    if (w.on && t + i < a.T) {
      const long long at = o + (long long)(t + i) * a.C;
      put<TX, V>((TX*)a.dx + at, dx);
      put<TG, V>((TG*)a.dg + at, dg);
      if constexpr (GATE) put<TX, V>((TX*)a.db + at, db);
    }
  }
}

// One token: elementwise on n = B C values.
template <typename TX, typename TG, bool GATE, int V>
__global__ void __launch_bounds__(kThreads) gscan_step(size_t n, const TX* x, const TG* g,
                                                       const TX* b, const float* h_in,
                                                       float* h_out, TX* out) {
  for (size_t i = ((size_t)blockIdx.x * kThreads + threadIdx.x) * V; i < n;
       i += (size_t)gridDim.x * kThreads * V) {
    float xv[V], gv[V], bv[V], h[V];
    widen<TX, V>(*reinterpret_cast<const typename Raw<TX, V>::type*>(x + i), xv);
    widen<TG, V>(*reinterpret_cast<const typename Raw<TG, V>::type*>(g + i), gv);
    if constexpr (GATE) widen<TX, V>(*reinterpret_cast<const typename Raw<TX, V>::type*>(b + i), bv);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float u = GATE ? bv[c] * xv[c] : xv[c];
      h[c] = carry_through(gv[c] * kLog2e, h_in ? h_in[i + c] : 0.f, u);
    }
    put<float, V>(h_out + i, h);
    put<TX, V>(out + i, h);
  }
}

// No token: the state passes through.
__global__ void __launch_bounds__(kThreads) gscan_none(size_t n, const float* h_in, float* h_out) {
  const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
  if (i < n) h_out[i] = h_in ? h_in[i] : 0.f;
}

// ---------------------------------------------------------------- host side

size_t ticket_bytes(int units) { return (size_t)units * kTicketStride * sizeof(unsigned); }

// How a call is spread over the GPU: a walk along the axis by workgroups of ct channels, or
// (chain) all steps at once.
struct Split {
  bool chain;
  int ct, nct;
  int block, blocks;   // tokens of a step, steps
  size_t ws;
};
Split split(int B, int T, int C, int in_dtype) {
  Split s;
  auto units = [&](int ct) { return (long long)B * ((C + ct - 1) / ct); };
  auto cut = [&](bool chain, int ct) {
    s.chain = chain;
    s.ct = ct;
    s.nct = (C + ct - 1) / ct;
    s.block = chain ? 16 * 512 / ct : 128;
    s.blocks = T / s.block + (T % s.block != 0);
    s.ws = chain ? ticket_bytes(B * s.nct) + ((size_t)s.blocks * B * C * 8 + 15) / 16 * 16 : 0;
  };
  // Short axes: one launch, no ticket.  16 x 512 x 1024 bfloat16 forward and backward 18 and 35
  // us, in steps at once 27 and 38; 16 x 2048 x 4096 303 and 582, in steps at once 289 and 510.
  if (T <= 512 || (T <= 1024 && units(64) >= 256)) {
    cut(false, units(64) >= 192 ? 64 : 16);
    return s;
  }
  // Rows of a tile fill a 128-byte line.  With few channels the time goes by the hand-over from
  // step to step (about 1.1 us for a window of them) and narrower tiles have longer steps: bfloat16
  // forward and backward 8 x 8192 x 768 in tiles of 64 and 32 channels 115 + 196 and 125 + 215 us,
  // 1 x 65536 x 768 124 + 206 and 128 + 211, 1 x 16384 x 128 27 + 37 and 18 + 26; float32
  // 8 x 4096 x 768 88 + 147 and 87 + 148, 1 x 32768 x 256 58 + 79 and 40 + 56.  In tiles of 32
  // and 16 bfloat16 1 x 131072 x 128 95 + 136 and 65 + 113, 1 x 100000 x 77 80 + 105 and 53 + 70,
  // but 2 x 60000 x 100 59 + 84 and 62 + 97, 1 x 16384 x 128 18.3 + 36.2 and 19.3 + 36.9.
  const long long all = (long long)B * C;
  cut(true, all <= 128 && T > 32768 ? 16 : in_dtype == GDN2_BF16 && all >= 1024 ? 64 : 32);
  if (s.blocks * units(s.ct) >= (1ll << 22)) cut(false, 64);   // a grid's threads: 32 bits
  return s;
}

int validate(int B, int T, int C, int in_dtype, int g_dtype) {
  if (B < 1 || C < 1 || T < 0) return GDN2_ERR_SHAPE;
  if (in_dtype != GDN2_F32 && in_dtype != GDN2_BF16) return GDN2_ERR_DTYPE;
  if (g_dtype != GDN2_F32 && !(g_dtype == GDN2_BF16 && in_dtype == GDN2_BF16))
    return GDN2_ERR_DTYPE;
  if (T > INT_MAX - 512 || C > INT_MAX - 64) return GDN2_ERR_SHAPE;
  // a launch's threads (up to 512 for 16 channels) within 32 bits, bytes of a tensor within 62
  if ((double)B * ((C + kMinTile - 1) / kMinTile) > 8.0e6) return GDN2_ERR_SHAPE;
  if ((double)B * T * C > 1e18) return GDN2_ERR_SHAPE;
  return GDN2_OK;
}

// A row operand: element-aligned, and whether 4-channel accesses fit it.
int check_rows(const Rows& r, int dtype, bool* vec) {
  const uintptr_t e = dtype == GDN2_F32 ? 4 : 2;
  if (!r.p) return GDN2_ERR_NULL;
  if ((uintptr_t)r.p % e) return GDN2_ERR_ALIGN;
  if ((uintptr_t)r.p % (4 * e) || r.sb % 4 || r.st % 4) *vec = false;
  return GDN2_OK;
}
int check_f32(const void* p, bool optional, bool* vec) {
  if (!p) return optional ? GDN2_OK : GDN2_ERR_NULL;
  if ((uintptr_t)p % 4) return GDN2_ERR_ALIGN;
  if ((uintptr_t)p % 16) *vec = false;
  return GDN2_OK;
}

// Words of 64 bits, cleared 16 bytes at a time.
int check_ws(const void* p, size_t need) {
  return !need ? GDN2_OK : !p ? GDN2_ERR_NULL : (uintptr_t)p % 16 ? GDN2_ERR_ALIGN : GDN2_OK;
}

template <typename TX, typename TG, bool GATE, int V, int CT>
void launch_tile(hipStream_t st, const ScanArgs& a, bool bwd) {
  const dim3 grid(8u * (unsigned)a.chunk), block(8 * CT);
  if (bwd)
    hipLaunchKernelGGL((gscan_bwd<TX, TG, GATE, V, CT>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((gscan_fwd<TX, TG, GATE, V, CT>), grid, block, 0, st, a);
}
template <typename TX, typename TG, bool GATE, int V, int CT>
void launch_chain(hipStream_t st, const ScanArgs& a, bool bwd, int n) {
  // tickets, then slots, all cleared
  const size_t tickets = ticket_bytes(a.B * a.nct), bytes = tickets + (size_t)n * a.B * a.C * 8;
  Chain ch;
  // Drawing from one counter takes 10 ns a ticket; where all workgroups start at once that is
  // waited for (1 x 4001 x 768 17.8 us, from the tiles' own 14.1), where they do not it keeps the
  // tiles abreast (1 x 131072 x 1024 313 us, from the tiles' own 386).
  ch.own = n * a.B * a.nct <= 2 * num_cus();
  ch.ticket = (unsigned*)a.ws;
  ch.slot = (unsigned long long*)((char*)a.ws + tickets);
  const size_t pieces = (bytes + 15) / 16, wgs = (pieces + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(chain_clear, dim3((unsigned)(wgs < 2048 ? wgs : 2048)), dim3(kThreads), 0, st,
                     (uint4*)a.ws, pieces);
  const dim3 grid((unsigned)(n * a.B * a.nct)), block(512);
  if (bwd)
    hipLaunchKernelGGL((chain_bwd<TX, TG, GATE, V, CT>), grid, block, 0, st, a, ch);
  else
    hipLaunchKernelGGL((chain_fwd<TX, TG, GATE, V, CT>), grid, block, 0, st, a, ch);
}
template <typename TX, typename TG, bool GATE, int V>
void launch_width(hipStream_t st, const ScanArgs& a, bool bwd, const Split& s) {
  if (s.chain) {
    if constexpr (sizeof(TX) == 2)   // float32 takes no steps in tiles of 64
      if (s.ct == 64) return launch_chain<TX, TG, GATE, V, 64>(st, a, bwd, s.blocks);
    if (s.ct == 32)
      launch_chain<TX, TG, GATE, V, 32>(st, a, bwd, s.blocks);
    else
      launch_chain<TX, TG, GATE, V, 16>(st, a, bwd, s.blocks);
  } else if (s.ct == 64) {
    launch_tile<TX, TG, GATE, V, 64>(st, a, bwd);
  } else {
    launch_tile<TX, TG, GATE, V, 16>(st, a, bwd);
  }
}
template <typename TX, typename TG>
hipError_t launch_types(hipStream_t st, const ScanArgs& a, bool bwd, bool vec,
                        const Split& s) {
  if (a.b.p)
    vec ? launch_width<TX, TG, true, 4>(st, a, bwd, s) : launch_width<TX, TG, true, 1>(st, a, bwd, s);
  else
    vec ? launch_width<TX, TG, false, 4>(st, a, bwd, s)
        : launch_width<TX, TG, false, 1>(st, a, bwd, s);
  return hipGetLastError();
}
int launch_scan(hipStream_t st, ScanArgs& a, int in_dtype, int g_dtype, bool bwd, bool vec) {
  const Split s = split(a.B, a.T, a.C, in_dtype);
  a.nct = s.nct;
  a.chunk = (int)(((long long)a.B * a.nct + 7) / 8);
  const hipError_t e = in_dtype == GDN2_F32 ? launch_types<float, float>(st, a, bwd, vec, s)
                       : g_dtype == GDN2_F32 ? launch_types<bf16_t, float>(st, a, bwd, vec, s)
                                             : launch_types<bf16_t, bf16_t>(st, a, bwd, vec, s);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

template <typename TX, typename TG>
hipError_t launch_step(hipStream_t st, size_t n, const void* x, const void* g, const void* b,
                       const float* h_in, float* h_out, void* out, bool vec) {
  // a grid's threads stay within 32 bits: the kernel walks over what lies beyond
  const size_t per = (size_t)kThreads * (vec ? 4 : 1), wgs = (n + per - 1) / per;
  const dim3 grid((unsigned)(wgs < 65536 ? wgs : 65536)), block(kThreads);
#define GDN2_STEP(GATE, V)                                                                   \
  hipLaunchKernelGGL((gscan_step<TX, TG, GATE, V>), grid, block, 0, st, n, (const TX*)x,     \
                     (const TG*)g, (const TX*)b, h_in, h_out, (TX*)out)
  if (b) {
    if (vec) GDN2_STEP(true, 4); else GDN2_STEP(true, 1);
  } else {
    if (vec) GDN2_STEP(false, 4); else GDN2_STEP(false, 1);
  }
#undef GDN2_STEP
  return hipGetLastError();
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_gated_scan_kept_bytes(int B, int T, int C, int in_dtype) {
  if (validate(B, T, C, in_dtype, GDN2_F32) != GDN2_OK) return 0;
  return (size_t)split(B, T, C, in_dtype).blocks * B * C * sizeof(float);
}

size_t gdn2_gated_scan_workspace_bytes(int B, int T, int C, int in_dtype) {
  if (validate(B, T, C, in_dtype, GDN2_F32) != GDN2_OK) return 0;
  return split(B, T, C, in_dtype).ws;
}

int gdn2_gated_scan_fwd(void* stream, int B, int T, int C, int in_dtype, int g_dtype,
                        const void* x, const long long* x_strides, const void* g,
                        const long long* g_strides, const void* b, const long long* b_strides,
                        const float* h0, void* out, float* h_final, float* kept, void* ws,
                        size_t ws_bytes) {
  int rc = validate(B, T, C, in_dtype, g_dtype);
  if (rc) return rc;
  const long long dense[2] = {(long long)T * C, C};
  auto rows = [&](const void* p, const long long* s) {
    return Rows{p, (s ? s : dense)[0], (s ? s : dense)[1]};
  };
  ScanArgs a = {};
  a.x = rows(x, x_strides);
  a.g = rows(g, g_strides);
  a.b = rows(b, b_strides);
  a.h0 = h0;
  a.out = out;
  a.h_final = h_final;
  a.kept = kept;
  a.ws = ws;
  a.B = B;
  a.T = T;
  a.C = C;
  bool vec = C % 4 == 0;
  if (T > 0) {
    if ((rc = check_rows(a.x, in_dtype, &vec)) || (rc = check_rows(a.g, g_dtype, &vec)) ||
        (rc = check_rows({out, 0, 0}, in_dtype, &vec)))
      return rc;
    if (b && (rc = check_rows(a.b, in_dtype, &vec))) return rc;
    const size_t need = gdn2_gated_scan_workspace_bytes(B, T, C, in_dtype);
    if ((rc = check_ws(ws, need))) return rc;
    if (ws_bytes < need) return GDN2_ERR_WORKSPACE;
  }
  if ((rc = check_f32(h_final, false, &vec)) || (rc = check_f32(h0, true, &vec)) ||
      (rc = check_f32(kept, true, &vec)))
    return rc;
  if (T == 0) {
    const size_t n = (size_t)B * C;
    hipLaunchKernelGGL(gscan_none, dim3((unsigned)((n + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, (hipStream_t)stream, n, h0, h_final);
    return hipGetLastError() == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
  }
  return launch_scan((hipStream_t)stream, a, in_dtype, g_dtype, false, vec);
}

int gdn2_gated_scan_bwd(void* stream, int B, int T, int C, int in_dtype, int g_dtype,
                        const void* x, const long long* x_strides, const void* g,
                        const long long* g_strides, const void* b, const long long* b_strides,
                        const void* dout, const long long* dout_strides, const float* dh_final,
                        const float* kept, void* dx, void* dg, void* db, float* dh0, void* ws,
                        size_t ws_bytes) {
  int rc = validate(B, T, C, in_dtype, g_dtype);
  if (rc) return rc;
  const long long dense[2] = {(long long)T * C, C};
  auto rows = [&](const void* p, const long long* s) {
    return Rows{p, (s ? s : dense)[0], (s ? s : dense)[1]};
  };
  ScanArgs a = {};
  a.x = rows(x, x_strides);
  a.g = rows(g, g_strides);
  a.b = rows(b, b_strides);
  a.dout = rows(dout, dout_strides);
  a.dh_final = dh_final;
  a.kept = const_cast<float*>(kept);
  a.dx = dx;
  a.dg = dg;
  a.db = db;
  a.dh0 = dh0;
  a.ws = ws;
  a.B = B;
  a.T = T;
  a.C = C;
  bool vec = C % 4 == 0;
  if (T == 0) return GDN2_ERR_SEQ_LEN;
  if ((rc = check_rows(a.x, in_dtype, &vec)) || (rc = check_rows(a.g, g_dtype, &vec)) ||
      (rc = check_rows({dx, 0, 0}, in_dtype, &vec)) ||
      (rc = check_rows({dg, 0, 0}, g_dtype, &vec)))
    return rc;
  if (b && ((rc = check_rows(a.b, in_dtype, &vec)) ||
            (rc = check_rows({db, 0, 0}, in_dtype, &vec))))
    return rc;
  if (dout && (rc = check_rows(a.dout, in_dtype, &vec))) return rc;
  if ((rc = check_f32(kept, false, &vec)) || (rc = check_f32(dh_final, true, &vec)) ||
      (rc = check_f32(dh0, true, &vec)))
    return rc;
  const size_t need = gdn2_gated_scan_workspace_bytes(B, T, C, in_dtype);
  if ((rc = check_ws(ws, need))) return rc;
  if (ws_bytes < need) return GDN2_ERR_WORKSPACE;
  return launch_scan((hipStream_t)stream, a, in_dtype, g_dtype, true, vec);
}

int gdn2_gated_scan_step(void* stream, long long n, int in_dtype, int g_dtype, const void* x,
                         const void* g, const void* b, const float* h_in, float* h_out,
                         void* out) {
  if (n < 0 || n > (1ll << 38)) return GDN2_ERR_SHAPE;
  int rc = validate(1, 1, 1, in_dtype, g_dtype);
  if (rc) return rc;
  if (n == 0) return GDN2_OK;
  bool vec = n % 4 == 0;
  if ((rc = check_rows({x, 0, 0}, in_dtype, &vec)) || (rc = check_rows({g, 0, 0}, g_dtype, &vec)) ||
      (rc = check_rows({out, 0, 0}, in_dtype, &vec)) || (rc = check_f32(h_out, false, &vec)) ||
      (rc = check_f32(h_in, true, &vec)))
    return rc;
  if (b && (rc = check_rows({b, 0, 0}, in_dtype, &vec))) return rc;
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e =
      in_dtype == GDN2_F32 ? launch_step<float, float>(st, n, x, g, b, h_in, h_out, out, vec)
      : g_dtype == GDN2_F32
          ? launch_step<bf16_t, float>(st, n, x, g, b, h_in, h_out, out, vec)
          : launch_step<bf16_t, bf16_t>(st, n, x, g, b, h_in, h_out, out, vec);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

}  // extern "C"
