// Gated linear recurrence over (B, T, C), elementwise in the C channels:
//   h_t = e^{g_t} h_{t-1} + b_t x_t,   out_t = h_t,   h_final = h_T,
// its backward pass and its step for one token.  A token with g_t = -inf starts
// anew: h_t = b_t x_t whatever h_{t-1} holds (NaN and infinities included), which
// separates the sequences of a packed batch.
//
// A run of tokens maps the state entering it to the one leaving it by h -> e^L h + H
// with L the sum of its g: two runs compose as (L1 + L2, e^{L2} H1 + H2).  L, not
// e^L, is carried, so that L = -inf says that the run holds a fresh start, and sums of
// small decays lose nothing.  Everything is held in float32.
//
// One workgroup walks the whole axis for 16 channels, 256 tokens at a time.  A thread
// takes V neighbouring channels (8- or 16-byte accesses) of S consecutive tokens: it
// composes its run in registers, the runs of a wave are composed by lane shuffles, the
// four waves' through LDS, and the thread then walks its tokens again from the state
// that enters them.  The data are read once, and the next 256 tokens are in flight
// meanwhile.  The backward pass needs the state before every token: the forward pass
// keeps the state that enters each 256 tokens (1/256 of the data), from which the
// backward forms them again on its way from the last 256 tokens to the first, so
// that it too reads every input once and never reads the outputs.
#include <limits.h>

#include "gdn2.h"
#include "gdn2_common.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 16;      // channels of a workgroup
constexpr int kBlock = 256;    // tokens of a step of the walk, and between kept states
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
  float* kept;                         // (ceil(T / kBlock), B, C) or null
  float* seg;                          // (nseg, 2, B, C): L and H (or D) of each segment
  int B, T, C, nct, nseg, seg_blocks;  // channel tiles; segments of seg_blocks steps
  int chunk;                           // work items of one XCD
};

// exp2 of a sum of g in units of log2(e).
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kNegInf = -__builtin_inff();

// e^l h + u, or u alone where l = -inf.
__device__ __forceinline__ float carry_through(float l, float h, float u) {
  return l == kNegInf ? u : fmaf(exp2_(l), h, u);
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

// Where a workgroup and a thread work.
template <int V>
struct Place {
  static constexpr int LPR = kTile / V;              // lanes across the channels
  static constexpr int TLW = 64 / LPR;               // runs of a wave
  static constexpr int S = kBlock * LPR / kThreads;  // tokens of a run
  int lane, wave, tl, c, b, seg;
  bool on;       // the channels exist
  bool idle;     // the workgroup has no work
  int blk0, blk1;
  __device__ Place(const ScanArgs& a) {
    // neighbouring channel tiles share cache lines: consecutive items on one XCD
    const int item = (blockIdx.x & 7) * a.chunk + (blockIdx.x >> 3);
    const int units = a.B * a.nct;
    idle = (blockIdx.x >> 3) >= a.chunk || item >= units * a.nseg;
    seg = item / units;
    const int unit = item - seg * units;
    b = unit / a.nct;
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    tl = lane / LPR;
    c = (unit - b * a.nct) * kTile + (lane % LPR) * V;
    on = c < a.C;
    if (!on) c = 0;   // loads stay in bounds, nothing is stored
    blk0 = seg * a.seg_blocks;
    const int n = (a.T + kBlock - 1) / kBlock;
    blk1 = blk0 + a.seg_blocks < n ? blk0 + a.seg_blocks : n;
  }
  // first token of the thread's run in step blk
  __device__ int first(int blk) const { return blk * kBlock + (wave * TLW + tl) * S; }
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
        L[c] += l;
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
    }
  }
}
// a h + u for one token of a run.
__device__ __forceinline__ float token(float a, float h, float u) {
  return fmaf(a, a < 0.f ? 0.f : h, u);
}

// The state that enters segment `seg`, from the earlier segments' compositions.
template <int V>
__device__ __forceinline__ void enter(const ScanArgs& a, size_t bc, int from, int to, int step,
                                      float (&h)[V]) {
  const size_t n = (size_t)a.B * a.C;
  for (int s = from; s != to; s += step) {
    const float* p = a.seg + 2 * n * s + bc;
#pragma unroll
    for (int c = 0; c < V; ++c) h[c] = carry_through(p[c], h[c], p[n + c]);
  }
}

// Forward.  SUMMARY: only the composition of each segment, into a.seg.
template <typename TX, typename TG, bool GATE, int V, bool SUMMARY>
__global__ void __launch_bounds__(kThreads) gscan_fwd(ScanArgs a) {
  using P = Place<V>;
  constexpr int S = P::S, LPR = P::LPR;
  __shared__ float sL[2][4][kTile], sH[2][4][kTile];
  const P w(a);
  if (w.idle) return;
  const int ci = (w.lane % LPR) * V;   // channel within the tile
  float h[V], Ls[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    h[c] = !SUMMARY && a.h0 ? a.h0[w.bc(a) + c] : 0.f;
    Ls[c] = 0.f;
  }
  if (!SUMMARY) enter<V>(a, w.bc(a), 0, w.seg, 1, h);
  Run<TX, V, S> x;
  Run<TG, V, S> g;
  std::conditional_t<GATE, Run<TX, V, S>, None> b;
  auto load = [&](int blk) {
    const int t = w.first(blk);
    x.load(a.x, w.b, w.c, t, a.T);
    g.load(a.g, w.b, w.c, t, a.T);
    if constexpr (GATE) b.load(a.b, w.b, w.c, t, a.T);
  };
  load(w.blk0);
  for (int blk = w.blk0; blk < w.blk1; ++blk) {
    const int t = w.first(blk);
    Factors<V, S> f;
    factors<TX, TG, GATE, V, S>(f, x, g, b, t, a.T);
    if (blk + 1 < w.blk1) load(blk + 1);
    float L[V], H[V], TL[V], TH[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      L[c] = f.L[c];
      H[c] = f.H[c];
    }
    wave_compose<V, LPR, false>(L, H, TL, TH, w.lane);
    const int buf = blk & 1;
    if (w.lane >= 64 - LPR) {
#pragma unroll
      for (int c = 0; c < V; ++c) {
        sL[buf][w.wave][ci + c] = TL[c];
        sH[buf][w.wave][ci + c] = TH[c];
      }
    }
    if (!SUMMARY && a.kept && w.on && w.wave == 0 && w.tl == 0)
      put<float, V>(a.kept + (size_t)blk * a.B * a.C + w.bc(a), h);
    lds_barrier();   // the other buffer is written next: one barrier a step
    float mine[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      mine[c] = h[c];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float l = sL[buf][k][ci + c];
        if (k == w.wave) mine[c] = h[c];
        h[c] = carry_through(l, h[c], sH[buf][k][ci + c]);
        if (SUMMARY) Ls[c] += l;
      }
    }
    if constexpr (!SUMMARY) {
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
  }
  if (w.on && w.wave == 0 && w.tl == 0) {
    if constexpr (SUMMARY) {
      const size_t n = (size_t)a.B * a.C;
      put<float, V>(a.seg + 2 * n * w.seg + w.bc(a), Ls);
      put<float, V>(a.seg + 2 * n * w.seg + n + w.bc(a), h);
    } else if (w.seg == a.nseg - 1) {
      put<float, V>(a.h_final + w.bc(a), h);
    }
  }
}

// Backward.  With e the gradient that reaches the state after token t from later tokens
// (dh_final after the last): dh = dout_t + e, dx = b dh, db = x dh, dg = a h_{t-1} dh,
// and a dh goes on to the token before; a run maps the e entering it from the right to
// e^L e + D.  SUMMARY: only L and D of each segment.
template <typename TX, typename TG, bool GATE, int V, bool SUMMARY>
__global__ void __launch_bounds__(kThreads) gscan_bwd(ScanArgs a) {
  using P = Place<V>;
  constexpr int S = P::S, LPR = P::LPR;
  __shared__ float sL[2][4][kTile], sH[2][4][kTile], sD[2][4][kTile];
  const P w(a);
  if (w.idle) return;
  const int ci = (w.lane % LPR) * V;
  float e[V], Ls[V];
#pragma unroll
  for (int c = 0; c < V; ++c) {
    e[c] = !SUMMARY && a.dh_final ? a.dh_final[w.bc(a) + c] : 0.f;
    Ls[c] = 0.f;
  }
  if (!SUMMARY) enter<V>(a, w.bc(a), a.nseg - 1, w.seg, -1, e);
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
    if constexpr (!SUMMARY) {
      x.load(a.x, w.b, w.c, t, a.T);
      if constexpr (GATE) b.load(a.b, w.b, w.c, t, a.T);
#pragma unroll
      for (int c = 0; c < V; ++c) h[c] = a.kept[(size_t)blk * a.B * a.C + w.bc(a) + c];
    }
  };
  load(w.blk1 - 1);
  for (int blk = w.blk1 - 1; blk >= w.blk0; --blk) {
    const int t = w.first(blk);
    Factors<V, S> f;
    float xv[S][V], bv[S][V], dv[S][V], hw[V];
    if constexpr (SUMMARY) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        float gv[V];
        widen<TG, V>(g.r[i], gv);
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const float l = t + i < a.T ? gv[c] * kLog2e : 0.f;
          f.a[i][c] = l == kNegInf ? -1.f : exp2_(l);
          f.L[c] = (i == 0 ? 0.f : f.L[c]) + l;
        }
      }
    } else {
      factors<TX, TG, GATE, V, S>(f, x, g, b, t, a.T);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        widen<TX, V>(x.r[i], xv[i]);
        if constexpr (GATE) widen<TX, V>(b.r[i], bv[i]);
      }
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
    if (blk > w.blk0) load(blk - 1);
    float L[V], H[V], R[V], D[V], TL[V], TH[V], TD[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      D[c] = 0.f;
#pragma unroll
      for (int i = S - 1; i >= 0; --i)
        D[c] = f.a[i][c] < 0.f ? 0.f : f.a[i][c] * (dv[i][c] + D[c]);
      R[c] = f.L[c];
      if constexpr (!SUMMARY) {
        L[c] = f.L[c];
        H[c] = f.H[c];
      }
    }
    const int buf = blk & 1;
    if constexpr (!SUMMARY) {
      wave_compose<V, LPR, false>(L, H, TL, TH, w.lane);
      if (w.lane >= 64 - LPR) {
#pragma unroll
        for (int c = 0; c < V; ++c) sH[buf][w.wave][ci + c] = TH[c];
      }
    }
    wave_compose<V, LPR, true>(R, D, TL, TD, w.lane);
    if (w.lane < LPR) {
#pragma unroll
      for (int c = 0; c < V; ++c) {
        sL[buf][w.wave][ci + c] = TL[c];
        sD[buf][w.wave][ci + c] = TD[c];
      }
    }
    lds_barrier();
    float mine[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      mine[c] = e[c];
#pragma unroll
      for (int k = 3; k >= 0; --k) {
        const float l = sL[buf][k][ci + c];
        if (k == w.wave) mine[c] = e[c];
        e[c] = carry_through(l, e[c], sD[buf][k][ci + c]);
        if (SUMMARY) Ls[c] += l;
      }
    }
    if constexpr (!SUMMARY) {
      float before[S][V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        float hc = hw[c];
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (k < w.wave) hc = carry_through(sL[buf][k][ci + c], hc, sH[buf][k][ci + c]);
        hc = carry_through(L[c], hc, H[c]);
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
  }
  if (w.on && w.wave == 0 && w.tl == 0) {
    if constexpr (SUMMARY) {
      const size_t n = (size_t)a.B * a.C;
      put<float, V>(a.seg + 2 * n * w.seg + w.bc(a), Ls);
      put<float, V>(a.seg + 2 * n * w.seg + n + w.bc(a), e);
    } else if (w.seg == 0 && a.dh0) {
      put<float, V>(a.dh0 + w.bc(a), e);
    }
  }
}

// One token: elementwise on n = B C values.
template <typename TX, typename TG, bool GATE, int V>
__global__ void __launch_bounds__(kThreads) gscan_step(size_t n, const TX* x, const TG* g,
                                                       const TX* b, const float* h_in,
                                                       float* h_out, TX* out) {
  const size_t i = ((size_t)blockIdx.x * kThreads + threadIdx.x) * V;
  if (i >= n) return;
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

// No token: the state passes through.
__global__ void __launch_bounds__(kThreads) gscan_none(size_t n, const float* h_in, float* h_out) {
  const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
  if (i < n) h_out[i] = h_in ? h_in[i] : 0.f;
}

// ---------------------------------------------------------------- host side

int blocks_of(int T) { return T / kBlock + (T % kBlock != 0); }

// Segments of the axis: where the (batch, channel tile) units leave most of the GPU
// idle, the axis is cut and a summary pass over the segments comes first.
int segments(int B, int T, int C) {
  const long long units = (long long)B * ((C + kTile - 1) / kTile);
  const int n = blocks_of(T);
  if (n < 8 || units >= 96) return 1;
  long long want = (256 + units - 1) / units;
  if (want > n / 4) want = n / 4;
  const int per = (int)((n + want - 1) / want);
  return (n + per - 1) / per;
}

int validate(int B, int T, int C, int in_dtype, int g_dtype) {
  if (B < 1 || C < 1 || T < 0) return GDN2_ERR_SHAPE;
  if (in_dtype != GDN2_F32 && in_dtype != GDN2_BF16) return GDN2_ERR_DTYPE;
  if (g_dtype != GDN2_F32 && !(g_dtype == GDN2_BF16 && in_dtype == GDN2_BF16))
    return GDN2_ERR_DTYPE;
  if (T > INT_MAX - kBlock || C > INT_MAX - kTile) return GDN2_ERR_SHAPE;
  // the launch's workgroups, and bytes of a tensor, within 31 and 62 bits
  if ((double)B * ((C + kTile - 1) / kTile) > 8.0e6) return GDN2_ERR_SHAPE;
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

template <typename TX, typename TG, bool GATE, int V>
hipError_t launch_scan(hipStream_t st, const ScanArgs& a, bool bwd) {
  const dim3 grid(8u * (unsigned)a.chunk), block(kThreads);
  if (bwd) {
    if (a.nseg > 1)
      hipLaunchKernelGGL((gscan_bwd<TX, TG, false, V, true>), grid, block, 0, st, a);
    hipLaunchKernelGGL((gscan_bwd<TX, TG, GATE, V, false>), grid, block, 0, st, a);
  } else {
    if (a.nseg > 1)
      hipLaunchKernelGGL((gscan_fwd<TX, TG, GATE, V, true>), grid, block, 0, st, a);
    hipLaunchKernelGGL((gscan_fwd<TX, TG, GATE, V, false>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}
template <typename TX, typename TG>
hipError_t launch_scan(hipStream_t st, const ScanArgs& a, bool bwd, bool vec) {
  if (a.b.p)
    return vec ? launch_scan<TX, TG, true, 4>(st, a, bwd) : launch_scan<TX, TG, true, 1>(st, a, bwd);
  return vec ? launch_scan<TX, TG, false, 4>(st, a, bwd) : launch_scan<TX, TG, false, 1>(st, a, bwd);
}
int launch_scan(hipStream_t st, ScanArgs& a, int in_dtype, int g_dtype, bool bwd, bool vec) {
  a.nct = (a.C + kTile - 1) / kTile;
  a.nseg = segments(a.B, a.T, a.C);
  const int n = blocks_of(a.T);
  a.seg_blocks = (n + a.nseg - 1) / a.nseg;
  a.chunk = (a.B * a.nct * a.nseg + 7) / 8;
  const hipError_t e = in_dtype == GDN2_F32 ? launch_scan<float, float>(st, a, bwd, vec)
                       : g_dtype == GDN2_F32 ? launch_scan<bf16_t, float>(st, a, bwd, vec)
                                             : launch_scan<bf16_t, bf16_t>(st, a, bwd, vec);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

template <typename TX, typename TG>
hipError_t launch_step(hipStream_t st, size_t n, const void* x, const void* g, const void* b,
                       const float* h_in, float* h_out, void* out, bool vec) {
  const size_t per = (size_t)kThreads * (vec ? 4 : 1);
  const dim3 grid((unsigned)((n + per - 1) / per)), block(kThreads);
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

size_t gdn2_gated_scan_kept_bytes(int B, int T, int C) {
  if (validate(B, T, C, GDN2_F32, GDN2_F32) != GDN2_OK) return 0;
  return (size_t)blocks_of(T) * B * C * sizeof(float);
}

size_t gdn2_gated_scan_workspace_bytes(int B, int T, int C) {
  if (validate(B, T, C, GDN2_F32, GDN2_F32) != GDN2_OK) return 0;
  const int nseg = segments(B, T, C);
  return nseg > 1 ? (size_t)nseg * 2 * B * C * sizeof(float) : 0;
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
  a.seg = (float*)ws;
  a.B = B;
  a.T = T;
  a.C = C;
  bool vec = C % 4 == 0;
  if (T > 0) {
    if ((rc = check_rows(a.x, in_dtype, &vec)) || (rc = check_rows(a.g, g_dtype, &vec)) ||
        (rc = check_rows({out, 0, 0}, in_dtype, &vec)))
      return rc;
    if (b && (rc = check_rows(a.b, in_dtype, &vec))) return rc;
    const size_t need = gdn2_gated_scan_workspace_bytes(B, T, C);
    if ((rc = check_f32(need ? ws : nullptr, need == 0, &vec))) return rc;
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
  a.seg = (float*)ws;
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
  const size_t need = gdn2_gated_scan_workspace_bytes(B, T, C);
  if ((rc = check_f32(need ? ws : nullptr, need == 0, &vec))) return rc;
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
