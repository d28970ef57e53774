// Short causal convolution over each channel of (B, T, C):
//   y_t = act(bias + sum_{k < W} w[k] x_{t - W + 1 + k}),   W = 2, 3 or 4,
// act the identity or silu(v) = v / (1 + e^{-v}); its backward pass and its step for one token.
// The W - 1 inputs before the first token come from a state (zeros without one), and the last
// W - 1 are given back as the next.  A token marked in `starts` begins a sequence: what came
// before it is dropped from the taps (not multiplied by zero: NaN does not pass).
//
// Everything is read once and written once, which bounds all of it: a thread walks along a run
// of tokens for its V channels (8- or 16-byte accesses) with the taps in registers, the
// next tokens' loads in flight.  The halo of a run, W - 1 tokens (twice that in the backward,
// which forms the pre-activation values again), is read from cache.  Sums are float32.
// 8 x 8192 x 768 in bfloat16: forward 35 to 41 us (5.8 to 4.9 TB/s), backward 75 packed (4.0 TB/s; its
// operations bound it: the pre-activation again, its sigmoid, 2 W multiply-adds a value) and 4 for
// its sums over runs.
#include <limits.h>

#include "gdn2.h"
#include "gdn2_common.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;       // tokens loaded at a time

struct ConvArgs {
  const void* x;
  long long xb, xt;             // elements from one batch entry, one token to the next
  const void* dy;
  long long db, dt;
  const float *w, *bias;        // (C, W), (C) or null
  const void *state, *dlast;    // (B, W - 1, C) or null
  const unsigned char* starts;  // (B, T) or null
  void *y, *last, *dx, *dstate; // y: the forward's output
  float* part;                  // (rows, C, W + 1) partial sums of dw and dbias
  int B, T, C, silu;
  int run, runs;                // tokens of a run, runs of T in workgroups' units
  int nct;                      // channel tiles
};

template <typename T, int V> struct Raw;
template <> struct Raw<float, 4> { using type = f32x4; };
template <> struct Raw<bf16_t, 4> { using type = bf16x4; };
template <> struct Raw<float, 2> { using type = float __attribute__((ext_vector_type(2))); };
template <> struct Raw<bf16_t, 2> { using type = bf16_t __attribute__((ext_vector_type(2))); };
template <> struct Raw<float, 1> { using type = float; };
template <> struct Raw<bf16_t, 1> { using type = bf16_t; };
template <typename T, int V> using raw_t = typename Raw<T, V>::type;

template <typename T, int V>
__device__ __forceinline__ void widen(const raw_t<T, V>& r, float (&f)[V]) {
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
    raw_t<T, V> r;
#pragma unroll
    for (int c = 0; c < V; ++c) r[c] = (T)f[c];
    *reinterpret_cast<raw_t<T, V>*>(p) = r;
  }
}

__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-v * 1.44269504088896340736f));
}

// Where a thread works: CT lanes across the channels, kThreads / CT runs of a workgroup.
template <int V, int CT>
struct Place {
  static constexpr int RUNS = kThreads / CT;
  int b, c, first, part;   // batch entry, channel, first token, run of the batch entry's
  int ci, r;               // lane across the channels, run within the workgroup
  bool on;
  __device__ Place(const ConvArgs& a) {
    const unsigned tile = blockIdx.x % a.nct, rest = blockIdx.x / a.nct;
    b = rest / a.runs;
    part = rest;
    ci = threadIdx.x % CT;
    r = threadIdx.x / CT;
    c = (tile * CT + ci) * V;
    on = c < a.C;
    if (!on) c = 0;        // loads stay in bounds, nothing is stored
    first = ((int)(rest - (unsigned)b * a.runs) * RUNS + r) * a.run;
  }
};

// x at token t (t < T), from the state before the first; zero without one.
template <typename TX, int V, int W>
__device__ __forceinline__ raw_t<TX, V> input(const ConvArgs& a, int b, int c, int t) {
  using R = raw_t<TX, V>;
  if (t >= 0)
    return *reinterpret_cast<const R*>((const TX*)a.x + b * a.xb + t * a.xt + c);
  if (a.state)
    return *reinterpret_cast<const R*>((const TX*)a.state +
                                       ((long long)b * (W - 1) + W - 1 + t) * a.C + c);
  R zero;
  if constexpr (V == 1) {
    zero = (TX)0.f;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) zero[k] = (TX)0.f;
  }
  return zero;
}
__device__ __forceinline__ bool starts_at(const ConvArgs& a, int b, int t) {
  return a.starts && t >= 0 && a.starts[(long long)b * a.T + t];
}

template <typename TX, int V, int W>
struct Weights {
  float w[W][V], bias[V];
  __device__ __forceinline__ void load(const ConvArgs& a, int c) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int k = 0; k < W; ++k) w[k][v] = a.w[(long long)(c + v) * W + k];
      bias[v] = a.bias ? a.bias[c + v] : 0.f;
    }
  }
};

// The taps of a token: x of the W - 1 tokens before it, zero before a start, oldest first.
template <typename TX, int V, int W>
struct Taps {
  float x[W - 1][V];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) x[k][v] = 0.f;
  }
  __device__ __forceinline__ void push(const float (&now)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int k = 0; k + 1 < W - 1; ++k) x[k][v] = x[k + 1][v];
      x[W - 2][v] = now[v];
    }
  }
  // The taps of token t.
  __device__ __forceinline__ void before(const ConvArgs& a, int b, int c, int t) {
    raw_t<TX, V> r[W - 1];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) r[k] = input<TX, V, W>(a, b, c, t - (W - 1) + k);
    clear();
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      if (starts_at(a, b, t - (W - 1) + k)) clear();
      float f[V];
      widen<TX, V>(r[k], f);
      push(f);
    }
  }
  __device__ __forceinline__ void sum(const Weights<TX, V, W>& m, const float (&now)[V],
                                      float (&pre)[V]) const {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = m.bias[v];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) s = fmaf(m.w[k][v], x[k][v], s);
      pre[v] = fmaf(m.w[W - 1][v], now[v], s);
    }
  }
};

template <typename TX, int V, int W, int CT>
__global__ void __launch_bounds__(kThreads) conv_fwd(ConvArgs a) {
  const Place<V, CT> p(a);
  if (!p.on || p.first >= a.T) return;
  Weights<TX, V, W> m;
  m.load(a, p.c);
  const int end = a.T - p.first < a.run ? a.T : p.first + a.run;
  raw_t<TX, V> raw[kAhead];
  bool fresh[kAhead] = {};
  const TX* px = (const TX*)a.x + p.b * a.xb + p.c;
  auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int ti = t + i < end ? t + i : end - 1;
      raw[i] = *reinterpret_cast<const raw_t<TX, V>*>(px + ti * a.xt);
      if (a.starts) fresh[i] = a.starts[(long long)p.b * a.T + ti];
    }
  };
  load(p.first);
  Taps<TX, V, W> taps;
  taps.before(a, p.b, p.c, p.first);
  TX* y = (TX*)a.y + (long long)p.b * a.T * a.C + p.c;
  for (int t = p.first; t < end; t += kAhead) {
    float now[kAhead][V];
    bool anew[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      widen<TX, V>(raw[i], now[i]);
      anew[i] = fresh[i];
    }
    if (t + kAhead < end) load(t + kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (t + i >= end) break;
      if (anew[i]) taps.clear();
      float pre[V];
      taps.sum(m, now[i], pre);
      if (a.silu) {
#pragma unroll
        for (int v = 0; v < V; ++v) pre[v] *= sigmoid(pre[v]);
      }
      put<TX, V>(y + (long long)(t + i) * a.C, pre);
      taps.push(now[i]);
    }
  }
  if (end == a.T) {
    TX* last = (TX*)a.last + (long long)p.b * (W - 1) * a.C + p.c;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) put<TX, V>(last + (long long)k * a.C, taps.x[k]);
  }
}

// Backward.  With p_t the value before the activation and dp_t = dy_t act'(p_t):
// dx_t = sum_d w[W - 1 - d] dp_{t + d} over the tokens t + d < t + W of its sequence, dw[k] =
// sum_t dp_t x_{t - W + 1 + k}, dbias = sum_t dp_t; the last inputs' gradients come in addition.
// A run walks on W - 1 tokens past its end for the sums that begin in it.
template <typename TX, int V, int W, int CT, bool STARTS>
__global__ void __launch_bounds__(kThreads, V == 2 ? 4 : 1) conv_bwd(ConvArgs a) {
  using P = Place<V, CT>;
  using R = raw_t<TX, V>;
  const P p(a);
  __shared__ float sums[P::RUNS][CT][V * (W + 1)];
  float dw[W][V], dbias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    dbias[v] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][v] = 0.f;
  }
  if (p.on && p.first < a.T) {
    Weights<TX, V, W> m;
    m.load(a, p.c);
    const int own = a.T - p.first < a.run ? a.T : p.first + a.run;   // end of the run
    const int end = a.T - own < W - 1 ? a.T : own + W - 1;           // and of the walk
    R rx[kAhead], rd[kAhead];
    bool fresh[kAhead] = {};
    const TX* px = (const TX*)a.x + p.b * a.xb + p.c;
    const bool has = a.dy;   // without it, x's values in its place, not used
    const TX* pd = has ? (const TX*)a.dy + p.b * a.db + p.c : px;
    const long long dt = has ? a.dt : a.xt;
    auto load = [&](int t) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int ti = t + i < end ? t + i : end - 1;
        rx[i] = *reinterpret_cast<const R*>(px + ti * a.xt);
        rd[i] = *reinterpret_cast<const R*>(pd + ti * dt);
        if (STARTS) fresh[i] = a.starts[(long long)p.b * a.T + ti];
      }
    };
    load(p.first);
    Taps<TX, V, W> taps;
    taps.before(a, p.b, p.c, p.first);
    // tokens of its sequence before a token that its sum reaches (at most W - 1)
    int age = W - 1;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) age = starts_at(a, p.b, p.first - (W - 1) + k) ? 0 : age + 1;
    // sums of the tokens t - d, which may still grow
    float sum[W][V];
#pragma unroll
    for (int d = 0; d < W; ++d)
#pragma unroll
      for (int v = 0; v < V; ++v) sum[d][v] = 0.f;
    TX* dx = (TX*)a.dx + (long long)p.b * a.T * a.C + p.c;
    TX* ds = (TX*)a.dstate + (long long)p.b * (W - 1) * a.C + p.c;
    // a finished sum, where this run owns it
    auto finish = [&](int t, const float (&f)[V]) {
      if (t >= p.first && t < own)
        put<TX, V>(dx + (long long)t * a.C, f);
      else if (t < 0 && p.first == 0 && a.dstate)
        put<TX, V>(ds + (long long)(W - 1 + t) * a.C, f);
    };
    // A group of tokens, taken out of the registers that the next one is then loaded into.
    float now[kAhead][V], d[kAhead][V];
    bool anew[kAhead];
    auto take = [&](int t) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        widen<TX, V>(rx[i], now[i]);
        anew[i] = fresh[i];
        widen<TX, V>(rd[i], d[i]);
#pragma unroll
        for (int v = 0; v < V; ++v) d[i][v] = has ? d[i][v] : 0.f;
      }
      load(t + kAhead < end ? t + kAhead : end - 1);
    };
    // Whether the next group is of the run, not its first and far from a start, in all lanes, as
    // nearly always: then there is nothing to choose, and the windows move once.
    auto plain = [&](int t) {
      bool yes = t > p.first && t + kAhead <= own && age >= W - 1;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) yes &= !fresh[i];
      return __all(yes);
    };
    auto quick = [&](int t) {
      constexpr int H = W - 1, N = H + kAhead;
      float x[N][V], s[N][V];   // tokens t - H ..
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k < H; ++k) {
          x[k][v] = taps.x[k][v];
          s[k][v] = sum[H - k][v];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          x[H + i][v] = now[i][v];
          s[H + i][v] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          float dp = d[i][v];
          if (a.silu) {
            float pre = m.bias[v];
#pragma unroll
            for (int k = 0; k < W; ++k) pre = fmaf(m.w[k][v], x[i + k][v], pre);
            const float g = sigmoid(pre);
            dp *= g * fmaf(pre, 1.f - g, 1.f);
          }
          dbias[v] += dp;
#pragma unroll
          for (int k = 0; k < W; ++k) {
            s[i + k][v] = fmaf(m.w[k][v], dp, s[i + k][v]);
            dw[k][v] = fmaf(dp, x[i + k][v], dw[k][v]);
          }
        }
#pragma unroll
        for (int k = 0; k < H; ++k) {
          taps.x[k][v] = x[kAhead + k][v];
          sum[H - k][v] = s[kAhead + k][v];
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) put<TX, V>(dx + (long long)(t + i - H) * a.C, s[i]);
      age += kAhead;
    };
    auto slow = [&](int t) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (t + i >= end) break;
        age = anew[i] ? 0 : age + 1;
        if (anew[i]) taps.clear();
        if (a.silu) {
          float pre[V];
          taps.sum(m, now[i], pre);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float s = sigmoid(pre[v]);
            d[i][v] *= s * fmaf(pre[v], 1.f - s, 1.f);
          }
        }
        const bool mine = t + i < own;
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
          for (int q = 0; q < W; ++q)
            if (q <= age) sum[q][v] = fmaf(m.w[W - 1 - q][v], d[i][v], sum[q][v]);
          if (mine) {
            dbias[v] += d[i][v];
            dw[W - 1][v] = fmaf(d[i][v], now[i][v], dw[W - 1][v]);
            // taps before a start are zero
#pragma unroll
            for (int k = 0; k < W - 1; ++k) dw[k][v] = fmaf(d[i][v], taps.x[k][v], dw[k][v]);
          }
        }
        finish(t + i - (W - 1), sum[W - 1]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
          for (int q = W - 1; q > 0; --q) sum[q][v] = sum[q - 1][v];
          sum[0][v] = 0.f;
        }
        taps.push(now[i]);
      }
    };
    // The loop of plain groups has one path, so that the stores behind a group's loads can be counted
    // when these are waited for; stores that a lane may leave out could not, and every group
    // waited for all stores before it (8 x 8192 x 768 bfloat16, W = 4, 129 us, so 81).  Loads from before
    // it are waited for ahead of it.
    for (int t = p.first; t < end; t += kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        asm volatile("" : "+v"(rx[i]));
        asm volatile("" : "+v"(rd[i]));
      }
      while (plain(t)) {
        take(t);
        quick(t);
        t += kAhead;
      }
      if (t >= end) break;
      take(t);
      slow(t);
    }
    // sum[q] is token end - q's: at the end of the axis the last inputs' gradients join it
    if (end == a.T) {
#pragma unroll
      for (int q = 1; q < W; ++q) {
        if (a.dlast && q - 1 <= age) {
          const R r = *reinterpret_cast<const R*>(
              (const TX*)a.dlast + ((long long)p.b * (W - 1) + W - 1 - q) * a.C + p.c);
          float f[V];
          widen<TX, V>(r, f);
#pragma unroll
          for (int v = 0; v < V; ++v) sum[q][v] += f[v];
        }
        finish(end - q, sum[q]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < W; ++k) sums[p.r][p.ci][v * (W + 1) + k] = dw[k][v];
    sums[p.r][p.ci][v * (W + 1) + W] = dbias[v];
  }
  __syncthreads();
  const int width = CT * V * (W + 1), c0 = (int)(blockIdx.x % a.nct) * CT * V;
  for (int e = threadIdx.x; e < width; e += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < P::RUNS; ++r) s += (&sums[r][0][0])[e];
    if (c0 + e / (W + 1) < a.C)
      a.part[((long long)p.part * a.C + c0) * (W + 1) + e] = s;
  }
}

// The partial sums of dw and dbias added in their order: 16 columns a workgroup, 64 rows at a
// time.  A grid of kSumsMost workgroups walks on over the columns.
constexpr unsigned kSumsMost = 1u << 20;   // a launch's threads stay within 32 bits
__global__ void __launch_bounds__(1024) conv_sums(const float* part, long long rows, int C, int W,
                                                  float* dw, float* dbias) {
  __shared__ float s[64][16];
  const int col = threadIdx.x & 15, r = threadIdx.x >> 4;
  const long long width = (long long)C * (W + 1);
  for (long long first = blockIdx.x * 16ll; first < width; first += gridDim.x * 16ll) {
    const long long at = first + col;
    float v = 0.f;
    if (at < width)
      for (long long k = r; k < rows; k += 64) v += part[k * width + at];
    s[r][col] = v;
    __syncthreads();
    if (r == 0 && at < width) {
      v = 0.f;
#pragma unroll
      for (int k = 0; k < 64; ++k) v += s[k][col];
      const long long c = at / (W + 1);
      const int k = (int)(at - c * (W + 1));
      if (k < W)
        dw[c * W + k] = v;
      else if (dbias)
        dbias[c] = v;
    }
    __syncthreads();   // the next columns' rows are written over what was read here
  }
}

// One token: a thread V channels of a batch entry; old and new state may be the same memory.
template <typename TX, int V, int W>
__global__ void __launch_bounds__(kThreads) conv_step(ConvArgs a) {
  const int per = a.C / V;
  const long long n = (long long)a.B * per;
  for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < n;
       e += (long long)gridDim.x * kThreads) {
    const int b = (int)(e / per), c = (int)(e - (long long)b * per) * V;
    Weights<TX, V, W> m;
    m.load(a, c);
    Taps<TX, V, W> taps;
    float now[V], pre[V];
    raw_t<TX, V> r[W];
#pragma unroll
    for (int k = 0; k < W; ++k) r[k] = input<TX, V, W>(a, b, c, k - (W - 1));
#pragma unroll
    for (int k = 0; k < W - 1; ++k) widen<TX, V>(r[k], taps.x[k]);
    widen<TX, V>(r[W - 1], now);
    taps.sum(m, now, pre);
    if (a.silu) {
#pragma unroll
      for (int v = 0; v < V; ++v) pre[v] *= sigmoid(pre[v]);
    }
    put<TX, V>((TX*)a.y + (long long)b * a.C + c, pre);
    TX* last = (TX*)a.last + (long long)b * (W - 1) * a.C + c;
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
      *reinterpret_cast<raw_t<TX, V>*>(last + (long long)k * a.C) = r[k + 1];
  }
}

struct Split {
  int ct, run, runs, nct;       // runs: workgroups along the tokens of a batch entry
};
// Lanes across the channels and tokens of a run, by sizes alone: the backward's workspace is
// sized for one channel a thread or two, whichever needs more.
Split split(int B, int T, int C, int V, bool back) {
  Split s;
  const int groups = (C + V - 1) / V;
  // 16 lanes across the channels where 64 would leave over a third of the lanes without any (8 x 8192 x
  // 288 in bfloat16 with 64 lanes 27 us, with 16 21; 3 x 1001 x 1003, one channel a lane, 7.5 and 11.5)
  const int lanes16 = (groups + 15) / 16 * 16, lanes64 = (groups + 63) / 64 * 64;
  s.ct = 2ll * lanes64 > 3ll * lanes16 ? 16 : 64;
  s.nct = (groups + s.ct - 1) / s.ct;
  const int per = kThreads / s.ct;
  // runs of 32 tokens where they make two workgroups a CU, else of 16 or 8 (runs of 32, 16 and 8: 8 x
  // 8192 x 768 in bfloat16 34, 35 and 36 us, 1 x 4096 x 768 10, 7.0 and 6.3, 8 x 2048 x 64 9.9, 6.5 and 4.8)
  // The backward, whose first and last tokens of a run take longer, has runs of 64 where they make six
  // (8 x 8192 x 768 packed 75 us, of 32 81; 6 x 8192 x 768 48 and 48)
  s.run = back ? 64 : 32;
  while (s.run > 8 && (double)B * s.nct * ((T + per * s.run - 1ll) / (per * s.run)) <
                          (s.run == 64 ? 1536 : 512))
    s.run /= 2;
  s.runs = (int)((T + (long long)per * s.run - 1) / ((long long)per * s.run));
  return s;
}

int validate(int B, int T, int C, int W, int dtype) {
  if (B < 1 || T < 0 || C < 1 || W < 2 || W > 4) return GDN2_ERR_SHAPE;
  // token numbers of a run and its halo stay within 31 bits, a launch's threads within 32
  if (T > INT_MAX - 1024 || C > (1 << 24)) return GDN2_ERR_SHAPE;
  for (int V : {1, 2, 4}) {
    const Split s = split(B, T, C, V, false);   // the backward has no more
    if ((double)B * s.nct * (s.runs < 1 ? 1 : s.runs) > (double)(1 << 23)) return GDN2_ERR_SHAPE;
  }
  if (dtype != GDN2_F32 && dtype != GDN2_BF16) return GDN2_ERR_DTYPE;
  return GDN2_OK;
}

// A row operand: element-aligned, and whether 4-channel accesses fit it.
int check(const void* p, long long sb, long long st, int dtype, bool optional, bool* vec) {
  const uintptr_t e = dtype == GDN2_F32 ? 4 : 2;
  if (!p) return optional ? GDN2_OK : GDN2_ERR_NULL;
  if ((uintptr_t)p % e) return GDN2_ERR_ALIGN;
  if ((uintptr_t)p % (4 * e) || sb % 4 || st % 4) *vec = false;
  return GDN2_OK;
}
int check_f32(const void* p, bool optional) {
  if (!p) return optional ? GDN2_OK : GDN2_ERR_NULL;
  return (uintptr_t)p % 4 ? GDN2_ERR_ALIGN : GDN2_OK;
}

enum Mode { kForward, kBackward, kStep };

// Channels of a thread of the backward, where four fit: their sums and windows would leave room for two
// waves a SIMD, those of two for four (8 x 8192 x 768 bfloat16, W = 4, 137 and 129 us, both before
// the loop of plain groups).
template <int V> constexpr int kBwd = V == 4 ? 2 : V;

template <typename TX, int V, int W>
void launch_width(hipStream_t st, ConvArgs& a, Mode mode) {
  if (mode == kStep) {
    const long long n = (long long)a.B * (a.C / V), wgs = (n + kThreads - 1) / kThreads;
    hipLaunchKernelGGL((conv_step<TX, V, W>), dim3((unsigned)(wgs < 65536 ? wgs : 65536)),
                       dim3(kThreads), 0, st, a);
    return;
  }
  const Split s = mode == kBackward ? split(a.B, a.T, a.C, kBwd<V>, true) : split(a.B, a.T, a.C, V, false);
  a.run = s.run, a.runs = s.runs, a.nct = s.nct;
  const dim3 grid((unsigned)((long long)a.B * s.runs * s.nct)), block(kThreads);
#define GDN2_CONV(CT)                                                             \
  if (mode == kForward)                                                           \
    hipLaunchKernelGGL((conv_fwd<TX, V, W, CT>), grid, block, 0, st, a);          \
  else if (a.starts)                                                              \
    hipLaunchKernelGGL((conv_bwd<TX, kBwd<V>, W, CT, true>), grid, block, 0, st, a); \
  else                                                                            \
    hipLaunchKernelGGL((conv_bwd<TX, kBwd<V>, W, CT, false>), grid, block, 0, st, a)
  if (s.ct == 16) {
    GDN2_CONV(16);
  } else {
    GDN2_CONV(64);
  }
#undef GDN2_CONV
}
template <typename TX, int V>
void launch_taps(hipStream_t st, ConvArgs& a, int W, Mode mode) {
  W == 2 ? launch_width<TX, V, 2>(st, a, mode)
  : W == 3 ? launch_width<TX, V, 3>(st, a, mode) : launch_width<TX, V, 4>(st, a, mode);
}
int launch(hipStream_t st, ConvArgs& a, int W, int dtype, bool vec, Mode mode) {
  if (dtype == GDN2_F32)
    vec ? launch_taps<float, 4>(st, a, W, mode) : launch_taps<float, 1>(st, a, W, mode);
  else
    vec ? launch_taps<bf16_t, 4>(st, a, W, mode) : launch_taps<bf16_t, 1>(st, a, W, mode);
  return hipGetLastError() == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_short_conv_bwd_workspace_bytes(int B, int T, int C, int W) {
  if (validate(B, T, C, W, GDN2_F32) != GDN2_OK || T == 0) return 0;
  const int r1 = split(B, T, C, 1, true).runs, r2 = split(B, T, C, 2, true).runs;
  return (size_t)B * (r1 > r2 ? r1 : r2) * C * (W + 1) * sizeof(float);
}

int gdn2_short_conv_fwd(void* stream, int B, int T, int C, int W, int dtype, int silu,
                        const void* x, const long long* x_strides, const float* w,
                        const float* bias, const void* state, const unsigned char* starts,
                        void* y, void* last) {
  int rc = validate(B, T, C, W, dtype);
  if (rc) return rc;
  if (silu != 0 && silu != 1) return GDN2_ERR_FLAGS;
  if (T == 0) return GDN2_ERR_SEQ_LEN;
  const long long dense[2] = {(long long)T * C, C};
  const long long* s = x_strides ? x_strides : dense;
  bool vec = C % 4 == 0;
  if ((rc = check(x, s[0], s[1], dtype, false, &vec)) ||
      (rc = check(y, 0, 0, dtype, false, &vec)) || (rc = check(last, 0, 0, dtype, false, &vec)) ||
      (rc = check(state, 0, 0, dtype, true, &vec)) || (rc = check_f32(w, false)) ||
      (rc = check_f32(bias, true)))
    return rc;
  if (state == last) return GDN2_ERR_FLAGS;   // read by other workgroups
  ConvArgs a = {};
  a.x = x, a.xb = s[0], a.xt = s[1], a.w = w, a.bias = bias, a.state = state, a.starts = starts;
  a.y = y, a.last = last, a.B = B, a.T = T, a.C = C, a.silu = silu;
  return launch((hipStream_t)stream, a, W, dtype, vec, kForward);
}

int gdn2_short_conv_bwd(void* stream, int B, int T, int C, int W, int dtype, int silu,
                        const void* x, const long long* x_strides, const float* w,
                        const float* bias, const void* state, const unsigned char* starts,
                        const void* dy, const long long* dy_strides, const void* dlast, void* dx,
                        float* dw, float* dbias, void* dstate, void* ws, size_t ws_bytes) {
  int rc = validate(B, T, C, W, dtype);
  if (rc) return rc;
  if (silu != 0 && silu != 1) return GDN2_ERR_FLAGS;
  if (T == 0) return GDN2_ERR_SEQ_LEN;
  const long long dense[2] = {(long long)T * C, C};
  const long long *s = x_strides ? x_strides : dense, *d = dy_strides ? dy_strides : dense;
  bool vec = C % 4 == 0;
  if ((rc = check(x, s[0], s[1], dtype, false, &vec)) ||
      (rc = check(dy, d[0], d[1], dtype, true, &vec)) ||
      (rc = check(dx, 0, 0, dtype, false, &vec)) || (rc = check(state, 0, 0, dtype, true, &vec)) ||
      (rc = check(dlast, 0, 0, dtype, true, &vec)) ||
      (rc = check(dstate, 0, 0, dtype, true, &vec)) || (rc = check_f32(w, false)) ||
      (rc = check_f32(bias, true)) || (rc = check_f32(dw, false)) ||
      (rc = check_f32(dbias, true)) || (rc = check_f32(ws, false)))
    return rc;
  if (ws_bytes < gdn2_short_conv_bwd_workspace_bytes(B, T, C, W)) return GDN2_ERR_WORKSPACE;
  ConvArgs a = {};
  a.x = x, a.xb = s[0], a.xt = s[1], a.w = w, a.bias = bias, a.state = state, a.starts = starts;
  a.dy = dy, a.db = d[0], a.dt = d[1], a.dlast = dlast, a.dx = dx, a.dstate = dstate;
  a.part = (float*)ws, a.B = B, a.T = T, a.C = C, a.silu = silu;
  if ((rc = launch((hipStream_t)stream, a, W, dtype, vec, kBackward))) return rc;
  const long long sums = ((long long)C * (W + 1) + 15) / 16;
  const unsigned wgs = sums < kSumsMost ? (unsigned)sums : kSumsMost;
  hipLaunchKernelGGL(conv_sums, dim3(wgs), dim3(1024), 0, (hipStream_t)stream, a.part,
                     (long long)B * a.runs, C, W, dw, dbias);
  return hipGetLastError() == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_short_conv_step(void* stream, int B, int C, int W, int dtype, int silu, const void* x,
                         const float* w, const float* bias, const void* state_in,
                         void* state_out, void* y) {
  if (B < 0) return GDN2_ERR_SHAPE;
  int rc = validate(1, 1, C, W, dtype);
  if (rc) return rc;
  if (silu != 0 && silu != 1) return GDN2_ERR_FLAGS;
  if (B == 0) return GDN2_OK;
  bool vec = C % 4 == 0;
  if ((rc = check(x, 0, 0, dtype, false, &vec)) || (rc = check(y, 0, 0, dtype, false, &vec)) ||
      (rc = check(state_out, 0, 0, dtype, false, &vec)) ||
      (rc = check(state_in, 0, 0, dtype, true, &vec)) || (rc = check_f32(w, false)) ||
      (rc = check_f32(bias, true)))
    return rc;
  ConvArgs a = {};
  a.x = x, a.xb = C, a.w = w, a.bias = bias, a.state = state_in, a.last = state_out, a.y = y;
  a.B = B, a.T = 1, a.C = C, a.silu = silu;
  return launch((hipStream_t)stream, a, W, dtype, vec, kStep);
}

}  // extern "C"
