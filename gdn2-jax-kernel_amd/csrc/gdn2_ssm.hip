// Selective state space scan over (B, T, C) with N states a channel:
//   d = softplus(dt + dt_bias)   (or dt + dt_bias as it is)
//   h_t[c,n] = e^{d_t[c] A[c,n]} h_{t-1}[c,n] + d_t[c] x_t[c] B_t[n]
//   y_t[c] = sum_n C_t[n] h_t[c,n] + D[c] x_t[c],   out_t = y_t silu(z_t),
// its backward pass and its step for one token.  B and C are shared by the C / G channels of a
// group.  A token marked in `starts` begins a sequence: the state before it is dropped, not
// multiplied by zero.
//
// A run of tokens maps the state entering it to the one leaving it by h -> e^{A S} h + H with S
// the sum of its d: one number a channel beside H.  The axis is cut into chunks: a first kernel
// composes every chunk (S and H), a second walks over the chunks, a third walks each chunk's
// tokens again from the state that enters it.  What bounds this is not memory but the
// exponentials, N for each token and channel, of which a SIMD starts a wave's every 16 cycles, and
// the three to five operations around each at 4: a wave of 64 lanes has a channel a lane and all
// its states in registers, so that nothing else is left to do but for B and C.  Those, the same for
// all lanes, a small kernel lays out as float32 rows, which each wave brings to its part of LDS,
// sixteen tokens at a time.  8 x 8192 x 768 x 16 in bfloat16, gated: rows 6 us, compositions 159,
// join 12, outputs 209, where the exponentials, multiplies and additions for the states alone need
// 28 and 32 cycles for 64 states, 143 and 164 us at 2.4 GHz; softplus and the gate, once for each
// token and channel, are most of the rest.
//
// Backward: the gradients that enter chunks from the right come the same way.  The forward
// keeps the state before every 16th token; from it a workgroup forms 16 tokens' states again,
// keeps them and their decays in registers, and walks back.  Here a lane has four states of a
// channel, and sums over states and over channels are formed by lane exchanges.  A state takes one
// exponential and about 20 operations, half of them for those sums, which bound it: 8 x 2048 x
// 1536 x 16 in 375 us (forward 86, 12 and 124, reverse 94 and 12, sums over workgroups 23).
// Sums over workgroups are written as partial sums and added in a fixed order.
// Everything is float32 between the inputs' and the outputs' types.
#include <limits.h>

#include "gdn2.h"
#include "gdn2_common.h"

namespace gdn2 {
namespace {

constexpr int kThreads = 256;
constexpr int kKeep = 16;      // tokens between kept states
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_inff();
constexpr long long kMaxStride = 1 << 25;   // elements from one token to the next

// Strides are in elements; channels are contiguous.
struct Rows {
  const void* p;
  long long sb, st;
};
struct SsmArgs {
  Rows x, dt, z, bm, cm, dout;
  const float *A, *D, *dt_bias, *h0, *dh_final;   // (C,N) (C) (C) (B,C,N) (B,C,N); or null but A
  const unsigned char* starts;                     // (B,T) or null
  void *out, *dx, *ddt, *dz, *dbm, *dcm;           // dense
  float *h_final, *dh0, *dA, *dD, *dbias;
  float* kept;                                     // (B, ceil(T / kKeep), C, NP) or null
  float* bc;      // (B, T, G, 2, NP): B and C in float32, the states past N zero
  // workspace
  float* part_bc; // (tiles, B, T, 2, NP)
  float* part_a;  // (B chunks, C, NP)
  float* part_c;  // (B chunks, 2, C)
  float* slot;    // (B, chunks, C, NP): state or gradient that enters a chunk
  float* sum;     // (B, chunks, C): S of a chunk, -inf where a sequence starts in it
  int B, T, C, G, N;
  int Cg, tiles;  // channels of a group, tiles of a group
  int L, chunks;  // tokens of a chunk
  int softplus;
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_(float x) { return __builtin_amdgcn_rcpf(x); }

// log(1 + e^v) = max(v, 0) + log1p(e^-|v|), log1p(u) = 2 artanh(r) with r = u / (2 + u) <= 1/3.
// artanh(r) = r p(r^2): p fitted for the least relative error up to 1/9, 2^-26.9 with these
// coefficients.  NaN comes through u.  All in all 6 units in the last place for |v| <= 4, 10 to 8, 16 at
// -16 and about |v| below: the rounding of |v| log2 e.
__device__ __forceinline__ float softplus(float v) {
  const float u = exp2_(-fabsf(v) * kLog2e), r = u * rcp_(2.f + u), q = r * r;
  float p = 0.14089167f;
  p = fmaf(p, q, 0.139803f);
  p = fmaf(p, q, 0.20012455f);
  p = fmaf(p, q, 0.33333158f);
  p = fmaf(p, q, 1.f);
  return fmaf(2.f * r, p, fmaxf(v, 0.f));
}
__device__ __forceinline__ float sigmoid(float v) { return rcp_(1.f + exp2_(-v * kLog2e)); }

template <typename T>
__device__ __forceinline__ float element(const Rows& r, int b, int t, int c) {
  return (float)((const T*)r.p)[b * r.sb + t * r.st + c];
}

// A value at a distance in bytes from a place that is the same for all lanes: one address in
// scalar registers, 32 bits a lane.
template <typename T>
__device__ __forceinline__ T at(const T* p, unsigned off) {
  return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + off);
}
template <typename T>
__device__ __forceinline__ void put(T* p, unsigned off, T v) {
  *reinterpret_cast<T*>(reinterpret_cast<char*>(p) + off) = v;
}

// B and C in float32, NP states each, four a thread.
template <typename TX>
__global__ void __launch_bounds__(kThreads) ssm_rows(SsmArgs a, int NP) {
  const int quads = NP / 4, shift = __builtin_ctz(quads);
  const long long n = (long long)a.B * a.T * a.G * 2 << shift;
  for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < n;
       e += (long long)gridDim.x * kThreads) {
    const int s = (int)(e & (quads - 1)) * 4;
    const long long row = e >> shift;          // ((b T + t) G + g) 2 + which
    const long long bt = a.G == 1 ? row >> 1 : (row >> 1) / a.G;
    const int g = (int)((row >> 1) - bt * a.G), b = (int)(bt / a.T), t = (int)(bt - (long long)b * a.T);
    const Rows& r = row & 1 ? a.cm : a.bm;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (s + k < a.N) v[k] = element<TX>(r, b, t, g * a.N + s + k);
    *reinterpret_cast<f32x4*>(a.bc + 4 * e) = v;
  }
}

// Where a wave of a channel a lane works.
struct WavePlace {
  int b, chunk, g, c, t0, t1;
  bool on, idle;
  __device__ WavePlace(const SsmArgs& a, int first_chunk, int chunks) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int nt = a.G * a.tiles;
    const int unit = blockIdx.x * (kThreads / 64) + wave;
    idle = unit >= a.B * chunks * nt;
    const int tile = unit % nt, rest = unit / nt;
    chunk = first_chunk + rest % chunks;
    b = rest / chunks;
    g = tile / a.tiles;
    const int first = (tile - g * a.tiles) * 64, cg = first + lane;
    on = cg < a.Cg;
    c = g * a.Cg + (on ? cg : first);      // lanes without a channel repeat the wave's first
    t0 = chunk * a.L;
    t1 = a.T - t0 < a.L ? a.T : t0 + a.L;
  }
};

constexpr int kAhead = 4;   // tokens loaded at a time

// NP states of (row, c) at p (rows of C channels), from and to float32.
template <int NP>
__device__ __forceinline__ void load_states(const float* p, float (&h)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; n += 4) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[n + e] = v[e];
  }
}
template <int NP>
__device__ __forceinline__ void store_states(float* p, const float (&h)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; n += 4)
    *reinterpret_cast<f32x4*>(p + n) = f32x4{h[n], h[n + 1], h[n + 2], h[n + 3]};
}
// N values at p, the others zero (all of them without p); no branches, so one wait for all.
template <int NP>
__device__ __forceinline__ void load_user(const float* p, int N, float (&h)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; ++n) h[n] = 0.f;
  if (!p) return;
  float v[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) v[n] = p[n < N ? n : N - 1];
#pragma unroll
  for (int n = 0; n < NP; ++n) h[n] = n < N ? v[n] : 0.f;
}

// Rows of B and C (W floats from `from` on of each row of bc) of 16 tokens in LDS, a part for each
// wave: a token's row is then the same 16-byte reads for all lanes.  (In scalar registers, read
// token by token, every token waited for its row: 1 x 4001 x 1536 x 16 composed in 38 us, so 30.)
template <int W>
struct WaveRows {
  static constexpr int PIECES = kKeep * W / 4, PER = (PIECES + 63) / 64;
  f32x4 r[PER];
  __device__ __forceinline__ void load(const float* rows, long long stride, int t, int t1) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int p = i * 64 + (threadIdx.x & 63), k = p / (W / 4);
      const int ti = t + k < t1 ? t + k : t1 - 1;
      r[i] = *reinterpret_cast<const f32x4*>(rows + ti * stride + p % (W / 4) * 4);
    }
  }
  __device__ __forceinline__ void store(float* lds) const {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int p = i * 64 + (threadIdx.x & 63);
      if (PIECES % 64 == 0 || p < PIECES) *reinterpret_cast<f32x4*>(lds + 4 * p) = r[i];
    }
    __builtin_amdgcn_wave_barrier();
  }
};

// Forward.  OUT: the tokens from the entering state, outputs and kept states; else the
// composition of chunks 0 .. chunks - 2, H of chunk k into slot k + 1.  STARTS apart: a branch in
// every token costs a copy of all states (8 x 8192 x 768 x 16 composed in 201 us, without 178 then).
template <typename TX, typename TD, int NP, bool STARTS, bool OUT>
__global__ void __launch_bounds__(kThreads, NP <= 16 ? 4 : 2) ssm_fwd(SsmArgs a) {
  const WavePlace w(a, 0, OUT ? a.chunks : a.chunks - 1);
  if (w.idle) return;
  const int nch = a.chunks;
  float A2[NP], h[NP];
  load_user<NP>(a.A + (long long)w.c * a.N, a.N, A2);
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] *= kLog2e;
    h[n] = 0.f;
  }
  const float bias = a.dt_bias ? a.dt_bias[w.c] : 0.f, D = OUT && a.D ? a.D[w.c] : 0.f;
  if (OUT) {
    if (w.chunk == 0)
      load_user<NP>(a.h0 ? a.h0 + ((long long)w.b * a.C + w.c) * a.N : nullptr, a.N, h);
    else
      load_states<NP>(a.slot + (((long long)w.b * nch + w.chunk) * a.C + w.c) * NP, h);
  }
  const int nb = (a.T + kKeep - 1) / kKeep;
  const TX* px = (const TX*)a.x.p + w.b * a.x.sb;
  const TD* pd = (const TD*)a.dt.p + w.b * a.dt.sb;
  const TX* pz = (const TX*)a.z.p + w.b * a.z.sb;
  const unsigned ox = (unsigned)w.c * sizeof(TX), od = (unsigned)w.c * sizeof(TD);
  const bool gate = OUT && a.z.p;
  TX rx[kAhead], rz[kAhead];
  TD rd[kAhead];
  auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const long long ti = t + i < w.t1 ? t + i : w.t1 - 1;
      rx[i] = at(px + ti * a.x.st, ox);
      rd[i] = at(pd + ti * a.dt.st, od);
      if (gate) rz[i] = at(pz + ti * a.z.st, ox);
    }
  };
  load(w.t0);
  float S = 0.f;
  bool fresh = false;
  TX* out = (TX*)a.out + (long long)w.b * a.T * a.C;
  constexpr int RW = OUT ? 2 * NP : NP;
  __shared__ __attribute__((aligned(16))) float lds[kThreads / 64][kKeep * RW];
  float* own = lds[threadIdx.x >> 6];
  const long long stride = (long long)a.G * 2 * NP;
  const float* bc = a.bc + (long long)w.b * a.T * stride + w.g * 2 * NP;
  WaveRows<RW> rows;
  rows.load(bc, stride, w.t0, w.t1);
  auto token = [&](int t, float x, float d, float z) {
    if (STARTS && a.starts[(long long)w.b * a.T + t]) {
      fresh = true;
#pragma unroll
      for (int n = 0; n < NP; ++n) h[n] = 0.f;
    }
    const float* row = own + t % kKeep * RW;
    const float u = d * x;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NP; n += 4) {
      const f32x4 Bv = *reinterpret_cast<const f32x4*>(row + n);
      f32x4 Cv;
      if (OUT) Cv = *reinterpret_cast<const f32x4*>(row + NP + n);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[n + k] = fmaf(exp2_(d * A2[n + k]), h[n + k], u * Bv[k]);
        if (OUT) y[k] = fmaf(h[n + k], Cv[k], y[k]);
      }
    }
    S += d;
    if (OUT) {
      float o = fmaf(D, x, (y[0] + y[1]) + (y[2] + y[3]));
      if (gate) o *= z * sigmoid(z);
      // by all lanes, the same value where one repeats another's channel: stores that a lane may leave
      // out cannot be counted, and loads behind them wait for all (8 x 2048 x 1536 x 16 135 us, so 133)
      put(out + (long long)t * a.C, ox, (TX)o);
    }
  };
  float x[kAhead], d[kAhead], z[kAhead];
  auto take = [&](int t) {
    if (t % kKeep == 0) {
      rows.store(own);
      if (t + kKeep < w.t1) rows.load(bc, stride, t + kKeep, w.t1);
      if (OUT && a.kept && w.on)
        store_states<NP>(a.kept + (((long long)w.b * nb + t / kKeep) * a.C + w.c) * NP, h);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      x[i] = (float)rx[i];
      d[i] = (float)rd[i] + bias;
      z[i] = gate ? (float)rz[i] : 0.f;
    }
    if (a.softplus) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) d[i] = softplus(d[i]);
    }
  };
  // the odd ones last, apart: within the loop they would cost a copy of all states
  int t = w.t0;
  for (; t + kAhead <= w.t1; t += kAhead) {
    take(t);
    load(t + kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) token(t + i, x[i], d[i], z[i]);
  }
  if (t < w.t1) {
    take(t);
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i)
      if (t + i < w.t1) token(t + i, x[i], d[i], z[i]);
  }
  if (!w.on) return;
  if (!OUT) {
    store_states<NP>(a.slot + (((long long)w.b * nch + w.chunk + 1) * a.C + w.c) * NP, h);
    a.sum[((long long)w.b * nch + w.chunk) * a.C + w.c] = fresh ? kNegInf : S;
  } else if (w.chunk == nch - 1) {
    float* p = a.h_final + ((long long)w.b * a.C + w.c) * a.N;
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (n < a.N) p[n] = h[n];
  }
}

// The gradient that leaves chunks 1 .. chunks - 1 at their beginning with none entering, into the
// slot of the chunk before, and S.
template <typename TX, typename TD, int NP, bool STARTS>
__global__ void __launch_bounds__(kThreads, NP <= 16 ? 4 : 2) ssm_rev(SsmArgs a) {
  const WavePlace w(a, 1, a.chunks - 1);
  if (w.idle) return;
  const int nch = a.chunks;
  float A2[NP], e[NP];
  load_user<NP>(a.A + (long long)w.c * a.N, a.N, A2);
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] *= kLog2e;
    e[n] = 0.f;
  }
  const float bias = a.dt_bias ? a.dt_bias[w.c] : 0.f;
  const TX* po = (const TX*)a.dout.p + w.b * a.dout.sb;
  const TD* pd = (const TD*)a.dt.p + w.b * a.dt.sb;
  const TX* pz = (const TX*)a.z.p + w.b * a.z.sb;
  const unsigned ox = (unsigned)w.c * sizeof(TX), od = (unsigned)w.c * sizeof(TD);
  const bool gate = a.z.p, has = a.dout.p;
  TX ro[kAhead], rz[kAhead];
  TD rd[kAhead];
  auto load = [&](int t) {   // tokens t, t - 1, ...
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const long long ti = t - i > w.t0 ? t - i : w.t0;
      if (has) ro[i] = at(po + ti * a.dout.st, ox);
      rd[i] = at(pd + ti * a.dt.st, od);
      if (gate) rz[i] = at(pz + ti * a.z.st, ox);
    }
  };
  float S = 0.f;
  bool fresh = false;
  __shared__ __attribute__((aligned(16))) float lds[kThreads / 64][kKeep * NP];
  float* own = lds[threadIdx.x >> 6];
  const long long stride = (long long)a.G * 2 * NP;
  const float* bc = a.bc + (long long)w.b * a.T * stride + (w.g * 2 + 1) * NP;
  WaveRows<NP> rows;
  const int block = (w.t1 - 1) / kKeep * kKeep;
  rows.load(bc, stride, block, w.t1);
  rows.store(own);
  if (block > w.t0) rows.load(bc, stride, block - kKeep, w.t1);
  auto token = [&](int t, float g, float d) {
    const float* row = own + t % kKeep * NP;
#pragma unroll
    for (int n = 0; n < NP; n += 4) {
      const f32x4 Cv = *reinterpret_cast<const f32x4*>(row + n);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        e[n + k] = exp2_(d * A2[n + k]) * fmaf(g, Cv[k], e[n + k]);
      // whole before the loop turns, or both factors are carried over
#pragma unroll
      for (int k = 0; k < 4; ++k) asm("" : "+v"(e[n + k]));
    }
    S += d;
    if (STARTS && a.starts[(long long)w.b * a.T + t]) {
      fresh = true;
#pragma unroll
      for (int n = 0; n < NP; ++n) e[n] = 0.f;
    }
  };
  float g[kAhead], d[kAhead];
  auto take = [&] {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      g[i] = has ? (float)ro[i] : 0.f;
      d[i] = (float)rd[i] + bias;
      if (gate) {
        const float z = (float)rz[i];
        g[i] *= z * sigmoid(z);
      }
    }
    if (a.softplus) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) d[i] = softplus(d[i]);
    }
  };
  auto turn = [&](int t) {   // once token t is done: the sixteen tokens before it are next
    if (t % kKeep == 0 && t > w.t0) {
      rows.store(own);
      if (t - kKeep > w.t0) rows.load(bc, stride, t - 2 * kKeep, w.t1);
    }
  };
  // the odd ones first, apart: within the loop they would cost a copy of all states
  int t = w.t1 - 1;
  load(t);
  const int odd = (w.t1 - w.t0) % kAhead;
  if (odd) {
    take();
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i)
      if (i < odd) token(t - i, g[i], d[i]);
    t -= odd;
    turn(t + 1);
    load(t);
  }
  for (; t >= w.t0; t -= kAhead) {
    take();
    load(t - kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) token(t - i, g[i], d[i]);
    turn(t - kAhead + 1);
  }
  if (!w.on) return;
  store_states<NP>(a.slot + (((long long)w.b * nch + w.chunk - 1) * a.C + w.c) * NP, e);
  a.sum[((long long)w.b * nch + w.chunk) * a.C + w.c] = fresh ? kNegInf : S;
}

// What enters each chunk but the first, from the compositions: a thread a state of a channel, the
// chunks in order (REV: from the last).  What enters the first is h0 (the gradient of h_final), which
// the walks read themselves.
constexpr int kJoin = 64;   // threads: few states are to reach all CUs
template <int NP, bool REV>
__global__ void __launch_bounds__(kJoin) ssm_join(SsmArgs a) {
  const long long e = (long long)blockIdx.x * kJoin + threadIdx.x;
  const int n = (int)(e % NP);
  const long long bc = e / NP;
  const int b = (int)(bc / a.C), c = (int)(bc - (long long)b * a.C);
  if (b >= a.B) return;
  const float A2 = n < a.N ? a.A[(long long)c * a.N + n] * kLog2e : 0.f;
  const float* first = REV ? a.dh_final : a.h0;
  float h = first && n < a.N ? first[bc * a.N + n] : 0.f;
  const int nch = a.chunks;
  const long long step = (REV ? -1ll : 1ll) * a.C;
  const long long at = ((long long)b * nch + (REV ? nch - 1 : 0)) * a.C + c;
  float* slot = a.slot + at * NP + n;
  const float* sum = a.sum + at;
  // compositions are read sixteen at a time, the next while these are applied (1 x 4001 x 1536 x 16, 126
  // chunks: 13 us; eight at a time, each waited for, 17)
  constexpr int U = 16;
  float H[U], S[U];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const long long k = k0 + i < nch ? k0 + i : nch - 1;
      H[i] = slot[k * step * NP];
      S[i] = sum[(k - 1) * step];
    }
  };
  auto apply = [&](int k, float Hk, float Sk) {
    h = Sk == kNegInf ? Hk : fmaf(exp2_(A2 * Sk), h, Hk);
    slot[k * step * NP] = h;
  };
  int k0 = 1;
  load(k0);
  for (; k0 + U <= nch; k0 += U) {
    float now[U], sums[U];
#pragma unroll
    for (int i = 0; i < U; ++i) now[i] = H[i], sums[i] = S[i];
    load(k0 + U);   // past the last chunk: its, read again and not used
#pragma unroll
    for (int i = 0; i < U; ++i) apply(k0 + i, now[i], sums[i]);
  }
#pragma unroll
  for (int i = 0; i < U - 1; ++i) {
    if (k0 + i >= nch) break;
    apply(k0 + i, H[i], S[i]);
  }
}

// ---- Backward ----------------------------------------------------------------------

// v + the value of the lane whose number differs in bit BIT, for sums over the low bits from bit 0
// on: lanes that differ in lower bits alone hold the same by then, so a mirror will do.
template <int BIT>
__device__ __forceinline__ float add_low(float v) {
  constexpr int ctrl = BIT == 0 ? 0xB1 : BIT == 1 ? 0x4E : BIT == 2 ? 0x141 : 0x140;
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                 0, __builtin_bit_cast(int, v), ctrl, 0xF, 0xF, true));
}
// Sum over the low LN bits of the lane's number.
template <int LN>
__device__ __forceinline__ float sum_low(float v) {
  v = add_low<0>(v);
  if constexpr (LN > 1) v = add_low<1>(v);
  if constexpr (LN > 2) v = add_low<2>(v);
  if constexpr (LN > 3) v = add_low<3>(v);
  return v;
}
// v0 and v1 summed over lane pairs that differ in bit 5 (4): v0's sum where the bit is 0, v1's
// where it is 1.
__device__ __forceinline__ float fold5(float v0, float v1) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v0), __float_as_uint(v1), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float fold4(float v0, float v1) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v0), __float_as_uint(v1), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int N>
__device__ __forceinline__ float add_rotated(float v) {   // within 16 lanes
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                 0, __builtin_bit_cast(int, v), 0x120 + N, 0xF, 0xF, true));
}
// Eight sums over all bits of the lane's number from LN on.  On return v[0] and v[1] are those of
// numbers 4 (bit 5) + 2 (bit 4) + 0 and 1.
template <int LN>
__device__ __forceinline__ void sum_high8(float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = fold5(v[k], v[k + 4]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    v[k] = fold4(v[k], v[k + 2]);
    if constexpr (LN <= 3) v[k] = add_rotated<8>(v[k]);
    if constexpr (LN <= 2) v[k] = add_rotated<4>(v[k]);
    if constexpr (LN <= 1) v[k] = add_rotated<2>(v[k]);
  }
}

// A workgroup walks a chunk of CT channels backwards, 16 tokens at a time.
template <int NP>
struct Bwd {
  static constexpr int NG = NP / 4;          // lanes of a channel, four states each
  static constexpr int LN = NG == 2 ? 1 : NG == 4 ? 2 : NG == 8 ? 3 : 4;
  static constexpr int CH = 64 / NG;         // channels of a wave
  static constexpr int CT = 4 * CH;          // and of a workgroup
  static constexpr int PER = kKeep * CT / kThreads;   // (token, channel) values of a thread
  static constexpr int STEP = kThreads / CT;          // tokens that the threads cover at a time
  struct Shared {
    float d[kKeep][CT], x[kKeep][CT], dy[kKeep][CT];
    float raw[kKeep][CT], dout[kKeep][CT], z[kKeep][CT];
    float sb[kKeep][CT], sa[kKeep][CT], y[kKeep][CT];   // sums over the states
    float bc[kKeep][2][NP];
    float red[4][kKeep][2][NP];                         // sums over a wave's channels
    unsigned fresh;                                     // bit i: token i starts a sequence
  };
};

template <typename TX, typename TD, int NP, bool STARTS>
__global__ void __launch_bounds__(kThreads, 2) ssm_bwd(SsmArgs a) {
  using P = Bwd<NP>;
  constexpr int NG = P::NG, CH = P::CH, CT = P::CT, PER = P::PER, STEP = P::STEP, LN = P::LN;
  __shared__ __attribute__((aligned(16))) typename P::Shared s;
  const int nt = a.G * a.tiles;
  const int tile = blockIdx.x % nt, rest = blockIdx.x / nt;
  const int chunk = rest % a.chunks, b = rest / a.chunks;
  const int g = tile / a.tiles, first = (tile - g * a.tiles) * CT;   // first channel of the group's
  const int t0 = chunk * a.L, t1 = a.T - t0 < a.L ? a.T : t0 + a.L;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nb = (a.T + kKeep - 1) / kKeep;

  // this thread's channel of the rows that are read and written, and its first token
  const int rc = tid % CT, ri = tid / CT;
  const bool r_on = first + rc < a.Cg;
  const int r_c = g * a.Cg + (r_on ? first + rc : 0);
  const float bias = a.dt_bias ? a.dt_bias[r_c] : 0.f, D = a.D ? a.D[r_c] : 0.f;
  float sum_D = 0.f, sum_bias = 0.f;
  const bool gate = a.z.p, has = a.dout.p;

  // this lane's channel and states
  const int ci = wave * CH + lane / NG, q = lane % NG;
  const bool on = first + ci < a.Cg;
  const int c = g * a.Cg + (on ? first + ci : 0);
  float A[4], e[4], dA[4] = {0.f, 0.f, 0.f, 0.f};
  const long long bc_c = (long long)b * a.C + c;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int n = 4 * q + k;
    A[k] = n < a.N ? a.A[(long long)c * a.N + n] : 0.f;
    e[k] = 0.f;
    if (chunk == a.chunks - 1 && a.dh_final && n < a.N) e[k] = a.dh_final[bc_c * a.N + n];
  }
  if (chunk < a.chunks - 1) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(
        a.slot + (((long long)b * a.chunks + chunk) * a.C + c) * NP + 4 * q);
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = v[k];
  }

  // What sixteen tokens need is loaded while the sixteen after them are worked on.  Rows: tokens ri,
  // ri + STEP, ... of this thread's channel; every sixteen tokens but the last lie in the chunk.
  constexpr int ROW = 2 * NP, BC = kKeep * ROW / kThreads;   // values of a thread of B's and C's rows
  const int last = (t1 - t0 - 1) / kKeep * kKeep + t0;
  const int c0 = g * a.Cg;
  const long long bt = (long long)b * a.T + last;
  const TX* px = (const TX*)a.x.p + b * a.x.sb + last * a.x.st + c0;
  const TD* pd = (const TD*)a.dt.p + b * a.dt.sb + last * a.dt.st + c0;
  const TX* po = (const TX*)a.dout.p + b * a.dout.sb + last * a.dout.st + c0;
  const TX* pz = (const TX*)a.z.p + b * a.z.sb + last * a.z.st + c0;
  const float* pbc = a.bc + (bt * a.G + g) * ROW;
  const float* pk = a.kept + (((long long)b * nb + last / kKeep) * a.C + c0) * NP;
  const unsigned char* ps = a.starts + bt;
  const unsigned cc = r_c - c0, ok = ((c - c0) * NP + 4 * q) * 4;
  TX rx[PER], ro[PER], rz[PER];
  TD rd[PER];
  float rbc[BC];
  f32x4 rk;
  bool rs = false;
  // first: the tokens at the chunk's end, of which not all need exist (the last one instead)
  auto load = [&](auto first) {
    constexpr bool FIRST = decltype(first)::value;
    const int most = t1 - last - 1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned k = FIRST && ri + i * STEP > most ? most : ri + (FIRST ? i * STEP : 0);
      const long long m = FIRST ? 0 : i * STEP;
      rx[i] = at(px + m * a.x.st, (k * (unsigned)a.x.st + cc) * (unsigned)sizeof(TX));
      rd[i] = at(pd + m * a.dt.st, (k * (unsigned)a.dt.st + cc) * (unsigned)sizeof(TD));
      if (has) ro[i] = at(po + m * a.dout.st, (k * (unsigned)a.dout.st + cc) * (unsigned)sizeof(TX));
      if (gate) rz[i] = at(pz + m * a.z.st, (k * (unsigned)a.z.st + cc) * (unsigned)sizeof(TX));
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      constexpr int S = kThreads / ROW;
      const unsigned j = tid / ROW, k = FIRST && (int)j + i * S > most ? most
                                                                     : j + (FIRST ? i * S : 0);
      const long long m = FIRST ? 0 : i * S;
      rbc[i] = at(pbc + m * a.G * ROW, (k * (unsigned)a.G * ROW + tid % ROW) * 4u);
    }
    rk = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(pk) + ok);
    if (STARTS) rs = lane < kKeep && (!FIRST || lane <= most) && at(ps, (unsigned)lane);
  };
  load(std::true_type{});
  const unsigned oo = ri * (unsigned)a.C + cc;      // of the rows that are written
  const long long o0 = bt * a.C + c0;
  TX *pdx = (TX*)a.dx + o0, *pdz = (TX*)a.dz + o0;
  TD* pdd = (TD*)a.ddt + o0;
  float* pp = a.part_bc + (((long long)tile * a.B + b) * a.T + last) * ROW;
  for (int t = last; t >= t0; t -= kKeep) {
    // stage: tokens past the end are neutral (d = x = dy = 0)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = ri + i * STEP;
      const bool real = r_on && t + k < t1;
      const float o = real && has ? (float)ro[i] : 0.f, raw = (float)rd[i] + bias;
      const float d = a.softplus ? softplus(raw) : raw;
      s.d[k][rc] = real ? d : 0.f;
      s.x[k][rc] = real ? (float)rx[i] : 0.f;
      s.raw[k][rc] = raw;
      s.dout[k][rc] = o;
      float dy = o;
      if (gate) {
        const float z = real ? (float)rz[i] : 0.f;
        s.z[k][rc] = z;
        dy *= z * sigmoid(z);
      }
      s.dy[k][rc] = dy;
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) (&s.bc[0][0][0])[tid + i * kThreads] = rbc[i];
    if (STARTS && wave == 0) {
      const unsigned long long m = __ballot(rs);
      if (lane == 0) s.fresh = (unsigned)m;
    }
    const f32x4 hv = rk;
    __syncthreads();
    if (t > t0) {
      px -= kKeep * a.x.st;
      pd -= kKeep * a.dt.st;
      po -= kKeep * a.dout.st;
      pz -= kKeep * a.z.st;
      pbc -= (long long)kKeep * a.G * ROW;
      pk -= (long long)a.C * NP;
      ps -= kKeep;
      load(std::false_type{});
    }
    const unsigned fresh = STARTS ? __builtin_amdgcn_readfirstlane(s.fresh) : 0u;

    // One token's values are read while the one before is worked on, and no further ahead: all of
    // them would not leave registers for the states.
    struct Token {
      float d, x, dy;
      f32x4 B, C;
    };
    auto read = [&](int i, bool back) {
      Token k;
      k.d = s.d[i][ci];
      k.x = s.x[i][ci];
      k.B = *reinterpret_cast<const f32x4*>(&s.bc[i][0][4 * q]);
      if (back) {
        k.dy = s.dy[i][ci];
        k.C = *reinterpret_cast<const f32x4*>(&s.bc[i][1][4 * q]);
      }
      return k;
    };
    float h[kKeep][4], dec[kKeep][4], now[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) now[k] = hv[k];
    Token next = read(0, false);
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const Token m = next;
      next = i + 1 < kKeep ? read(i + 1, false) : read(i, true);
      const float u = m.d * m.x, d2 = m.d * kLog2e;
      const bool f = STARTS && (fresh >> i & 1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        dec[i][k] = exp2_(d2 * A[k]);
        now[k] = fmaf(dec[i][k], f ? 0.f : now[k], u * m.B[k]);
        h[i][k] = now[k];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // Every lane of a channel holds the sums over its states, and several lanes the same sums over the
    // channels: each keeps those of its tokens in turn, and all write together, without a branch
    // in every token (8 x 2048 x 1536 x 16 411 us, so 373).
    constexpr int CP = 16 / NG;              // lanes with the same sums over channels
    const int cp = (lane & 15) / NG;
    float keep_b = 0.f, keep_a = 0.f, keep_y = 0.f, keep0 = 0.f, keep1 = 0.f;
#pragma unroll
    for (int i = kKeep - 1; i >= 0; --i) {
      const Token m = next;
      if (i) next = read(i - 1, true);
      const float u = m.d * m.x;
      const bool f = STARTS && (fresh >> i & 1);
      float v[8], sb = 0.f, sa = 0.f, y = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float dh = fmaf(m.dy, m.C[k], e[k]);
        v[k] = dh * u;               // of B
        v[4 + k] = m.dy * h[i][k];   // of C
        sb = fmaf(dh, m.B[k], sb);
        const float back = f ? 0.f : dh * dec[i][k];
        const float through = f ? 0.f : back * (i ? h[i - 1][k] : hv[k]);
        sa = fmaf(through, A[k], sa);
        dA[k] = fmaf(through, m.d, dA[k]);
        y = fmaf(m.C[k], h[i][k], y);
        e[k] = back;
      }
      sb = sum_low<LN>(sb);
      sa = sum_low<LN>(sa);
      y = sum_low<LN>(y);
      const bool mine = q == i % NG;
      keep_b = mine ? sb : keep_b;
      keep_a = mine ? sa : keep_a;
      keep_y = mine ? y : keep_y;
      if (i % NG == 0) {
        s.sb[i + q][ci] = keep_b;
        s.sa[i + q][ci] = keep_a;
        s.y[i + q][ci] = keep_y;
      }
      sum_high8<LN>(v);
      const bool held = CP == 1 || cp == i % CP;
      keep0 = held ? v[0] : keep0;
      keep1 = held ? v[1] : keep1;
      if (i % CP == 0) {
        float* r = &s.red[wave][i + cp][lane >> 5][4 * q + 2 * (lane >> 4 & 1)];
        r[0] = keep0;
        r[1] = keep1;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    // sums over the states to gradients of x, dt and z; sums over the waves' channels
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = ri + i * STEP;
      if (!r_on || t + k >= t1) continue;
      const float d = s.d[k][rc], x = s.x[k][rc], dy = s.dy[k][rc], sb = s.sb[k][rc];
      const long long m = (long long)i * STEP * a.C;
      put(pdx + m, oo * (unsigned)sizeof(TX), (TX)fmaf(d, sb, D * dy));
      float dd = fmaf(x, sb, s.sa[k][rc]);
      if (a.softplus) dd *= sigmoid(s.raw[k][rc]);
      put(pdd + m, oo * (unsigned)sizeof(TD), (TD)dd);
      sum_bias += dd;
      sum_D = fmaf(dy, x, sum_D);
      if (gate) {
        const float z = s.z[k][rc], sg = sigmoid(z), y = fmaf(D, x, s.y[k][rc]);
        put(pdz + m, oo * (unsigned)sizeof(TX),
            (TX)(s.dout[k][rc] * y * sg * fmaf(z, 1.f - sg, 1.f)));
      }
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      const int k = tid + i * kThreads;
      const float* r = &s.red[0][0][0][0] + k;
      if (k / ROW < t1 - t)
        put(pp, k * 4u, (r[0] + r[kKeep * ROW]) + (r[2 * kKeep * ROW] + r[3 * kKeep * ROW]));
    }
    pdx -= (long long)kKeep * a.C;
    pdd -= (long long)kKeep * a.C;
    pdz -= (long long)kKeep * a.C;
    pp -= kKeep * ROW;
    __syncthreads();   // the next tokens are staged over what was read here
  }

  const long long row = (long long)b * a.chunks + chunk;
  if (on) {
    *reinterpret_cast<f32x4*>(a.part_a + (row * a.C + c) * NP + 4 * q) =
        f32x4{dA[0], dA[1], dA[2], dA[3]};
    if (chunk == 0 && a.dh0) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (4 * q + k < a.N) a.dh0[bc_c * a.N + 4 * q + k] = e[k];
    }
  }
  s.sb[ri][rc] = sum_D;
  s.sa[ri][rc] = sum_bias;
  __syncthreads();
  if (tid < CT && r_on) {
    float u = 0.f, v = 0.f;
#pragma unroll
    for (int k = 0; k < STEP; ++k) {
      u += s.sb[k][rc];
      v += s.sa[k][rc];
    }
    a.part_c[row * 2 * a.C + r_c] = u;
    a.part_c[(row * 2 + 1) * a.C + r_c] = v;
  }
}

// Partial sums added in their order.  The first workgroups: the gradients of A, D and dt_bias, 64
// columns each (C NP of part_a, then 2 C of part_c), 16 rows at a time, walking on over the columns
// where kSumsMost are too few.  The others: those of B and C, the tiles of a group for each value.
constexpr int kSumsMost = 1 << 20;   // a launch's threads stay within 32 bits
template <typename TX>
__global__ void __launch_bounds__(1024) ssm_sums(SsmArgs a, int NP, int first) {
  if ((int)blockIdx.x >= first) {
    const long long bt = (long long)a.B * a.T, n = bt * a.G * 2 * NP;
    for (long long e = (long long)(blockIdx.x - first) * 1024 + threadIdx.x; e < n;
         e += (long long)(gridDim.x - first) * 1024) {
      const long long row = e / (2 * NP);    // bt G + g
      const int k = (int)(e - row * 2 * NP), g = (int)(row % a.G);
      const int s = k % NP;
      if (s >= a.N) continue;
      const float* p = a.part_bc + ((long long)g * a.tiles * bt + row / a.G) * 2 * NP + k;
      float v = 0.f;
      for (int i = 0; i < a.tiles; ++i) v += p[i * bt * 2 * NP];
      ((TX*)(k < NP ? a.dbm : a.dcm))[row * a.N + s] = (TX)v;
    }
    return;
  }
  __shared__ float sum[16][64];
  const int col = threadIdx.x & 63, r = threadIdx.x >> 6;
  const long long wa = (long long)a.C * NP, wc = 2ll * a.C, rows = (long long)a.B * a.chunks;
  for (long long c0 = blockIdx.x * 64ll; c0 < wa + wc; c0 += first * 64ll) {
    const long long at = c0 + col;
    float v = 0.f;
    if (at < wa) {
      for (long long k = r; k < rows; k += 16) v += a.part_a[k * wa + at];
    } else if (at < wa + wc) {
      for (long long k = r; k < rows; k += 16) v += a.part_c[k * wc + at - wa];
    }
    sum[r][col] = v;
    __syncthreads();
    if (r == 0) {
      v = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) v += sum[k][col];
      if (at < wa) {
        const long long c = at / NP;
        const int n = (int)(at - c * NP);
        if (n < a.N) a.dA[c * a.N + n] = v;
      } else if (at < wa + a.C) {
        if (a.dD) a.dD[at - wa] = v;
      } else if (at < wa + wc) {
        if (a.dbias) a.dbias[at - wa - a.C] = v;
      }
    }
    __syncthreads();   // the next columns' rows are written over what was read here
  }
}

// One token: NG lanes a channel, four states each.
struct StepArgs {
  const void *x, *dt, *bm, *cm, *z;
  const float *A, *D, *dt_bias, *h_in;
  float* h_out;
  void* out;
  int B, C, G, N, Cg, softplus;
};
template <typename TX, typename TD, int NP>
__global__ void __launch_bounds__(kThreads) ssm_step(StepArgs a) {
  constexpr int NG = NP / 4;
  const int q = threadIdx.x % NG;
  const long long n = (long long)a.B * a.C;
  // every lane group of a wave walks the same number of times: its exchanges need all lanes
  const long long per = kThreads / NG, rounds = (n + per * gridDim.x - 1) / (per * gridDim.x);
  for (long long r = 0; r < rounds; ++r) {
    const long long e = (r * gridDim.x + blockIdx.x) * per + threadIdx.x / NG;
    const bool on = e < n;
    const long long bc = on ? e : n - 1;
    const int b = (int)(bc / a.C), c = (int)(bc - (long long)b * a.C);
    const long long g = (long long)b * a.G + c / a.Cg;
    const float x = (float)((const TX*)a.x)[bc];
    float d = (float)((const TD*)a.dt)[bc] + (a.dt_bias ? a.dt_bias[c] : 0.f);
    if (a.softplus) d = softplus(d);
    const float u = d * x;
    float y = 0.f, h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = 4 * q + k;
      h[k] = 0.f;
      if (s < a.N) {
        const float was = a.h_in ? a.h_in[bc * a.N + s] : 0.f;
        const float in = u * (float)((const TX*)a.bm)[g * a.N + s];
        h[k] = fmaf(exp2_(d * (a.A[(long long)c * a.N + s] * kLog2e)), was, in);
        y = fmaf(h[k], (float)((const TX*)a.cm)[g * a.N + s], y);
      }
    }
#pragma unroll
    for (int m = 1; m < NG; m *= 2) y += __shfl_xor(y, m);
    if (!on) continue;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (4 * q + k < a.N) a.h_out[bc * a.N + 4 * q + k] = h[k];
    if (q == 0) {
      if (a.D) y = fmaf(a.D[c], x, y);
      if (a.z) {
        const float z = (float)((const TX*)a.z)[bc];
        y *= z * sigmoid(z);
      }
      ((TX*)a.out)[bc] = (TX)y;
    }
  }
}

// ---- Host ----------------------------------------------------------------------------

int padded(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

// Channels of a workgroup of the backward.
int bwd_tile(int NP) { return 4 * (64 / (NP / 4)); }

struct Split {
  int np, L, chunks;
  int tiles, btiles;            // of a group: waves' (64 channels) and the backward's
  size_t bc, slot, sum, part_bc, part_a, part_c;   // bytes, multiples of 16
  // the forward's rows of B and C are in its workspace or, kept for the backward, behind the states
  size_t fwd() const { return slot + sum + bc; }
  size_t bwd() const { return slot + sum + part_bc + part_a + part_c; }
};
// (sizes that are refused need only come out large)
size_t round16(double n) { return n > 1e17 ? (size_t)1 << 58 : ((size_t)n + 15) / 16 * 16; }

// Chunks by sizes alone: the forward and the backward cut the axis alike.
Split split(int B, int T, int C, int G, int N) {
  Split s;
  s.np = padded(N);
  const int Cg = C / G;
  s.tiles = (Cg + 63) / 64;
  s.btiles = (Cg + bwd_tile(s.np) - 1) / bwd_tile(s.np);
  // chunks of 128 tokens where they make four waves a SIMD, else of 64 or 32, and of 16 where those
  // would not give every SIMD one.  Forward in us, chunks of 16, 32, 64 and 128 tokens:
  //   1 x 500 x 768 x 16     30   39   60  103     (0.4 waves a SIMD with 16 tokens)
  //   1 x 4001 x 1536 x 16  104   88   96  119     (2.9 with 32)
  //   4 x 2048 x 768 x 64   283  238  249  302     (3 with 32)
  //   8 x 2048 x 1536 x 16  259  222  212  215     (6 with 64)
  //   8 x 8192 x 768 x 16   522  425  396  394     (6 with 128)
  s.L = 128;
  auto waves = [&] { return (double)B * G * s.tiles * ((T + s.L - 1) / s.L); };
  while ((s.L > 32 && waves() < 4096) || (s.L > 16 && waves() < 1024)) s.L /= 2;
  s.chunks = T ? (T + s.L - 1) / s.L : 1;
  const double bt = (double)B * T, rows = (double)B * s.chunks;
  s.bc = round16(bt * G * 2 * s.np * 4);
  s.slot = s.chunks > 1 ? round16(rows * C * s.np * 4) : 0;
  s.sum = s.chunks > 1 ? round16(rows * C * 4) : 0;
  s.part_bc = round16((double)s.btiles * G * bt * 2 * s.np * 4);
  s.part_a = round16(rows * C * s.np * 4);
  s.part_c = round16(rows * 2 * C * 4);
  return s;
}

int validate(int B, int T, int C, int G, int N, int in_dtype, int dt_dtype) {
  if (B < 1 || T < 0 || C < 1 || G < 1 || G > C || C % G || N < 1 || N > 64) return GDN2_ERR_SHAPE;
  // channels and sixteen tokens' rows are reached in 32 bits (of bytes)
  if (T > INT_MAX - 1024 || C > (1 << 24) || G > (1 << 18)) return GDN2_ERR_SHAPE;
  if (in_dtype != GDN2_F32 && in_dtype != GDN2_BF16) return GDN2_ERR_DTYPE;
  if (dt_dtype != GDN2_F32 && dt_dtype != in_dtype) return GDN2_ERR_DTYPE;
  // a launch's threads stay within 32 bits and its waves' numbers within 31: one wave for at
  // least 16 tokens of at most 64 channels, one thread for a state
  const Split s = split(B, T, C, G, N);
  if ((double)B * G * s.tiles * s.chunks > (double)(1 << 25) ||
      (double)B * G * s.btiles * s.chunks > (double)(1 << 23) ||
      (double)B * C * s.np > (double)(1ll << 30))
    return GDN2_ERR_SHAPE;
  return GDN2_OK;
}

int check_rows(const Rows& r, int dtype, bool optional) {
  if (!r.p) return optional ? GDN2_OK : GDN2_ERR_NULL;
  return (uintptr_t)r.p % (dtype == GDN2_F32 ? 4 : 2) ? GDN2_ERR_ALIGN : GDN2_OK;
}
int check_f32(const void* p, bool optional) {
  if (!p) return optional ? GDN2_OK : GDN2_ERR_NULL;
  return (uintptr_t)p % 4 ? GDN2_ERR_ALIGN : GDN2_OK;
}
int check_ws(const void* p, size_t need, size_t have) {
  if (!need) return GDN2_OK;
  return !p ? GDN2_ERR_NULL : (uintptr_t)p % 16 ? GDN2_ERR_ALIGN
         : have < need ? GDN2_ERR_WORKSPACE : GDN2_OK;
}

unsigned groups_of(double n, double per, double most = 65536) {
  const double w = (n + per - 1) / per;
  return (unsigned)(w < most ? w : most);
}

template <typename TX>
void launch_rows(hipStream_t st, const SsmArgs& a, int NP) {
  hipLaunchKernelGGL((ssm_rows<TX>), dim3(groups_of((double)a.B * a.T * a.G * 2 * (NP / 4), kThreads)),
                     dim3(kThreads), 0, st, a, NP);
}

template <typename TX, typename TD, int NP, bool STARTS>
void launch_fwd(hipStream_t st, const SsmArgs& a) {
  const long long waves = (long long)a.B * a.G * a.tiles;
  launch_rows<TX>(st, a, NP);
  if (a.chunks > 1) {
    hipLaunchKernelGGL((ssm_fwd<TX, TD, NP, STARTS, false>),
                       dim3((unsigned)((waves * (a.chunks - 1) + 3) / 4)), dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL((ssm_join<NP, false>),
                       dim3((unsigned)(((long long)a.B * a.C * NP + kJoin - 1) / kJoin)),
                       dim3(kJoin), 0, st, a);
  }
  hipLaunchKernelGGL((ssm_fwd<TX, TD, NP, STARTS, true>), dim3((unsigned)((waves * a.chunks + 3) / 4)),
                     dim3(kThreads), 0, st, a);
}

template <typename TX, typename TD, int NP, bool STARTS>
void launch_bwd(hipStream_t st, SsmArgs a) {
  const long long waves = (long long)a.B * a.G * a.tiles;
  if (a.chunks > 1) {
    hipLaunchKernelGGL((ssm_rev<TX, TD, NP, STARTS>), dim3((unsigned)((waves * (a.chunks - 1) + 3) / 4)),
                       dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL((ssm_join<NP, true>),
                       dim3((unsigned)(((long long)a.B * a.C * NP + kJoin - 1) / kJoin)),
                       dim3(kJoin), 0, st, a);
  }
  a.tiles = (a.Cg + bwd_tile(NP) - 1) / bwd_tile(NP);
  hipLaunchKernelGGL((ssm_bwd<TX, TD, NP, STARTS>),
                     dim3((unsigned)((long long)a.B * a.G * a.tiles * a.chunks)), dim3(kThreads), 0,
                     st, a);
  const int first = (int)groups_of((double)a.C * (NP + 2), 64, kSumsMost);
  hipLaunchKernelGGL((ssm_sums<TX>),
                     dim3(first + groups_of((double)a.B * a.T * a.G * 2 * NP, 1024, 16384)), dim3(1024),
                     0, st, a, NP, first);
}

template <typename TX, typename TD>
hipError_t launch_types(hipStream_t st, const SsmArgs& a, bool bwd) {
  switch (padded(a.N)) {
#define GDN2_CASE(NP)                                                              \
  case NP:                                                                         \
    if (a.starts)                                                                  \
      bwd ? launch_bwd<TX, TD, NP, true>(st, a) : launch_fwd<TX, TD, NP, true>(st, a);   \
    else                                                                           \
      bwd ? launch_bwd<TX, TD, NP, false>(st, a) : launch_fwd<TX, TD, NP, false>(st, a); \
    break
    GDN2_CASE(8);
    GDN2_CASE(16);
    GDN2_CASE(32);
    GDN2_CASE(64);
#undef GDN2_CASE
  }
  return hipGetLastError();
}
int launch(hipStream_t st, const SsmArgs& a, int in_dtype, int dt_dtype, bool bwd) {
  const hipError_t e = in_dtype == GDN2_F32    ? launch_types<float, float>(st, a, bwd)
                       : dt_dtype == GDN2_F32 ? launch_types<bf16_t, float>(st, a, bwd)
                                              : launch_types<bf16_t, bf16_t>(st, a, bwd);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

template <typename TX, typename TD>
hipError_t launch_step(hipStream_t st, const StepArgs& a) {
  const int NP = padded(a.N);
  const dim3 grid(groups_of((double)a.B * a.C, kThreads / (NP / 4))), block(kThreads);
  switch (NP) {
    case 8: hipLaunchKernelGGL((ssm_step<TX, TD, 8>), grid, block, 0, st, a); break;
    case 16: hipLaunchKernelGGL((ssm_step<TX, TD, 16>), grid, block, 0, st, a); break;
    case 32: hipLaunchKernelGGL((ssm_step<TX, TD, 32>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((ssm_step<TX, TD, 64>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}

// The inputs that the forward and the backward share.
int set_inputs(SsmArgs& a, int B, int T, int C, int G, int N, int in_dtype, int dt_dtype,
               int softplus, const void* const* ins, const long long* strides, const float* A,
               const float* D, const float* dt_bias, const unsigned char* starts) {
  if (softplus != 0 && softplus != 1) return GDN2_ERR_FLAGS;
  if (!ins) return GDN2_ERR_NULL;
  const long long widths[5] = {C, C, C, (long long)G * N, (long long)G * N};
  Rows* rows[5] = {&a.x, &a.dt, &a.z, &a.bm, &a.cm};
  int rc;
  for (int i = 0; i < 5; ++i) {
    *rows[i] = Rows{ins[i], strides ? strides[2 * i] : T * widths[i],
                    strides ? strides[2 * i + 1] : widths[i]};
    if ((rc = check_rows(*rows[i], i == 1 ? dt_dtype : in_dtype, i == 2))) return rc;
    if (rows[i]->p && (rows[i]->st < 0 || rows[i]->st > kMaxStride)) return GDN2_ERR_SHAPE;
  }
  if ((rc = check_f32(A, false)) || (rc = check_f32(D, true)) || (rc = check_f32(dt_bias, true)))
    return rc;
  a.A = A, a.D = D, a.dt_bias = dt_bias, a.starts = starts, a.softplus = softplus;
  a.B = B, a.T = T, a.C = C, a.G = G, a.N = N, a.Cg = C / G;
  return GDN2_OK;
}
// Bytes of the kept states, without the rows of B and C behind them.
size_t kept_states(int B, int T, int C, int N) {
  return (size_t)B * ((T + kKeep - 1) / kKeep) * C * padded(N) * sizeof(float);
}
void set_workspace(SsmArgs& a, const Split& s, void* ws, void* kept) {
  char* p = (char*)ws;
  a.slot = (float*)p;
  a.sum = (float*)(p += s.slot);
  a.bc = a.part_bc = (float*)(p += s.sum);
  a.part_a = (float*)(p += s.part_bc);
  a.part_c = (float*)(p += s.part_a);
  if (kept) a.bc = (float*)((char*)kept + kept_states(a.B, a.T, a.C, a.N));
  a.kept = (float*)kept;
  a.tiles = s.tiles, a.L = s.L, a.chunks = s.chunks;
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

size_t gdn2_selective_scan_kept_bytes(int B, int T, int C, int G, int N) {
  if (validate(B, T, C, G, N, GDN2_F32, GDN2_F32) != GDN2_OK) return 0;
  return kept_states(B, T, C, N) + split(B, T, C, G, N).bc;
}

size_t gdn2_selective_scan_workspace_bytes(int B, int T, int C, int G, int N, int backward) {
  if (validate(B, T, C, G, N, GDN2_F32, GDN2_F32) != GDN2_OK || T == 0) return 0;
  const Split s = split(B, T, C, G, N);
  return backward ? s.bwd() : s.fwd();
}

int gdn2_selective_scan_fwd(void* stream, int B, int T, int C, int G, int N, int in_dtype,
                            int dt_dtype, int softplus, const void* const* ins,
                            const long long* strides, const float* A, const float* D,
                            const float* dt_bias, const float* h0, const unsigned char* starts,
                            void* out, float* h_final, float* kept, void* ws, size_t ws_bytes) {
  int rc = validate(B, T, C, G, N, in_dtype, dt_dtype);
  if (rc) return rc;
  if (T == 0) return GDN2_ERR_SEQ_LEN;
  SsmArgs a = {};
  if ((rc = set_inputs(a, B, T, C, G, N, in_dtype, dt_dtype, softplus, ins, strides, A, D, dt_bias,
                       starts)))
    return rc;
  if ((rc = check_rows({out, 0, 0}, in_dtype, false)) || (rc = check_f32(h_final, false)) ||
      (rc = check_f32(h0, true)))
    return rc;
  if ((uintptr_t)kept % 16) return GDN2_ERR_ALIGN;
  if (h0 == h_final) return GDN2_ERR_FLAGS;    // read by other workgroups
  const Split s = split(B, T, C, G, N);
  if ((rc = check_ws(ws, s.fwd(), ws_bytes))) return rc;
  set_workspace(a, s, ws, kept);
  a.h0 = h0, a.out = out, a.h_final = h_final;
  return launch((hipStream_t)stream, a, in_dtype, dt_dtype, false);
}

int gdn2_selective_scan_bwd(void* stream, int B, int T, int C, int G, int N, int in_dtype,
                            int dt_dtype, int softplus, const void* const* ins,
                            const long long* strides, const float* A, const float* D,
                            const float* dt_bias, const unsigned char* starts, const void* dout,
                            const long long* dout_strides, const float* dh_final,
                            const float* kept, void* const* outs, float* dA, float* dD,
                            float* ddt_bias, float* dh0, void* ws, size_t ws_bytes) {
  int rc = validate(B, T, C, G, N, in_dtype, dt_dtype);
  if (rc) return rc;
  if (T == 0) return GDN2_ERR_SEQ_LEN;
  SsmArgs a = {};
  if ((rc = set_inputs(a, B, T, C, G, N, in_dtype, dt_dtype, softplus, ins, strides, A, D, dt_bias,
                       starts)))
    return rc;
  if (!outs) return GDN2_ERR_NULL;
  for (int i = 0; i < 5; ++i)
    if ((rc = check_rows({outs[i], 0, 0}, i == 1 ? dt_dtype : in_dtype, i == 2 && !a.z.p)))
      return rc;
  a.dout = Rows{dout, dout_strides ? dout_strides[0] : (long long)T * C,
                dout_strides ? dout_strides[1] : C};
  if (dout && (a.dout.st < 0 || a.dout.st > kMaxStride)) return GDN2_ERR_SHAPE;
  if ((rc = check_rows(a.dout, in_dtype, true)) || (rc = check_f32(dh_final, true)) ||
      (rc = check_f32(kept, false)) || (rc = check_f32(dA, false)) || (rc = check_f32(dD, true)) ||
      (rc = check_f32(ddt_bias, true)) || (rc = check_f32(dh0, true)))
    return rc;
  if ((uintptr_t)kept % 16) return GDN2_ERR_ALIGN;
  const Split s = split(B, T, C, G, N);
  if ((rc = check_ws(ws, s.bwd(), ws_bytes))) return rc;
  set_workspace(a, s, ws, const_cast<float*>(kept));
  a.dx = outs[0], a.ddt = outs[1], a.dz = outs[2], a.dbm = outs[3], a.dcm = outs[4];
  a.dh_final = dh_final;
  a.dA = dA, a.dD = dD, a.dbias = ddt_bias, a.dh0 = dh0;
  return launch((hipStream_t)stream, a, in_dtype, dt_dtype, true);
}

int gdn2_selective_scan_step(void* stream, int B, int C, int G, int N, int in_dtype, int dt_dtype,
                             int softplus, const void* x, const void* dt, const float* A,
                             const void* Bm, const void* Cm, const float* D, const void* z,
                             const float* dt_bias, const float* h_in, float* h_out, void* out) {
  if (B < 0) return GDN2_ERR_SHAPE;
  int rc = validate(1, 1, C, G, N, in_dtype, dt_dtype);
  if (rc) return rc;
  if (softplus != 0 && softplus != 1) return GDN2_ERR_FLAGS;
  if (B == 0) return GDN2_OK;
  for (const void* p : {x, Bm, Cm, (const void*)out})
    if ((rc = check_rows({p, 0, 0}, in_dtype, false))) return rc;
  if ((rc = check_rows({dt, 0, 0}, dt_dtype, false)) ||
      (rc = check_rows({z, 0, 0}, in_dtype, true)))
    return rc;
  if ((rc = check_f32(A, false)) || (rc = check_f32(D, true)) || (rc = check_f32(dt_bias, true)) ||
      (rc = check_f32(h_in, true)) || (rc = check_f32(h_out, false)))
    return rc;
  StepArgs a = {x, dt, Bm, Cm, z, A, D, dt_bias, h_in, h_out, out, B, C, G, N, C / G, softplus};
  const hipError_t e =
      in_dtype == GDN2_F32   ? launch_step<float, float>((hipStream_t)stream, a)
      : dt_dtype == GDN2_F32 ? launch_step<bf16_t, float>((hipStream_t)stream, a)
                             : launch_step<bf16_t, bf16_t>((hipStream_t)stream, a);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

}  // extern "C"
