// RMS norm of x + residual, with its output in the input's type (and its backward) or in
// 8 bits with a scale for each row; rows in 8 bits without a norm, and back.
//
//   h = x + residual, rounded to the residual's type and returned;
//   y = h w rstd,  rstd = 1 / sqrt(mean h^2 + eps).
// In 8 bits: t = h w, m = max |t| of the row, q = round(127 t / m) (ties to even), the
// row's scale m rstd / 127.  rstd cancels from q, which therefore does not depend on the
// order of any sum.  A row of zeros has scale 0; one that holds NaN or an infinity has
// scale NaN and q = 0, so that everything computed from it is NaN.
// Backward, with n = h rstd, dn = dy w:
//   dh_total = rstd (dn - n mean(dn n)) + dh,   dx = dr = dh_total,   dw = sum dy n.
//
// All of these are bound by memory traffic: a row is read once into registers (8 values
// a thread and chunk, 16-byte accesses), reduced over its 64 to 1024 threads and
// written from the registers.  Sums and the norm's factors are float32.  A copy of 1 GiB reaches
// 5.16 TB/s on this card; these, with a residual, bfloat16: norm of 65536 x 768 73 us (5.5 TB/s),
// 16384 x 4096 95 (5.7); in 8 bits 65 (5.4), 84 (5.6).  Calls of a few hundred MB pass a copy's
// rate because part of their data is still in the last-level cache (256 MB): 4096 x 8192, 268 MB in
// all, 41 and 37 us (6.5 and 6.4 TB/s).
#include "gdn2.h"
#include "gdn2_common.h"

namespace gdn2 {
namespace {

constexpr int kMaxWidth = 16384;        // of a norm
constexpr int kMaxQuant = 32768;        // of rows in 8 bits without one
// Below this 127 / m overflows; rows this small count as zero.
constexpr float kTiny = 1e-36f;

struct NormArgs {
  const void *x, *r, *w;        // r: residual or null
  long long ldx, ldr;           // elements between rows
  void *y, *h;                  // dense; y null in 8 bits
  signed char* q;
  long long ldq;
  float *scale, *rstd;          // rstd: null unless the backward follows
  float eps;
  int M, C, w_bf16;
};

// 8 values at column c of a row of C, as they are stored.  VEC: the row is aligned to 16 bytes
// and C a multiple of 8; else the same accesses start at any value, and only a row's last piece
// goes value by value (65536 x 767 bfloat16, norm, in 8 bits, backward: 93, 82, 135 to 156 us; all
// value by value 291, 249, 197).  The backward, with two waves a SIMD to cover it, waits for
// that piece in three operands and a result of every row (65536 x 768 75 us).
template <typename V, typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
  V v;
};
template <typename V, typename T, bool VEC>
__device__ __forceinline__ V take(const T* p) {
  if constexpr (VEC)
    return *reinterpret_cast<const V*>(p);
  else
    return reinterpret_cast<const Loose<V, T>*>(p)->v;
}
template <typename V, typename T, bool VEC>
__device__ __forceinline__ void give(T* p, const V& v) {
  if constexpr (VEC)
    *reinterpret_cast<V*>(p) = v;
  else
    reinterpret_cast<Loose<V, T>*>(p)->v = v;
}
template <typename T, bool VEC> struct Raw8 {
  using V = std::conditional_t<sizeof(T) == 4, f32x4, bf16x8>;
  static constexpr int N = 16 / sizeof(T), P = 8 / N;   // values of an access, accesses
  V v[P];
  __device__ __forceinline__ void load(const T* row, int c, int C) {
    if (VEC ? c < C : c + 8 <= C) {
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = take<V, T, VEC>(row + c + i * N);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e / N][e % N] = !VEC && c + e < C ? row[c + e] : (T)0.f;
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return (float)v[e / N][e % N]; }
};
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int c, int C, float (&f)[8]) {
  Raw8<T, VEC> r;
  r.load(row, c, C);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = r[e];
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int c, int C, const float (&f)[8]) {
  if (VEC ? c < C : c + 8 <= C) {
    if constexpr (sizeof(T) == 4) {
      give<f32x4, T, VEC>(row + c, f32x4{f[0], f[1], f[2], f[3]});
      give<f32x4, T, VEC>(row + c + 4, f32x4{f[4], f[5], f[6], f[7]});
    } else {
      give<bf16x8, T, VEC>(row + c, make_op(f, (bf16x8*)nullptr));
    }
  } else if constexpr (!VEC) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < C) row[c + e] = from_f<T>(f[e]);
  }
}
template <bool VEC>
__device__ __forceinline__ void load_w(const void* w, int bf16, int c, int C, float (&f)[8]) {
  if (bf16)
    load8<bf16_t, VEC>((const bf16_t*)w, c, C, f);
  else
    load8<float, VEC>((const float*)w, c, C, f);
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  return x;
}
// Largest of the bit patterns of non-negative floats: NaN counts as the largest.
__device__ __forceinline__ unsigned wave_max(unsigned x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const unsigned y = __shfl_xor(x, m);
    x = x > y ? x : y;
  }
  return x;
}
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

enum { kNorm, kNorm8, kQuant };

// Threads of a workgroup with TPR threads to a row: a row alone, or four of a wave each.
template <int TPR> constexpr int kNT = TPR == 64 ? 256 : TPR;

// TPR threads take a row, NCH chunks of 8 values each.
template <typename TX, typename TR, int MODE, int TPR, int NCH, bool VEC>
__global__ void __launch_bounds__(kNT<TPR>) norm_fwd(NormArgs a) {
  constexpr int NT = kNT<TPR>, NW = TPR / 64;
  __shared__ float s_sum[NW];
  __shared__ unsigned s_max[NW];
  const int tid = threadIdx.x % TPR;
  const long long wg = (long long)blockIdx.y * gridDim.x + blockIdx.x;
  const long long row = wg * (NT / TPR) + threadIdx.x / TPR;
  if (row >= a.M) return;   // whole waves, and whole workgroups where a row has several
  const TX* x = (const TX*)a.x + row * a.ldx;
  float v[NCH][8];
#pragma unroll
  for (int j = 0; j < NCH; ++j) load8<TX, VEC>(x, (j * TPR + tid) * 8, a.C, v[j]);
  if (MODE != kQuant && a.r) {
    const TR* r = (const TR*)a.r + row * a.ldr;
    TR* h = (TR*)a.h + row * a.C;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = (j * TPR + tid) * 8;
      float f[8];
      load8<TR, VEC>(r, c, a.C, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = to_f(from_f<TR>(v[j][e] + f[e]));
      store8<TR, VEC>(h, c, a.C, v[j]);
    }
  }
  float rstd = 1.f, w[NCH][8];
  unsigned top = 0;
  if constexpr (MODE != kQuant) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      float part = 0.f;
      load_w<VEC>(a.w, a.w_bf16, (j * TPR + tid) * 8, a.C, w[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        part = fmaf(v[j][e], v[j][e], part);
        if (MODE == kNorm8) v[j][e] *= w[j][e];
      }
      sum += part;
    }
    sum = wave_sum(sum);
    if constexpr (NW > 1) {
      if (tid % 64 == 0) s_sum[tid / 64] = sum;
      lds_barrier();
      sum = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) sum += s_sum[k];
    }
    rstd = 1.f / sqrtf(sum / (float)a.C + a.eps);
    if (a.rstd && tid == 0) a.rstd[row] = rstd;
  }
  if constexpr (MODE == kNorm) {
    TX* y = (TX*)a.y + row * a.C;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = v[j][e] * rstd * w[j][e];
      store8<TX, VEC>(y, (j * TPR + tid) * 8, a.C, v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned u = magnitude(v[j][e]);
        top = top > u ? top : u;
      }
    top = wave_max(top);
    if constexpr (NW > 1) {
      if (tid % 64 == 0) s_max[tid / 64] = top;
      lds_barrier();
#pragma unroll
      for (int k = 0; k < NW; ++k) top = top > s_max[k] ? top : s_max[k];
    }
    const float m = __uint_as_float(top);
    const bool bad = top >= 0x7f800000u, zero = m < kTiny;
    const float inv = bad || zero ? 0.f : (1.f / m) * 127.f;
    if (tid == 0)
      a.scale[row] = bad ? __uint_as_float(0x7fc00000u) : zero ? 0.f : m * rstd / 127.f;
    signed char* q = a.q + row * a.ldq;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = (j * TPR + tid) * 8;
      unsigned p[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = bad ? 0 : (int)rintf(v[j][e] * inv);
        p[e / 4] |= ((unsigned)i & 0xffu) << (8 * (e % 4));
      }
      // the bytes between C and the next multiple of 16 are zeroed: ldq is one
      if (c < (int)a.ldq) *reinterpret_cast<uint2*>(q + c) = make_uint2(p[0], p[1]);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize(const signed char* q, long long ldq,
                                                  const float* scale, T* y, long long M, int C) {
  const int per = (C + 7) / 8;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < M * per;
       i += (long long)gridDim.x * 256) {
    const long long row = i / per;
    const int c = (int)(i - row * per) * 8;
    const float s = scale[row];
    float f[8];
    if (VEC || c + 8 <= C) {
      const uint2 p = take<uint2, signed char, VEC>(q + row * ldq + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)(signed char)((e < 4 ? p.x : p.y) >> (8 * (e % 4)));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = c + e < C ? (float)q[row * ldq + c + e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= s;
    store8<T, VEC>(y + row * C, c, C, f);
  }
}

struct NormBwdArgs {
  const void *h, *w, *dy, *dh;   // h, dy, dh dense; dy or dh may be null
  const float* rstd;
  void *dx, *dr;                 // dr: null where the residual's gradient is dx itself
  float* part;                   // (workgroups, C)
  int M, C, w_bf16, groups;      // groups of TPR threads in the launch
};

// A group of TPR threads takes the rows group, group + groups, ...; dw gathers in its
// registers (a thread keeps its columns), then over the workgroup's groups in LDS and, by
// norm_dw, over the workgroups, always in the same order.  The next row is in flight while one
// is worked on.  With a partial sum of dw for each wave and no row ahead 65536 x 768 bfloat16
// took 95 us, 4096 x 8192 87, 2048 x 2048 19; so 76 (5.3 TB/s), 44 and 12.  Rows past 8192 values
// with a float32 stream do not fit the registers of two waves a SIMD: 12 to 44 bytes a lane go
// through scratch memory (4096 x 16384 float32 213 us, 5.0 TB/s).
template <typename TX, typename TR, int TPR, int NCH, bool VEC>
__global__ void __launch_bounds__(kNT<TPR>) norm_bwd(NormBwdArgs a) {
  constexpr int NT = kNT<TPR>, NW = TPR / 64, NG = NT / TPR;
  __shared__ float s_sum[2][NW];
  __shared__ float s_dw[NG > 1 ? NG : 1][NG > 1 ? NCH * TPR * 8 : 1];
  const int tid = threadIdx.x % TPR;
  const int group = blockIdx.x * NG + threadIdx.x / TPR;
  float w[NCH][8], dw[NCH][8];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    load_w<VEC>(a.w, a.w_bf16, (j * TPR + tid) * 8, a.C, w[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[j][e] = 0.f;
  }
  Raw8<TR, VEC> rh[NCH], rg[NCH];
  Raw8<TX, VEC> ry[NCH];
  float r_next = 0.f;
  auto load = [&](long long row) {
    r_next = a.rstd[row];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = (j * TPR + tid) * 8;
      rh[j].load((const TR*)a.h + row * a.C, c, a.C);
      if (a.dy) ry[j].load((const TX*)a.dy + row * a.C, c, a.C);
      if (a.dh) rg[j].load((const TR*)a.dh + row * a.C, c, a.C);
    }
  };
  constexpr bool AHEAD = NCH <= 2;   // the registers of wider rows are full
  int flip = 0;
  if (AHEAD && group < a.M) load(group);
  for (long long row = group; row < a.M; row += a.groups, flip ^= 1) {
    if (!AHEAD) load(row);
    const float rstd = r_next;
    float n[NCH][8], d[NCH][8], sum = 0.f;
    Raw8<TR, VEC> g[NCH];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[j][e] = rh[j][e] * rstd;
        d[j][e] = a.dy ? ry[j][e] : 0.f;
      }
      g[j] = rg[j];
    }
    if (AHEAD && row + a.groups < a.M) load(row + a.groups);
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      float part = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[j][e] = fmaf(d[j][e], n[j][e], dw[j][e]);
        d[j][e] *= w[j][e];
        part = fmaf(d[j][e], n[j][e], part);
      }
      sum += part;
    }
    sum = wave_sum(sum);
    if constexpr (NW > 1) {
      if (tid % 64 == 0) s_sum[flip][tid / 64] = sum;   // two buffers: one barrier a row
      lds_barrier();
      sum = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) sum += s_sum[flip][k];
    }
    const float mean = sum / (float)a.C;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c = (j * TPR + tid) * 8;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o[e] = fmaf(rstd, d[j][e] - n[j][e] * mean, a.dh ? g[j][e] : 0.f);
      store8<TX, VEC>((TX*)a.dx + row * a.C, c, a.C, o);
      if (a.dr) store8<TR, VEC>((TR*)a.dr + row * a.C, c, a.C, o);
    }
  }
  if constexpr (NG > 1) {
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        store4(&s_dw[threadIdx.x / TPR][(j * TPR + tid) * 8 + e],
               f32x4{dw[j][e], dw[j][e + 1], dw[j][e + 2], dw[j][e + 3]});
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += NT) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NG; ++k) s += s_dw[k][c];
      a.part[(size_t)blockIdx.x * a.C + c] = s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NCH; ++j)
      store8<float, VEC>(a.part + (size_t)blockIdx.x * a.C, (j * TPR + tid) * 8, a.C, dw[j]);
  }
}

// dw[c] = sum over the partial sums, in a fixed order: 32 columns a workgroup, 32 groups of
// rows, then a tree.
__global__ void __launch_bounds__(1024) norm_dw(const float* part, int groups, int C, void* dw,
                                                int bf16) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32, c = blockIdx.x * 32 + tx;
  float sum = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int g = ty; g < groups; g += 32) sum += part[(size_t)g * C + c];
  }
  s[ty][tx] = sum;
  __syncthreads();
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    if (ty < m) s[ty][tx] += s[ty + m][tx];
    __syncthreads();
  }
  if (ty == 0 && c < C) {
    if (bf16)
      ((bf16_t*)dw)[c] = (bf16_t)s[0][tx];
    else
      ((float*)dw)[c] = s[0][tx];
  }
}

// ---------------------------------------------------------------- host side

// Workgroups along a grid's first axis, whose threads have to stay within 32 bits: norms go on
// along the second (walking over the rows instead keeps the weight in registers from row to
// row, and fewer waves in flight: 65536 x 768 in 8 bits 73 us, from 66), dequantize walks.
unsigned grid_of(long long wgs) { return (unsigned)(wgs < 65536 ? wgs : 65536); }

int validate(int M, int C, int x_dtype, int r_dtype, int w_dtype, int most = kMaxWidth) {
  if (M < 0 || C < 1 || C > most) return GDN2_ERR_SHAPE;
  if (x_dtype != GDN2_F32 && x_dtype != GDN2_BF16) return GDN2_ERR_DTYPE;
  if (r_dtype != GDN2_F32 && !(r_dtype == GDN2_BF16 && x_dtype == GDN2_BF16))
    return GDN2_ERR_DTYPE;
  if (w_dtype != GDN2_F32 && w_dtype != GDN2_BF16) return GDN2_ERR_DTYPE;
  return GDN2_OK;
}
size_t size_of(int dtype) { return dtype == GDN2_F32 ? 4 : 2; }
// Element-aligned (an error otherwise), and whether 16-byte accesses fit rows ld apart.
int check(const void* p, int dtype, long long ld, bool optional, bool* vec) {
  if (!p) return optional ? GDN2_OK : GDN2_ERR_NULL;
  if ((uintptr_t)p % size_of(dtype)) return GDN2_ERR_ALIGN;
  if ((uintptr_t)p % 16 || (ld * (long long)size_of(dtype)) % 16) *vec = false;
  return GDN2_OK;
}

// Threads and chunks of a row by its width.  WIDE: up to kMaxQuant (a norm's backward
// would not fit the registers of 1024 threads with 4 chunks).
template <bool WIDE, typename F>
void by_width(int C, F f) {
#define GDN2_W(TPR, NCH) \
  return f(std::integral_constant<int, TPR>{}, std::integral_constant<int, NCH>{})
  if (C <= 512) GDN2_W(64, 1);
  if (C <= 1024) GDN2_W(64, 2);
  if (C <= 2048) GDN2_W(128, 2);
  if (C <= 4096) GDN2_W(256, 2);
  if (C <= 8192) GDN2_W(512, 2);
  if (!WIDE || C <= 16384) GDN2_W(512, 4);
  if constexpr (WIDE) GDN2_W(1024, 4);
#undef GDN2_W
}
// Workgroups of the backward launch, each with a partial sum of dw; `per`: row groups of one.
// At most 2048 waves, two to a SIMD (4096: 65536 x 768 bfloat16 87 us, 2048 76; 16384 x 4096 113
// and 101), and, down to one workgroup a CU, at least four rows a group.
int bwd_workgroups(int M, int C, int* per) {
  int tpr = 64;
  by_width<false>(C, [&](auto t, auto) { tpr = decltype(t)::value; });
  *per = tpr == 64 ? 4 : 1;
  constexpr int WAVES = 2048;
  long long groups = WAVES / (tpr / 64);
  const long long few = M / 4 > 256 ? M / 4 : 256;
  if (groups > few) groups = few;
  if (groups > M) groups = M;
  return (int)((groups + *per - 1) / *per);
}

template <typename TX, typename TR, int MODE>
hipError_t launch_fwd(hipStream_t st, const NormArgs& a, bool vec) {
  by_width<MODE == kQuant>(a.C, [&](auto t, auto n) {
    constexpr int TPR = decltype(t)::value, NCH = decltype(n)::value;
    constexpr int NT = kNT<TPR>, ROWS = NT / TPR;
    const long long wgs = ((long long)a.M + ROWS - 1) / ROWS;
    const dim3 grid(grid_of(wgs), (unsigned)((wgs + 65535) / 65536)), block(NT);
    if (vec)
      hipLaunchKernelGGL((norm_fwd<TX, TR, MODE, TPR, NCH, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((norm_fwd<TX, TR, MODE, TPR, NCH, false>), grid, block, 0, st, a);
  });
  return hipGetLastError();
}
template <int MODE>
int launch_fwd(hipStream_t st, const NormArgs& a, int x_dtype, int r_dtype, bool vec) {
  hipError_t e;
  if constexpr (MODE == kQuant)
    e = x_dtype == GDN2_F32 ? launch_fwd<float, float, MODE>(st, a, vec)
                            : launch_fwd<bf16_t, bf16_t, MODE>(st, a, vec);
  else
    e = x_dtype == GDN2_F32   ? launch_fwd<float, float, MODE>(st, a, vec)
        : r_dtype == GDN2_F32 ? launch_fwd<bf16_t, float, MODE>(st, a, vec)
                              : launch_fwd<bf16_t, bf16_t, MODE>(st, a, vec);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}
template <typename TX, typename TR>
hipError_t launch_bwd(hipStream_t st, const NormBwdArgs& a, int wgs, bool vec) {
  by_width<false>(a.C, [&](auto t, auto n) {
    constexpr int TPR = decltype(t)::value, NCH = decltype(n)::value;
    constexpr int NT = kNT<TPR>;
    const dim3 grid((unsigned)wgs), block(NT);
    if (vec)
      hipLaunchKernelGGL((norm_bwd<TX, TR, TPR, NCH, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((norm_bwd<TX, TR, TPR, NCH, false>), grid, block, 0, st, a);
  });
  return hipGetLastError();
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

int gdn2_rms_norm(void* stream, int M, int C, int x_dtype, int r_dtype, int w_dtype,
                  const void* x, long long x_stride, const void* residual,
                  long long r_stride, const void* weight, float eps, void* y, void* h,
                  float* rstd) {
  int rc = validate(M, C, x_dtype, r_dtype, w_dtype);
  if (rc) return rc;
  if (!(eps >= 0.f)) return GDN2_ERR_SHAPE;
  if (M == 0) return GDN2_OK;
  bool vec = C % 8 == 0;
  if ((rc = check(x, x_dtype, x_stride, false, &vec)) ||
      (rc = check(residual, r_dtype, r_stride, true, &vec)) ||
      (rc = check(weight, w_dtype, 0, false, &vec)) || (rc = check(y, x_dtype, C, false, &vec)) ||
      (rc = check(h, r_dtype, C, !residual, &vec)) ||
      (rc = check(rstd, GDN2_F32, 0, true, &vec)))
    return rc;
  NormArgs a = {};
  a.x = x, a.ldx = x_stride, a.r = residual, a.ldr = r_stride, a.w = weight;
  a.y = y, a.h = h, a.rstd = rstd, a.eps = eps, a.M = M, a.C = C, a.w_bf16 = w_dtype == GDN2_BF16;
  return launch_fwd<kNorm>((hipStream_t)stream, a, x_dtype, r_dtype, vec);
}

int gdn2_rms_norm_int8(void* stream, int M, int C, int x_dtype, int r_dtype, int w_dtype,
                       const void* x, long long x_stride, const void* residual,
                       long long r_stride, const void* weight, float eps, void* q,
                       long long q_stride, float* scale, void* h) {
  int rc = validate(M, C, x_dtype, r_dtype, w_dtype);
  if (rc) return rc;
  if (!(eps >= 0.f) || q_stride < C) return GDN2_ERR_SHAPE;
  if (M == 0) return GDN2_OK;
  bool vec = C % 8 == 0, q_vec = true;
  if ((rc = check(x, x_dtype, x_stride, false, &vec)) ||
      (rc = check(residual, r_dtype, r_stride, true, &vec)) ||
      (rc = check(weight, w_dtype, 0, false, &vec)) ||
      (rc = check(h, r_dtype, C, !residual, &vec)) ||
      (rc = check(scale, GDN2_F32, 0, false, &q_vec)))
    return rc;
  if (!q) return GDN2_ERR_NULL;
  if ((uintptr_t)q % 16 || q_stride != (C + 15) / 16 * 16) return GDN2_ERR_ALIGN;
  NormArgs a = {};
  a.x = x, a.ldx = x_stride, a.r = residual, a.ldr = r_stride, a.w = weight;
  a.h = h, a.q = (signed char*)q, a.ldq = q_stride, a.scale = scale;
  a.eps = eps, a.M = M, a.C = C, a.w_bf16 = w_dtype == GDN2_BF16;
  return launch_fwd<kNorm8>((hipStream_t)stream, a, x_dtype, r_dtype, vec);
}

int gdn2_quantize_int8(void* stream, int M, int C, int x_dtype, const void* x,
                       long long x_stride, void* q, long long q_stride, float* scale) {
  int rc = validate(M, C, x_dtype, x_dtype, GDN2_F32, kMaxQuant);
  if (rc) return rc;
  if (q_stride < C) return GDN2_ERR_SHAPE;
  if (M == 0) return GDN2_OK;
  bool vec = C % 8 == 0, q_vec = true;
  if ((rc = check(x, x_dtype, x_stride, false, &vec)) ||
      (rc = check(scale, GDN2_F32, 0, false, &q_vec)))
    return rc;
  if (!q) return GDN2_ERR_NULL;
  if ((uintptr_t)q % 16 || q_stride != (C + 15) / 16 * 16) return GDN2_ERR_ALIGN;
  NormArgs a = {};
  a.x = x, a.ldx = x_stride, a.q = (signed char*)q, a.ldq = q_stride, a.scale = scale;
  a.M = M, a.C = C;
  return launch_fwd<kQuant>((hipStream_t)stream, a, x_dtype, x_dtype, vec);
}

int gdn2_dequantize_int8(void* stream, int M, int C, int out_dtype, const void* q,
                         long long q_stride, const float* scale, void* out) {
  int rc = validate(M, 1, out_dtype, out_dtype, GDN2_F32);
  if (rc) return rc;
  if (C < 1 || C > 0x7fffffff - 8) return GDN2_ERR_SHAPE;
  if (M == 0) return GDN2_OK;
  const long long n = (long long)M * ((C + 7ll) / 8);
  bool vec = C % 8 == 0, s_vec = true;
  if ((rc = check(out, out_dtype, C, false, &vec)) ||
      (rc = check(scale, GDN2_F32, 0, false, &s_vec)))
    return rc;
  if (!q) return GDN2_ERR_NULL;
  if ((uintptr_t)q % 8 || q_stride % 8) vec = false;
  const dim3 grid(grid_of((n + 255) / 256)), block(256);
  hipStream_t st = (hipStream_t)stream;
#define GDN2_DQ(T, VEC)                                                                   \
  hipLaunchKernelGGL((dequantize<T, VEC>), grid, block, 0, st, (const signed char*)q,     \
                     q_stride, scale, (T*)out, (long long)M, C)
  if (out_dtype == GDN2_F32) {
    if (vec) GDN2_DQ(float, true); else GDN2_DQ(float, false);
  } else {
    if (vec) GDN2_DQ(bf16_t, true); else GDN2_DQ(bf16_t, false);
  }
#undef GDN2_DQ
  return hipGetLastError() == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_rms_norm_bwd_workspace_bytes(int M, int C) {
  if (validate(M, C, GDN2_F32, GDN2_F32, GDN2_F32) != GDN2_OK) return 0;
  int per = 1;
  return (size_t)bwd_workgroups(M, C, &per) * C * sizeof(float);
}

int gdn2_rms_norm_bwd(void* stream, int M, int C, int x_dtype, int r_dtype, int w_dtype,
                      const void* h, const void* weight, const float* rstd, const void* dy,
                      const void* dh, void* dx, void* dr, void* dw, void* ws,
                      size_t ws_bytes) {
  int rc = validate(M, C, x_dtype, r_dtype, w_dtype);
  if (rc) return rc;
  bool vec = C % 8 == 0, any = true;
  if ((rc = check(dw, w_dtype, 0, false, &any))) return rc;
  const size_t need = gdn2_rms_norm_bwd_workspace_bytes(M, C);
  if (M > 0) {
    if ((rc = check(h, r_dtype, C, false, &vec)) || (rc = check(weight, w_dtype, 0, false, &vec)) ||
        (rc = check(rstd, GDN2_F32, 0, false, &any)) || (rc = check(dy, x_dtype, C, true, &vec)) ||
        (rc = check(dh, r_dtype, C, true, &vec)) || (rc = check(dx, x_dtype, C, false, &vec)) ||
        (rc = check(dr, r_dtype, C, true, &vec)) || (rc = check(ws, GDN2_F32, C, false, &vec)))
      return rc;
    if (ws_bytes < need) return GDN2_ERR_WORKSPACE;
  }
  NormBwdArgs a = {};
  a.h = h, a.w = weight, a.dy = dy, a.dh = dh, a.rstd = rstd, a.dx = dx, a.dr = dr;
  a.part = (float*)ws, a.M = M, a.C = C, a.w_bf16 = w_dtype == GDN2_BF16;
  int per = 1;
  const int wgs = bwd_workgroups(M, C, &per);
  a.groups = wgs * per;
  hipStream_t st = (hipStream_t)stream;
  hipError_t e = hipSuccess;
  if (M > 0)
    e = x_dtype == GDN2_F32   ? launch_bwd<float, float>(st, a, wgs, vec)
        : r_dtype == GDN2_F32 ? launch_bwd<bf16_t, float>(st, a, wgs, vec)
                              : launch_bwd<bf16_t, bf16_t>(st, a, wgs, vec);
  if (e != hipSuccess) return GDN2_ERR_LAUNCH;
  hipLaunchKernelGGL(norm_dw, dim3((unsigned)((C + 31) / 32)), dim3(1024), 0, st, a.part,
                     M > 0 ? wgs : 0, C, dw, w_dtype == GDN2_BF16);
  return hipGetLastError() == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

}  // extern "C"
