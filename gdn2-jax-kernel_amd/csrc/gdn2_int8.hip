// Matrix product in 8-bit integers with a scale for each row of both operands:
//   out[m][n] = sx[m] sw[n] sum_k x[m][k] w[n][k]  (+ bias[n]),
// x (M,K) activations, w (N,K) weight, both with contiguous k.  The sums are exact in 32
// bits (K <= 131071), so no order of theirs can change a result; the scales are applied in
// float32 and the result is rounded once.
//
// Tiled kernel: BM x BN outputs a workgroup, 64-byte slices of k staged through LDS by
// global_load_lds in four buffers (three in flight), v_mfma_i32_16x16x64_i8.  The 16-byte
// pieces of a row are permuted within it by the row number, so that the eight lanes
// that LDS serves together read eight different bank groups; as the DMA writes LDS in lane
// order, the lanes' global addresses are permuted instead.  The weight is the left operand,
// its rows dealt to the fragments so that a lane ends up with eight neighbouring columns of
// one output row, stored as 16 bytes of bfloat16.
//
// Few rows (M <= 64): the weight's traffic is all that counts.  A workgroup takes 16
// weight rows and its eight waves the slices of k in turn, straight from memory to
// registers; their sums meet in LDS.
//
// k past K: rows are readable up to a multiple of 16 bytes, loads are clamped there, and
// the activations' bytes from K on are zeroed in the last slice.
#include <limits.h>

#include "gdn2.h"
#include "gdn2_common.h"

namespace gdn2 {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct MmArgs {
  const signed char *x, *w;
  long long ldx, ldw;          // bytes between rows
  const float *sx, *sw, *bias; // bias may be null
  void* out;                   // (M, N) dense
  int M, N, K;
  int tm, tn, chunk;           // tiles; tiles of one XCD
  int vec;                     // 16-byte stores fit
};

__device__ __forceinline__ i32x4 mma8(const i32x4& x, const i32x4& y, const i32x4& c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, c, 0, 0, 0);
}

// Zero the bytes of a 16-byte piece from byte n on (n may be <= 0 or >= 16).
__device__ __forceinline__ i32x4 keep_bytes(i32x4 v, int n) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int k = n - 4 * d;
    const unsigned mask = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
    v[d] = (int)((unsigned)v[d] & mask);
  }
  return v;
}

constexpr int kBK = 64, kStages = 4;

// Place of piece c of row r within its 64-byte row: activations' fragments read rows
// i = 0..15, the weight's rows 8 (i / 4) + i % 4 (+ 4).
__device__ __forceinline__ int swz_x(int r) { return (r >> 1) & 3; }
__device__ __forceinline__ int swz_w(int r) { return ((r >> 1) & 1) | ((r >> 2) & 2); }

template <int BM, int BN, int WR, int WC, typename TO>
__global__ void __launch_bounds__(64 * WR * WC) int8_mm(MmArgs a) {
  constexpr int NW = WR * WC, WM = BM / WR, WN = BN / WC;   // waves, and a wave's tile
  constexpr int MI = WM / 16, NI = WN / 16;
  constexpr int STAGE = (BM + BN) * kBK;
  constexpr int NL = STAGE / 1024 / NW;                     // DMA instructions of a wave
  static_assert(STAGE % (1024 * NW) == 0 && NI % 2 == 0 && BM % 16 == 0, "tile");
  __shared__ __attribute__((aligned(16))) char lds[kStages][STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & 15, lg = lane >> 4;

  // tiles: neighbours on one XCD, four rows of tiles before the next column
  const int item = (blockIdx.x & 7) * a.chunk + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= a.chunk || item >= a.tm * a.tn) return;
  const int group = item / (4 * a.tn), in_group = item - group * 4 * a.tn;
  const int rows = a.tm - 4 * group < 4 ? a.tm - 4 * group : 4;
  const int m0 = (4 * group + in_group % rows) * BM, n0 = (in_group / rows) * BN;

  // this lane's source of each DMA: row and piece of the staged tile
  const char* src[NL];
  int at[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = (wave * NL + i) * 16 + lane / 4, p = lane % 4;
    if (r < BM) {
      const int m = m0 + r < a.M ? m0 + r : a.M - 1;
      src[i] = (const char*)a.x + m * a.ldx;
      at[i] = 16 * (p ^ swz_x(r));
    } else {
      const int rn = r - BM, n = n0 + rn < a.N ? n0 + rn : a.N - 1;
      src[i] = (const char*)a.w + n * a.ldw;
      at[i] = 16 * (p ^ swz_w(rn));
    }
  }
  const int last = (a.K + 15) / 16 * 16 - 16;   // the last readable piece of a row
  auto load = [&](int kb) {
    char* dst = lds[kb % kStages] + wave * NL * 1024;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int k = kb * kBK + at[i];
      lds_dma16(src[i] + (k < last ? k : last), dst + i * 1024);
    }
  };

  const int wm = (wave / WC) * WM, wn = (wave % WC) * WN;
  i32x4 acc[NI][MI];
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[j][i] = i32x4{0, 0, 0, 0};

  const int nk = (a.K + kBK - 1) / kBK;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s)
    if (s < nk) load(s);
  for (int kb = 0; kb < nk; ++kb) {
    // slice kb has arrived once only the later ones (kStages - 2 of them) are in flight
    if (kb + kStages - 1 <= nk)
      wait_vmcnt<(kStages - 2) * NL>();
    else
      wait_vmcnt<0>();
    lds_barrier();   // also: every wave is done with slice kb - 1, whose buffer is next
    if (kb + kStages - 1 < nk) load(kb + kStages - 1);
    const char* sx = lds[kb % kStages];
    const char* sw = sx + BM * kBK;
    i32x4 fw[NI], fx[MI];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int r = wn + (j / 2) * 32 + (li / 4) * 8 + (j & 1) * 4 + li % 4;
      fw[j] = *reinterpret_cast<const i32x4*>(sw + r * kBK + 16 * (lg ^ swz_w(r)));
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = wm + i * 16 + li;
      fx[i] = *reinterpret_cast<const i32x4*>(sx + r * kBK + 16 * (lg ^ swz_x(r)));
    }
    if (kb * kBK + kBK > a.K) {
#pragma unroll
      for (int i = 0; i < MI; ++i) fx[i] = keep_bytes(fx[i], a.K - kb * kBK - 16 * lg);
    }
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int i = 0; i < MI; ++i) acc[j][i] = mma8(fw[j], fx[i], acc[j][i]);
  }

  // lane: row m = li of tile i, columns 8 lg .. 8 lg + 7 of the tile pair j, j + 1
  TO* out = (TO*)a.out;
#pragma unroll
  for (int j = 0; j < NI; j += 2) {
    const int n = n0 + wn + j * 16 + lg * 8;
    float sw[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int ne = n + e < a.N ? n + e : a.N - 1;
      sw[e] = a.sw[ne];
      bias[e] = a.bias ? a.bias[ne] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + wm + i * 16 + li;
      if (m >= a.M) continue;
      const float s = a.sx[m];
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = (float)acc[j + e / 4][i][e % 4] * s * sw[e];
        if (a.bias) y[e] += bias[e];
      }
      TO* p = out + (long long)m * a.N + n;
      if (a.vec && n + 8 <= a.N) {
        if constexpr (sizeof(TO) == 2) {
          *reinterpret_cast<bf16x8*>(p) = make_op(y, (bf16x8*)nullptr);
        } else {
          store4(p, f32x4{y[0], y[1], y[2], y[3]});
          store4(p + 4, f32x4{y[4], y[5], y[6], y[7]});
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < a.N) p[e] = from_f<TO>(y[e]);
      }
    }
  }
}

// 16 weight rows and all of x's (up to 16 MT) a workgroup; wave w takes the slices of 128
// bytes w, w + 8, ... of k.
template <int MT, typename TO>
__global__ void __launch_bounds__(512) int8_mm_rows(MmArgs a) {
  constexpr int NW = 8;
  __shared__ int sum[NW][MT][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int n = n0 + li < a.N ? n0 + li : a.N - 1;
  const char* w = (const char*)a.w + n * a.ldw;
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = i * 16 + li < a.M ? i * 16 + li : a.M - 1;
    x[i] = (const char*)a.x + m * a.ldx;
  }
  const int last = (a.K + 15) / 16 * 16 - 16;
  i32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = i32x4{0, 0, 0, 0};
  for (int k0 = wave * 128; k0 < a.K; k0 += NW * 128) {
    i32x4 fw[2], fx[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 64 * h + 16 * lg, kc = k < last ? k : last;
      fw[h] = *reinterpret_cast<const i32x4*>(w + kc);
#pragma unroll
      for (int i = 0; i < MT; ++i) fx[h][i] = *reinterpret_cast<const i32x4*>(x[i] + kc);
    }
    if (k0 + 128 > a.K) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          fx[h][i] = keep_bytes(fx[h][i], a.K - (k0 + 64 * h + 16 * lg));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = mma8(fw[h], fx[h][i], acc[i]);
  }
  // lane: columns 4 lg + r, row li
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[wave][i][li][4 * lg + r] = acc[i][r];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 256; e += 64 * NW) {
    const int m = e / 16, c = e % 16;
    if (m < a.M && n0 + c < a.N) {
      int s = 0;
#pragma unroll
      for (int k = 0; k < NW; ++k) s += sum[k][m / 16][m % 16][c];
      float y = (float)s * a.sx[m] * a.sw[n0 + c];
      if (a.bias) y += a.bias[n0 + c];
      ((TO*)a.out)[(long long)m * a.N + n0 + c] = from_f<TO>(y);
    }
  }
}

template <int BM, int BN, int WR, int WC, typename TO>
void launch_tiles(hipStream_t st, MmArgs a) {
  a.tm = (a.M + BM - 1) / BM;
  a.tn = (a.N + BN - 1) / BN;
  a.chunk = (a.tm * a.tn + 7) / 8;
  hipLaunchKernelGGL((int8_mm<BM, BN, WR, WC, TO>), dim3(8u * (unsigned)a.chunk),
                     dim3(64 * WR * WC), 0, st, a);
}

template <typename TO>
hipError_t launch_mm(hipStream_t st, const MmArgs& a) {
  const long long cus = num_cus();
  auto tiles = [&](int bm, int bn) {
    return (((long long)a.M + bm - 1) / bm) * (((long long)a.N + bn - 1) / bn);
  };
  if (a.M <= 64) {
    const dim3 grid((unsigned)((a.N + 15) / 16)), block(512);
    if (a.M <= 16)
      hipLaunchKernelGGL((int8_mm_rows<1, TO>), grid, block, 0, st, a);
    else if (a.M <= 32)
      hipLaunchKernelGGL((int8_mm_rows<2, TO>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((int8_mm_rows<4, TO>), grid, block, 0, st, a);
  } else if (tiles(256, 256) >= cus) {
    launch_tiles<256, 256, 2, 4, TO>(st, a);
  } else if (tiles(128, 128) >= cus) {
    launch_tiles<128, 128, 2, 2, TO>(st, a);
  } else {
    launch_tiles<128, 64, 2, 2, TO>(st, a);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" int gdn2_int8_matmul(void* stream, int M, int N, int K, int out_dtype, const void* x,
                                long long x_stride, const float* x_scale, const void* w,
                                long long w_stride, const float* w_scale, const float* bias,
                                void* out) {
  if (M < 0 || N < 1 || K < 1 || K > 131071) return GDN2_ERR_SHAPE;
  if (out_dtype != GDN2_F32 && out_dtype != GDN2_BF16) return GDN2_ERR_DTYPE;
  const long long row = (K + 15ll) / 16 * 16;
  if (x_stride < row || w_stride < row) return GDN2_ERR_SHAPE;
  // tiles are counted in 31 bits, and a tile's row numbers may pass the end by 255
  if (M > INT_MAX - 256 || N > INT_MAX - 256 ||
      ((M + 127ll) / 128) * ((N + 63ll) / 64) > (1ll << 30))
    return GDN2_ERR_SHAPE;
  if (M == 0) return GDN2_OK;
  const size_t es = out_dtype == GDN2_F32 ? 4 : 2;
  for (const void* p : {x, (const void*)x_scale, w, (const void*)w_scale, (const void*)out})
    if (!p) return GDN2_ERR_NULL;
  if ((uintptr_t)x % 16 || (uintptr_t)w % 16 || x_stride % 16 || w_stride % 16)
    return GDN2_ERR_ALIGN;
  if ((uintptr_t)x_scale % 4 || (uintptr_t)w_scale % 4 || (uintptr_t)bias % 4 ||
      (uintptr_t)out % es)
    return GDN2_ERR_ALIGN;
  MmArgs a = {};
  a.x = (const signed char*)x, a.w = (const signed char*)w, a.ldx = x_stride, a.ldw = w_stride;
  a.sx = x_scale, a.sw = w_scale, a.bias = bias, a.out = out, a.M = M, a.N = N, a.K = K;
  a.vec = (uintptr_t)out % 16 == 0 && ((size_t)N * es) % 16 == 0;
  const hipError_t e = out_dtype == GDN2_F32 ? launch_mm<float>((hipStream_t)stream, a)
                                             : launch_mm<bf16_t>((hipStream_t)stream, a);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}
