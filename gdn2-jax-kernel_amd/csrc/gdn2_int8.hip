// Matrix product in 8-bit integers with a scale for each row of both operands:
//   out[m][n] = sx[m] sw[n] sum_k x[m][k] w[n][k]  (+ bias[n]),
// x (M,K) activations, w (N,K) weight, both with contiguous k.  The sums are exact in 32
// bits (K <= 131071), so no order of theirs can change a result; the scales are applied in
// float32 and the result is rounded once.
//
// Tiled kernel: BM x BN outputs a workgroup, slices of 128 bytes of k staged through LDS by
// global_load_lds in a ring, v_mfma_i32_16x16x64_i8 (the 32x32x32 form reaches 3.4 P/s from
// registers, this one 4.0).  Half a slice is multiplied while the other's fragments are
// read.  Slices of whole cache lines: with 64 bytes 128 x 128 tiles reach 1.65 P/s at
// 8192 x 8192 x 8192, with 128 2.08; 192 x 128 reach 2.20 (the traffic from L2 and through LDS
// bounds them, which is read without conflicts, not the matrix cores, 51% busy).  The 16-byte
// pieces of a row are permuted within it by the row number, so that the eight lanes that LDS
// serves together read different banks; as the DMA writes LDS in lane order, the lanes' global
// addresses are permuted instead.  The weight is the left operand, its rows dealt to the fragments so that a lane
// ends up with eight neighbouring columns of one output row.  Several workgroups share a CU, so
// that one's start and stores pass under another's products (one that walks over many
// tiles and loads ahead instead waits for its stores: 65536 x 4608 x 768 418 us against 372).
// Where K is short the stores still add to the loads: 65536 x 4608 x 768 takes 308-322 us (1.4-1.5
// P/s), without its stores 223, without its products 270, its stores alone 110.
//
// Few rows: the weight's traffic is all that counts.  A workgroup takes 16 weight rows and
// its eight waves the slices of k in turn, straight from memory to registers; their sums meet
// in LDS.
//
// k past K: rows are readable up to a multiple of 16 bytes, loads are clamped there, and
// the activations' bytes from K on are zeroed in the last slice.
#include <limits.h>

#include "gdn2.h"
#include "gdn2_common.h"

namespace gdn2 {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
// 16 bytes at any value of TO: rows of results start where N puts them (32768 x 1500 x 1000 with
// bfloat16 results 80 us, stored value by value 155)
template <typename TO>
struct __attribute__((packed, aligned(sizeof(TO)))) Piece {
  i32x4 v;
};

struct MmArgs {
  const signed char *x, *w;
  long long ldx, ldw;          // bytes between rows
  const float *sx, *sw, *bias; // bias may be null
  void* out;                   // (M, N) dense
  int M, N, K;
  int tm, tn, chunk;           // tiles; tiles of one XCD
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

// Bytes of k of a slice: whole 128-byte lines.
constexpr int kBK = 128;

// Place of 16-byte piece c of row r within its slice: piece c ^ swz(r).  Activations'
// fragments read rows i = 0..15, the weight's rows 8 (i / 4) + i % 4 (+ 4).
__device__ __forceinline__ int swz_x(int r) { return r & 7; }
__device__ __forceinline__ int swz_w(int r) { return (r & 3) | ((r >> 1) & 4); }

// The 16-byte pieces of two halves of a row's columns, as lanes 16 lg + li hold them for rows
// li = 0..15 (t0: the first half, t1: the second), dealt so that t0 holds both halves of the
// rows 0..7 and t1 those of the rows 8..15: lanes li and li ^ 8 exchange a piece.  Each of
// the two stores that follow then writes 128 bytes of eight rows, not 64 of sixteen.
__device__ __forceinline__ void whole_lines(i32x4& t0, i32x4& t1) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    // row_ror:8, written to the lanes 8..15 of a row alone, and to 0..7
    const int first = t0[d];
    t0[d] = __builtin_amdgcn_update_dpp(first, t1[d], 0x128, 0xF, 0xC, false);
    t1[d] = __builtin_amdgcn_update_dpp(t1[d], first, 0x128, 0xF, 0x3, false);
  }
}

// Eight values from column n on of a vector of N, those past the end repeating the last.
__device__ __forceinline__ void load_columns(const float* v, int n, int N, float (&f)[8]) {
  if (n + 8 <= N) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const i32x4 r = reinterpret_cast<const Piece<float>*>(v + n)[h].v;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * h + e] = __int_as_float(r[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = v[n + e < N ? n + e : N - 1];
  }
}

// The scales of a wave's part from row m and column n on: rows 16 i + li, columns
// 32 j + 8 lg + e.
template <int NI, int MI>
struct Scales {
  float row[MI], col[NI / 2][8];
  __device__ __forceinline__ void load(const MmArgs& a, int m, int n, int li, int lg) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = m + 16 * i + li;
      row[i] = a.sx[r < a.M ? r : a.M - 1];
    }
#pragma unroll
    for (int j = 0; j < NI / 2; ++j) load_columns(a.sw, n + 32 * j + 8 * lg, a.N, col[j]);
  }
};

// Scale, convert and store a wave's part: the fragment pair 2 j, 2 j + 1 of tile i holds row li,
// columns 32 j + 8 lg + e.  m, n: its first row and column.
template <typename TO, int NI, int MI>
__device__ __forceinline__ void store_part(const MmArgs& a, const i32x4 (&acc)[NI][MI], int m,
                                           int n, int li, int lg, const Scales<NI, MI>& sc) {
  // before the first store, which could alias it for all the compiler knows
  float bi[NI / 2][8];
#pragma unroll
  for (int j = 0; j < NI / 2; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) bi[j][e] = 0.f;
    if (a.bias) load_columns(a.bias, n + 32 * j + 8 * lg, a.N, bi[j]);
  }
  auto result = [&](int i, int j, float (&y)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e] = fmaf((float)acc[2 * j + e / 4][i][e % 4] * sc.row[i], sc.col[j][e], bi[j][e]);
  };
  auto piece = [](const float (&y)[8], int half) {   // float32: the half of it
    i32x4 r;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if constexpr (sizeof(TO) == 4)
        r[d] = __float_as_int(y[4 * half + d]);
      else
        r[d] = __builtin_bit_cast(int, bf16x2{(bf16_t)y[2 * d], (bf16_t)y[2 * d + 1]});
    }
    return r;
  };
  TO* out = (TO*)a.out + (long long)m * a.N + n;
  if ((sizeof(TO) == 4 || NI % 4 == 0) && n + 16 * NI <= a.N && m + 16 * MI <= a.M) {
    // two halves of 128 bytes: float32 the two pieces of 8 values, bfloat16 two fragment pairs
    const bool high = li >= 8;
    constexpr int STEP = sizeof(TO) == 4 ? 1 : 2;
    TO* p = out + (long long)(li & 7) * a.N + 8 * lg + (sizeof(TO) == 4 ? 4 : 32) * high;
#pragma unroll
    for (int i = 0; i < MI; ++i, p += 16ll * a.N)
#pragma unroll
      for (int j = 0; j + STEP <= NI / 2; j += STEP) {
        float y0[8], y1[8];
        result(i, j, y0);
        if constexpr (STEP == 2) result(i, j + 1, y1);
        i32x4 t0 = piece(y0, 0), t1 = piece(STEP == 2 ? y1 : y0, 1);
        whole_lines(t0, t1);
        reinterpret_cast<Piece<TO>*>(p + 32 * j)->v = t0;
        reinterpret_cast<Piece<TO>*>(p + 8ll * a.N + 32 * j)->v = t1;
      }
    return;
  }
  TO* p = out + (long long)li * a.N + 8 * lg;
#pragma unroll
  for (int i = 0; i < MI; ++i, p += 16ll * a.N)
    if (m + 16 * i + li < a.M) {
#pragma unroll
      for (int j = 0; j < NI / 2; ++j) {
        float y[8];
        result(i, j, y);
        const int left = a.N - (n + 32 * j + 8 * lg);
        if (left >= 8) {
          Piece<TO>* q = reinterpret_cast<Piece<TO>*>(p + 32 * j);
          q[0].v = piece(y, 0);
          if constexpr (sizeof(TO) == 4) q[1].v = piece(y, 1);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) p[32 * j + e] = from_f<TO>(y[e]);
        }
      }
    }
}

// BM x BN outputs; WR x WC waves; ST slices of k in LDS; PER_CU workgroups on a CU.
template <int BM_, int BN_, int WR_, int WC_, int ST_, int PER_CU_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WR = WR_, WC = WC_, ST = ST_, PER_CU = PER_CU_;
  static constexpr int NW = WR * WC, WM = BM / WR, WN = BN / WC;   // waves, and a wave's part
  static constexpr int MI = WM / 16, NI = WN / 16;
  static constexpr int STAGE = (BM + BN) * kBK;
  static constexpr int NL = STAGE / 1024 / NW;                     // DMA instructions of a wave
  static_assert(STAGE % (1024 * NW) == 0 && NI % 2 == 0 && BM % 16 == 0, "tile");
};

template <typename C, typename TO>
__global__ void __launch_bounds__(64 * C::NW, C::NW * C::PER_CU / 4) int8_mm(MmArgs a) {
  constexpr int BM = C::BM, BN = C::BN, NW = C::NW, MI = C::MI, NI = C::NI, NL = C::NL;
  constexpr int ST = C::ST;
  __shared__ __attribute__((aligned(16))) char lds[ST * C::STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, lg = lane >> 4;

  // Tiles: neighbours on one XCD, eight rows of tiles before the next column, so that what runs
  // together on an XCD shares rows and columns in its L2 (65536 x 4608 x 768 with 2, 4, 8, 16, 32
  // rows 367, 338, 334, 331, 366 us; 8192 x 8192 x 2048 169, 150, 151, 155, 184).
  constexpr int GROUP = 8;
  const int item = (blockIdx.x & 7) * a.chunk + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= a.chunk || item >= a.tm * a.tn) return;
  const int group = item / (GROUP * a.tn), in_group = item - group * GROUP * a.tn;
  const int rows = a.tm - GROUP * group < GROUP ? a.tm - GROUP * group : GROUP;
  const int m0 = (GROUP * group + in_group % rows) * BM, n0 = (in_group / rows) * BN;

  // the source of each DMA: eight rows of one operand from a wave's address on, this lane's
  // row and piece of the slice in 32 bits
  const char* base[NL];
  unsigned off[NL];
  int at[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const bool act = (wave * NL + i) * 8 < BM;
    const int r = (wave * NL + i) * 8 + lane / 8 - (act ? 0 : BM);
    const int most = act ? a.M - 1 - m0 : a.N - 1 - n0;
    at[i] = 16 * (lane % 8 ^ (act ? swz_x(r) : swz_w(r)));
    base[i] = (const char*)(act ? a.x + m0 * a.ldx : a.w + n0 * a.ldw);
    off[i] = (unsigned)(r < most ? r : most) * (unsigned)(act ? a.ldx : a.ldw) + at[i];
  }
  const int last = (a.K + 15) / 16 * 16 - 16;   // the last readable piece of a row
  auto load = [&](int kb, int buf) {
    char* dst = lds + buf * C::STAGE + wave * NL * 1024;
    if ((kb + 1) * kBK <= last + 16) {
#pragma unroll
      for (int i = 0; i < NL; ++i) lds_dma16(base[i] + kb * kBK + (size_t)off[i], dst + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int past = kb * kBK + at[i] - last;
        lds_dma16(base[i] + kb * kBK + (long long)off[i] - (past > 0 ? past : 0), dst + i * 1024);
      }
    }
  };

  // this lane's fragments in a slice; the slice's second half is 64 bytes on (^ 64)
  const int wm = (wave / C::WC) * C::WM, wn = (wave % C::WC) * C::WN;
  int rw[NI], rx[MI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int r = wn + (j / 2) * 32 + (li / 4) * 8 + (j & 1) * 4 + li % 4;
    rw[j] = (BM + r) * kBK + 16 * (lg ^ swz_w(r));
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int r = wm + i * 16 + li;
    rx[i] = r * kBK + 16 * (lg ^ swz_x(r));
  }
  struct Frags {
    i32x4 w[NI], x[MI];
  };
  auto read = [&](Frags& f, int buf, int half) {
    const char* s = lds + buf * C::STAGE;
#pragma unroll
    for (int j = 0; j < NI; ++j) f.w[j] = *reinterpret_cast<const i32x4*>(s + (rw[j] ^ half));
#pragma unroll
    for (int i = 0; i < MI; ++i) f.x[i] = *reinterpret_cast<const i32x4*>(s + (rx[i] ^ half));
  };
  i32x4 acc[NI][MI];
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[j][i] = i32x4{0, 0, 0, 0};
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[j][i] = mma8(f.w[j], f.x[i], acc[j][i]);
  };

  // read first, used last: at the end they would be waited for (65536 x 4608 x 768 329 us, so 322)
  Scales<NI, MI> scales;
  scales.load(a, m0 + wm, n0 + wn, li, lg);
  const int nk = (a.K + kBK - 1) / kBK;
#pragma unroll
  for (int s = 0; s < ST; ++s)
    if (s < nk) load(s, s);
  if (nk >= ST)
    wait_vmcnt<(ST - 1) * NL>();
  else
    wait_vmcnt<0>();
  lds_barrier();
  // a half slice is multiplied while the next one is read
  Frags f0, f1;
  read(f0, 0, 0);
  for (int k0 = 0; k0 < nk; k0 += ST) {
#pragma unroll
    for (int buf = 0; buf < ST; ++buf) {
      const int kb = k0 + buf;
      if (kb >= nk) break;
      read(f1, buf, 64);
      if (kb * kBK + kBK > a.K) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          f0.x[i] = keep_bytes(f0.x[i], a.K - kb * kBK - 16 * lg);
          f1.x[i] = keep_bytes(f1.x[i], a.K - kb * kBK - 64 - 16 * lg);
        }
      }
      multiply(f0);
      // slice kb + 1 has arrived once only the ST - 2 later ones are in flight; every wave has
      // read slice kb, whose buffer is free
      if (kb + ST <= nk)
        wait_vmcnt<(ST - 2) * NL>();
      else
        wait_vmcnt<0>();
      lds_barrier();
      if (kb + ST < nk) load(kb + ST, buf);
      read(f0, (buf + 1) % ST, 0);   // after the last slice: stale data that nothing uses
      multiply(f1);
    }
  }

  store_part<TO>(a, acc, m0 + wm, n0 + wn, li, lg, scales);
}

// 16 weight rows and all of x's (up to 16 MT) a workgroup; wave w takes the slices of 128
// bytes w, w + 8, ... of k.
template <int MT, typename TO>
__global__ void __launch_bounds__(512) int8_mm_rows(MmArgs a) {
  constexpr int NW = 8;
  __shared__ int sum[NW][MT][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int n = n0 + li < a.N ? n0 + li : a.N - 1;
  const char* w = (const char*)a.w + n * a.ldw;
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + i * 16 + li < a.M ? m0 + i * 16 + li : a.M - 1;
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
    const int ml = e / 16, c = e % 16, m = m0 + ml;
    if (m < a.M && n0 + c < a.N) {
      int s = 0;
#pragma unroll
      for (int k = 0; k < NW; ++k) s += sum[k][ml / 16][ml % 16][c];
      const float y = fmaf((float)s * a.sx[m], a.sw[n0 + c], a.bias ? a.bias[n0 + c] : 0.f);
      ((TO*)a.out)[(long long)m * a.N + n0 + c] = from_f<TO>(y);
    }
  }
}

template <typename C, typename TO>
void launch_tiles(hipStream_t st, MmArgs a) {
  a.tm = (a.M + C::BM - 1) / C::BM;
  a.tn = (a.N + C::BN - 1) / C::BN;
  a.chunk = (a.tm * a.tn + 7) / 8;
  hipLaunchKernelGGL((int8_mm<C, TO>), dim3(8u * (unsigned)a.chunk), dim3(64 * C::NW), 0, st, a);
}
template <int MT, typename TO>
void launch_rows(hipStream_t st, const MmArgs& a) {
  hipLaunchKernelGGL((int8_mm_rows<MT, TO>),
                     dim3((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * MT - 1) / (16 * MT))),
                     dim3(512), 0, st, a);
}

template <typename TO>
hipError_t launch_mm(hipStream_t st, const MmArgs& a) {
  // (M x N x K, bfloat16 results, one kernel, us)
  const int cus = num_cus();
  auto tiles = [&](int bm, int bn) {
    return (((long long)a.M + bm - 1) / bm) * (((long long)a.N + bn - 1) / bn);
  };
  // Few rows, or few columns of few rows: 1 x 4608 x 768 2.9 (64 x 64 tiles: 4.0),
  // 8 x 8192 x 8192 14.3 (18.7), 32 x 4096 x 4096 7.6 (10.6), 500 x 200 x 300 2.8 (4.0),
  // 128 x 64 x 8192 12.3 (16.8); but 64 x 4608 x 768 5.2 (4.6), 300 x 1024 x 8192 33.6 (18.4).
  if (a.M <= 16) {
    launch_rows<1, TO>(st, a);
  } else if (a.M <= 32 || tiles(32, 16) <= cus) {
    launch_rows<2, TO>(st, a);
    // All tiles at once on the CUs, three each: 512 x 4096 x 4096 15.8 (128 x 128: 24.0),
    // 1024 x 2048 x 2048 10.0 (14.2); but 3000 x 3000 x 3000, 2209 tiles, 55.4 (47.7).
  } else if (tiles(64, 64) <= 3 * cus) {
    launch_tiles<Tile<64, 64, 2, 2, 3, 3>, TO>(st, a);
  } else {
    // 192 x 128 does a unit of work in 0.92 of the time of 128 x 128 (8192 x 8192 x 8192 500 and
    // 530, 65536 x 4608 x 768 308 and 336) where the rounds of two workgroups a CU come
    // out as well: 3000 x 3000 x 3000 37.8 and 47.7, but 4096 x 4096 x 4096 71.6 and 69.3,
    // 16384 x 512 x 1024 16.9 and 14.5.  A last round that is not full counts half as one.
    auto cost = [&](int bm, double unit) {
      const double r = (double)tiles(bm, 128) / (2 * cus);
      return (r < 1 ? 1 : (r + (double)(long long)(r + 0.999999)) / 2) * bm * unit;
    };
    if (cost(192, 0.92) < cost(128, 1.0))
      launch_tiles<Tile<192, 128, 2, 2, 2, 2>, TO>(st, a);
    else
      launch_tiles<Tile<128, 128, 2, 2, 2, 2>, TO>(st, a);
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
  // rows of a tile are reached in 32 bits
  if (x_stride > (1 << 24) || w_stride > (1 << 24)) return GDN2_ERR_SHAPE;
  // a launch's threads stay within 32 bits (128 x 128 tiles of 256, 16 columns of 512), and a
  // tile's row numbers, which may pass the end by 255, within 31
  if (M > INT_MAX - 256 || N > (1 << 26) || ((M + 127ll) / 128) * ((N + 127ll) / 128) > (1ll << 23))
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
  const hipError_t e = out_dtype == GDN2_F32 ? launch_mm<float>((hipStream_t)stream, a)
                                             : launch_mm<bf16_t>((hipStream_t)stream, a);
  return e == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}
