// Host-side checks of the entry points of the short convolution, the selective scan and the 8-bit
// floating-point operators, built without running device code under AddressSanitizer and
// UndefinedBehaviorSanitizer by tests/test_state_space_host.py: sizes and refusals over shapes
// that include the extremes of int.  Every call that could launch is given a null pointer, so
// none does.  Exit status 0 when every check holds.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "gdn2.h"

static int g_fail = 0;
#define CHECK(cond)                                                           \
  do {                                                                        \
    if (!(cond)) {                                                            \
      std::fprintf(stderr, "check failed at line %d: %s\n", __LINE__, #cond); \
      ++g_fail;                                                               \
    }                                                                         \
  } while (0)

int main() {
  const int sizes[] = {INT_MIN, -1, 0, 1, 2, 3, 16, 63, 64, 100, 513, 4096, 1 << 17, 1 << 18,
                       1 << 24, (1 << 24) + 1, 1 << 30, INT_MAX - 1024, INT_MAX - 256, INT_MAX};
  const int few[] = {INT_MIN, -1, 0, 1, 2, 3, 4, 16, 64, 65, INT_MAX};
  const int types[] = {-1, GDN2_F32, GDN2_BF16, GDN2_BF16_F32, INT_MAX};
  const long long strides[] = {LLONG_MIN, -16, 0, 16, 1 << 20, 1ll << 25, LLONG_MAX};
  void* p = (void*)(uintptr_t)0x100000;
  float* f = (float*)p;
  const void* ins[5] = {p, p, p, p, p};
  void* outs[5] = {p, p, p, p, p};
  void* none[5] = {};
  long n = 0;
  for (int b : sizes)
    for (int t : sizes)
      for (int c : sizes) {
        for (int w : few) {
          const size_t ws = gdn2_short_conv_bwd_workspace_bytes(b, t, c, w);
          if (b < 1 || t < 1 || c < 1 || w < 2 || w > 4) CHECK(ws == 0);
          if (ws) CHECK(ws >= (size_t)b * c * (w + 1) * 4);
          for (int ty : types) {
            CHECK(gdn2_short_conv_fwd(nullptr, b, t, c, w, ty, 1, p, nullptr, f, f, p, nullptr, p,
                                      nullptr) < 0);
            CHECK(gdn2_short_conv_bwd(nullptr, b, t, c, w, ty, 1, p, nullptr, f, f, p, nullptr, p,
                                      nullptr, p, nullptr, f, f, p, p, ws) < 0);
            n += 2;
          }
        }
        for (int g : few)
          for (int s : {-1, 0, 1, 7, 16, 33, 64, 65}) {
            const size_t kept = gdn2_selective_scan_kept_bytes(b, t, c, g, s);
            const size_t wf = gdn2_selective_scan_workspace_bytes(b, t, c, g, s, 0);
            const size_t wb = gdn2_selective_scan_workspace_bytes(b, t, c, g, s, 1);
            if (b < 1 || t < 1 || c < 1 || g < 1 || s < 1 || s > 64 || c % (g > 0 ? g : 1))
              CHECK(wf == 0 && wb == 0);
            if (kept && t > 0) {
              CHECK(kept >= ((double)b * c * ((t + 15) / 16) * s + 2.0 * b * t * g * s) * 4);
              CHECK(wf >= 2.0 * b * t * g * s * 4 && wb % 16 == 0 && wf % 16 == 0);
            }
            CHECK(gdn2_selective_scan_fwd(nullptr, b, t, c, g, s, GDN2_BF16, GDN2_F32, 1, ins,
                                          nullptr, f, f, f, f, nullptr, nullptr, f, f, p, wf) < 0);
            CHECK(gdn2_selective_scan_bwd(nullptr, b, t, c, g, s, GDN2_F32, GDN2_F32, 1, ins,
                                          nullptr, f, f, f, nullptr, p, nullptr, f, f, none, f, f,
                                          f, f, p, wb) < 0);
            n += 5;
          }
      }
  for (long long st : strides) {
    const long long all[10] = {st, st, st, st, st, st, st, st, st, st};
    CHECK(gdn2_selective_scan_fwd(nullptr, 2, 5, 8, 2, 4, GDN2_F32, GDN2_F32, 0, ins, all, f, f, f,
                                  f, nullptr, nullptr, f, f, p, 1 << 20) < 0);
    CHECK(gdn2_selective_scan_bwd(nullptr, 2, 5, 8, 2, 4, GDN2_F32, GDN2_F32, 0, ins, all, f, f, f,
                                  nullptr, p, all, f, f, outs, nullptr, f, f, f, p, 1 << 24) < 0);
    n += 2;
  }
  for (int m : sizes)
    for (int k : sizes)
      for (int nn : sizes) {
        const size_t kb = gdn2_fp8_linear_kept_bytes(m, nn, k, 1, 1);
        const size_t wf = gdn2_fp8_linear_workspace_bytes(m, nn, k, 0);
        const size_t wb = gdn2_fp8_linear_workspace_bytes(m, nn, k, 1);
        if (m < 1 || nn < 1 || k < 1) CHECK(kb == 0 && wf == 0 && wb == 0);
        if (kb) CHECK(kb >= (double)k * m + (double)k * nn && wf >= ((double)m + nn) * k);
        const int rows = m == 0 ? 1 : m;
        for (int ty : types) {
          CHECK(gdn2_fp8_linear_fwd(nullptr, rows, nn, k, ty, p, k, p, k, f, 1, 1, nullptr, p, p,
                                    wf) < 0);
          CHECK(gdn2_fp8_linear_bwd(nullptr, m, nn, k, ty, nullptr, nn, p, 1, 1, p, p, f, p, wb) < 0);
          for (long long s : strides) {
            CHECK(gdn2_fp8_matmul(nullptr, rows, nn, k, ty, p, s, f, s, p, s, 128, f, s, f,
                                  nullptr) < 0);
            CHECK(gdn2_quantize_fp8(nullptr, rows, k, ty, nullptr, s, 0, p,
                                    ((long long)k + 15) / 16 * 16, f, nullptr, 0, nullptr, nullptr,
                                    nullptr) < 0);
            n += 2;
          }
          const long long two[2] = {1, 1};
          CHECK(gdn2_dequantize_fp8(nullptr, rows, k, ty, p, 16, 1, f, two, nullptr) < 0);
          n += 3;
        }
      }
  for (int b : sizes)
    for (int c : sizes)
      for (int g : few) {
        const int rows = b == 0 ? 1 : b;
        CHECK(gdn2_short_conv_step(nullptr, rows, c, 4, GDN2_F32, 1, p, f, f, p, p, nullptr) < 0);
        CHECK(gdn2_selective_scan_step(nullptr, rows, c, g, 16, GDN2_F32, GDN2_F32, 1, p, p, f, p, p,
                                       f, p, f, f, f, nullptr) < 0);
        n += 2;
      }
  std::printf("%ld calls, %d failures\n", n, g_fail);
  return g_fail ? 1 : 0;
}
