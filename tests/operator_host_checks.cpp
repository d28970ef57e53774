// Host-side checks of the entry points of the gated recurrence, the RMS norm and the 8-bit
// product, built without running device code under AddressSanitizer and
// UndefinedBehaviorSanitizer by tests/test_operators_host.py: sizes and refusals over shapes
// that include the extremes of int.  Every call that could launch is given a null pointer, so
// none does.  Exit status 0 when every check holds.
#include <climits>
#include <cstdint>
#include <cstdio>

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
  const int sizes[] = {INT_MIN, -1, 0, 1, 2, 16, 63, 64, 100, 512, 513, 1024, 4096, 16384, 16385,
                       32768, 131071, 131072, 1 << 24, 1 << 30, INT_MAX - 512, INT_MAX - 256,
                       INT_MAX - 255, INT_MAX};
  const int types[] = {-1, GDN2_F32, GDN2_BF16, GDN2_BF16_F32, INT_MAX};
  const long long strides[] = {LLONG_MIN, -16, 0, 16, 1 << 20, LLONG_MAX};
  void* p = (void*)(uintptr_t)0x100000;
  float* f = (float*)p;
  long n = 0;
  for (int a : sizes)
    for (int b : sizes)
      for (int c : sizes)
        for (int t : types) {
          const size_t kept = gdn2_gated_scan_kept_bytes(a, b, c, t);
          const size_t ws = gdn2_gated_scan_workspace_bytes(a, b, c, t);
          const int rc = gdn2_gated_scan_fwd(nullptr, a, b, c, t, GDN2_F32, p, nullptr, p, nullptr,
                                             nullptr, nullptr, nullptr, p, nullptr, f, p, ws);
          CHECK(rc < 0);   // h_final is null
          if (a < 1 || b < 0 || c < 1 || (t != GDN2_F32 && t != GDN2_BF16))
            CHECK(kept == 0 && ws == 0 && (rc == GDN2_ERR_SHAPE || rc == GDN2_ERR_DTYPE));
          if (rc == GDN2_ERR_NULL && b > 0) {
            // a state for at most 128 tokens each, and at least 512
            const double bc = (double)a * c;
            CHECK(kept >= bc * (b / 512) * 4 && kept <= bc * (b / 128 + 1.0) * 4);
            CHECK(b <= 512 ? ws == 0 : ws % 16 == 0);
          }
          CHECK(gdn2_gated_scan_bwd(nullptr, a, b, c, t, GDN2_F32, p, nullptr, p, nullptr, nullptr,
                                    nullptr, nullptr, nullptr, nullptr, nullptr, p, p, nullptr,
                                    nullptr, p, ws) < 0);
          for (long long s : strides)
            CHECK(gdn2_int8_matmul(nullptr, a == 0 ? 1 : a, b, c, t, p, s, f, p, s, f, nullptr,
                                   nullptr) < 0);
          n += 5;
        }
  for (int m : sizes)
    for (int c : sizes)
      for (int t : types) {
        const size_t ws = gdn2_rms_norm_bwd_workspace_bytes(m, c);
        if (m < 0 || c < 1 || c > 16384) CHECK(ws == 0);
        const int rows = m == 0 ? 1 : m;
        CHECK(gdn2_rms_norm(nullptr, rows, c, t, t, GDN2_F32, p, c, nullptr, 0, p, 0.f, nullptr,
                            nullptr, nullptr) < 0);
        CHECK(gdn2_rms_norm_int8(nullptr, rows, c, t, t, GDN2_F32, p, c, nullptr, 0, p, 0.f,
                                 nullptr, ((long long)c + 15) / 16 * 16, f, nullptr) < 0);
        CHECK(gdn2_rms_norm_bwd(nullptr, m, c, t, t, GDN2_F32, p, p, f, p, p, p, nullptr, nullptr,
                                p, ws) < 0);
        CHECK(gdn2_quantize_int8(nullptr, rows, c, t, p, c, nullptr,
                                 ((long long)c + 15) / 16 * 16, f) < 0);
        CHECK(gdn2_dequantize_int8(nullptr, rows, c, t, nullptr, c, f, p) < 0);
        n += 6;
      }
  for (long long k : strides)
    for (int t : types)
      CHECK(gdn2_gated_scan_step(nullptr, k == 0 ? 1 : k, t, t, p, p, nullptr, nullptr, nullptr,
                                 p) < 0);
  std::printf("%ld calls, %d failures\n", n, g_fail);
  return g_fail ? 1 : 0;
}
