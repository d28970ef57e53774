// The launches of the short convolution, the selective scan and the 8-bit floating-point operators
// over sizes up to the largest that their entry points take, built with the kernels' host code alone by
// tests/test_launch_sizes_host.py.  The runtime's launch is defined here: it only looks at the
// grid, so no call needs a GPU and every pointer is a number that nothing follows.  A launch's threads
// have to stay below 2^32 along each axis; one that does not would be refused after the launches
// before it have run.  Exit status 0 when every check holds.
#include <hip/hip_runtime_api.h>

#include <climits>
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "gdn2.h"

static int g_fail = 0;
static long g_launches = 0, g_bad = 0;
static dim3 g_grid, g_block;

extern "C" {
void** __hipRegisterFatBinary(const void*) { static void* h; return &h; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*,
                           void*, int*) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t) {
  g_grid = grid, g_block = block;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
  *grid = g_grid, *block = g_block, *shared = 0, *stream = nullptr;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t, hipStream_t) {
  ++g_launches;
  auto fits = [](unsigned g, unsigned b) {
    return g > 0 && b > 0 && (unsigned long long)g * b < 1ull << 32;
  };
  const bool ok = fits(grid.x, block.x) && fits(grid.y, block.y) && fits(grid.z, block.z) &&
                  grid.y < 65536 && grid.z < 65536 && block.x * block.y * block.z <= 1024;
  g_bad += !ok;
  return ok ? hipSuccess : hipErrorInvalidConfiguration;
}
hipError_t hipGetLastError() { return g_bad ? hipErrorInvalidConfiguration : hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { *v = 256; return hipSuccess; }
}

// A call is refused before its first launch, or all of its launches fit.
static bool call(const char* what, long long a, long long b, long long c, long long d, int rc) {
  const bool taken = rc == GDN2_OK, ok = g_bad == 0 && taken == (g_launches > 0);
  if (!ok) {
    if (++g_fail <= 20)
      std::fprintf(stderr, "%s(%lld, %lld, %lld, %lld): %d after %ld launches, %ld too large\n", what, a,
                   b, c, d, rc, g_launches, g_bad);
  }
  g_launches = g_bad = 0;
  return taken;
}

static void* const p = (void*)(uintptr_t)0x100000;
static float* const f = (float*)p;
static const size_t kAll = ~(size_t)0 >> 1;
static const int kSizes[] = {1, 2, 3, 16, 64, 100, 768, 4096, 65536, 1 << 20, 4050000, 1 << 23,
                             13421772, 13421773, 14913081, 15999999, 1 << 24, 1 << 26, 1 << 27, 1 << 30,
                             INT_MAX - 1024, INT_MAX};
static long g_taken = 0, g_calls = 0;

static void conv() {
  for (int B : kSizes)
    for (int T : kSizes)
      for (int C : kSizes)
        for (int W : {2, 3, 4})
          for (int dt : {GDN2_F32, GDN2_BF16}) {
            const bool fwd = call("conv_fwd", B, T, C, W, gdn2_short_conv_fwd(
                nullptr, B, T, C, W, dt, 1, p, nullptr, f, f, nullptr, nullptr, p, p));
            const bool bwd = call("conv_bwd", B, T, C, W, gdn2_short_conv_bwd(
                nullptr, B, T, C, W, dt, 1, p, nullptr, f, f, nullptr, nullptr, p, nullptr, p, p, f, f,
                nullptr, p, kAll));
            g_fail += fwd != bwd;    // what runs forward runs backward
            g_taken += fwd + bwd, g_calls += 2;
            if (T == 1) {
              g_taken += call("conv_step", B, C, W, dt, gdn2_short_conv_step(
                  nullptr, B, C, W, dt, 1, p, f, f, p, p, p));
              ++g_calls;
            }
          }
}

static void scan() {
  const void* ins[5] = {p, p, p, p, p};
  void* outs[5] = {p, p, p, p, p};
  for (int B : kSizes)
    for (int T : kSizes)
      for (int C : kSizes)
        for (int G : {1, 2, 100, 65536, 1 << 18})
          for (int N : {1, 8, 16, 21, 64}) {
            if (C % G) continue;
            const bool fwd = call("scan_fwd", B, T, C, G * 100ll + N, gdn2_selective_scan_fwd(
                nullptr, B, T, C, G, N, GDN2_BF16, GDN2_F32, 1, ins, nullptr, f, f, f, nullptr, nullptr,
                p, f, f, p, kAll));
            const bool bwd = call("scan_bwd", B, T, C, G * 100ll + N, gdn2_selective_scan_bwd(
                nullptr, B, T, C, G, N, GDN2_F32, GDN2_F32, 1, ins, nullptr, f, f, f, nullptr, p,
                nullptr, f, f, outs, f, f, f, f, p, kAll));
            g_fail += fwd != bwd;
            g_taken += fwd + bwd, g_calls += 2;
            if (T == 1) {
              g_taken += call("scan_step", B, C, G, N, gdn2_selective_scan_step(
                  nullptr, B, C, G, N, GDN2_F32, GDN2_F32, 1, p, p, f, p, p, f, p, f, f, f, p));
              ++g_calls;
            }
          }
}

static void fp8() {
  for (int M : kSizes)
    for (int N : kSizes) {
      const long long up = (N + 15ll) / 16 * 16, down = (M + 15ll) / 16 * 16, two[2] = {1, 1};
      for (int dt : {GDN2_F32, GDN2_BF16}) {
        for (int blocks : {0, 1})
          g_taken += call("quantize", M, N, dt, blocks, gdn2_quantize_fp8(
              nullptr, M, N, dt, p, N, blocks, p, up, f, p, down, f, f, f)), ++g_calls;
        if (N <= INT_MAX - 256)
          g_taken += call("dequantize", M, N, dt, 0, gdn2_dequantize_fp8(
              nullptr, M, N, dt, p, up, 1, f, two, p)), ++g_calls;
        for (int K : kSizes) {
          const long long ld = (K + 15ll) / 16 * 16;
          for (int rows : {1, 128})
            g_taken += call("matmul", M, N, K, rows, gdn2_fp8_matmul(
                nullptr, M, N, K, dt, p, ld, f, M, p, ld, rows, f,
                rows == 1 ? N : (K + 127ll) / 128, f, p)), ++g_calls;
          const bool fwd = call("linear_fwd", M, N, K, dt, gdn2_fp8_linear_fwd(
              nullptr, M, N, K, dt, p, K, p, K, f, 1, 1, p, p, p, kAll));
          const bool bwd = call("linear_bwd", M, N, K, dt, gdn2_fp8_linear_bwd(
              nullptr, M, N, K, dt, p, N, p, 1, 1, p, p, f, p, kAll));
          g_fail += fwd != bwd;
          g_taken += fwd + bwd, g_calls += 2;
        }
      }
    }
}

int main() {
  conv();
  scan();
  fp8();
  std::printf("%ld calls, %ld taken, %d failures\n", g_calls, g_taken, g_fail);
  return g_fail || !g_taken ? 1 : 0;
}
