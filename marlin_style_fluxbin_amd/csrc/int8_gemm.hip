// Products of 8-bit rows (int8_launch.h): the sums in whole numbers on the int8 matrix cores, exact
// in any order, the scales and the bias in fp32, one rounding.
#include "int8_gemm.h"

namespace fx {
namespace {

// Four waves, each 32 rows of the weight by 32 of the activations, operands straight from memory.
__global__ __launch_bounds__(256) void int8_gemm_direct_kernel(const Int8GemmArgs g) {
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int r = lane & 15, k16 = (lane >> 4) * 16;
  const int n0 = int(blockIdx.x) * 64 + (wave & 1) * 32, m0 = int(blockIdx.y) * 64 + (wave >> 1) * 32;
  const int8_t *pw[2], *pa[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {  // rows past the last: the last again, not stored
    pw[t] = g.w + min(n0 + 16 * t + r, g.N - 1) * g.w_stride;
    pa[t] = g.a + min(m0 + 16 * t + r, g.M - 1) * g.a_stride;
  }
  i32x4_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = i32x4_t{0, 0, 0, 0};
  for (int k = k16; k - k16 < g.K; k += 64) {
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    u32x4_t w[2], a[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      w[t] = k < g.K ? *reinterpret_cast<const u32x4_t*>(pw[t] + k) : zero;
      a[t] = k < g.K ? *reinterpret_cast<const u32x4_t*>(pa[t] + k) : zero;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma_i8_16(w[i], a[j], acc[i][j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int m = m0 + 16 * j + r;
    if (m >= g.M) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = n0 + 16 * i + (lane >> 4) * 4;
      if (n < g.N) store4(g, m, n, acc[i][j]);
    }
  }
}

}  // namespace

Int8GemmPlan plan_int8_gemm(int M, int N, int K) { return {0, 1, K}; }

bool launch_int8_gemm(const Int8GemmPlan& plan, const Int8GemmArgs& g, hipStream_t s) {
  const dim3 grid(unsigned(g.N + 63) / 64, unsigned(g.M + 63) / 64);
  hipLaunchKernelGGL(int8_gemm_direct_kernel, grid, dim3(256), 0, s, g);
  return true;
}

}  // namespace fx
