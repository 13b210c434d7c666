// Products of few 8-bit rows (a decode step, a small batch): the weight is read once, straight into
// the matrix cores' operands.
#pragma once
#include "int8_gemm.h"

namespace fx {

// 16 rows of the weight by at most 16 of the activations a workgroup, its W waves dealing the
// columns in pieces of 128: a wave's sums are over its own columns and are added through LDS, so that
// one launch has a burst of the whole weight in flight.  Bound by the weight's bytes (24576 x 4096 at
// one row 19.7 us, 5.1 TB/s; 4096 x 4096 5.1 us, of which a launch is 4): every wave issues UN pieces'
// loads in front of its first product (left to the compiler's order, 20.4).  32 rows of the weight a
// workgroup took 7.2 us for 5.1, two tiles of activations more than int8_gemm_tile.h.
template <int W, int UN>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(1, 4))) void int8_gemm_few_kernel(const Int8GemmArgs g) {
  __shared__ i32x4_t sums[W][64];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int r = lane & 15, k16 = (lane >> 4) * 16;
  const int n0 = xcd_local_index8(blockIdx.x, gridDim.x) * 16;
  const int w_stride = int(g.w_stride), a_stride = int(g.a_stride);
  // rows past the last: no access, zeros
  const auto rw = buffer_resource_2g(g.w + n0 * g.w_stride, unsigned(min(16, g.N - n0) - 1) * w_stride + g.K);
  const auto ra = buffer_resource_2g(g.a, unsigned(g.M - 1) * a_stride + g.K);
  const int w_at = n0 + r < g.N ? r * w_stride + k16 : kOutOfRange;
  const int a_at = r < g.M ? r * a_stride + k16 : kOutOfRange;
  i32x4_t acc = {0, 0, 0, 0};
  for (int k0 = wave * 128; k0 < g.K; k0 += W * 128 * UN) {
    u32x4_t w[UN][2], a[UN][2];
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + u * W * 128 + h * 64;
        const int out = k + k16 < g.K ? 0 : kOutOfRange;  // (an offset with this bit is past every range)
        w[u][h] = load_b128_stream(rw, (w_at + k) | out, 0);
        a[u][h] = load_b128(ra, (a_at + k) | out, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) acc = mfma_i8_16(w[u][h], a[u][h], acc);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
    i32x4_t total = sums[0][lane];
#pragma unroll
    for (int v = 1; v < W; ++v) total += sums[v][lane];
    const int m = r, n = n0 + (lane >> 4) * 4;
    if (m < g.M && n < g.N) store4(g, m, n, total);
  }
}

}  // namespace fx
