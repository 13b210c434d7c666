// Products of few 8-bit rows (a decode step, a small batch): the weight is read once, straight into
// the matrix cores' operands.
#pragma once
#include "int8_gemm.h"
#include "int8_row.h"

namespace fx {

constexpr int kFewCodes = 16384;  // bytes of codes that a workgroup quantizes for itself

// 16 bytes at any address, and n <= 16 of them (the others 0).
__device__ __forceinline__ u32x4_t any_b128(const int8_t* p) {
  u32x4_t v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ u32x4_t part_b128(const int8_t* p, int n) {
  if (n >= 16) return any_b128(p);
  u32x4_t v = {0u, 0u, 0u, 0u};
  for (int e = 0; e < n; ++e) v[e >> 2] |= unsigned(uint8_t(p[e])) << (8 * (e & 3));
  return v;
}

// RT x 16 rows of the weight by MT x 16 of the activations a workgroup, its W waves dealing the
// columns in pieces of 128: a wave's sums are over its own columns and are added through LDS, so that
// one launch has a burst of the whole weight in flight.  Bound by the weight's bytes (24576 x 4096 at
// one row 19.7 us, 5.1 TB/s; 4096 x 4096 5.4 us, of which a launch is 2): every wave issues UN pieces'
// loads in front of its first product (left to the compiler's order, 20.4).
//
// ANY: rows of any length at any address (elsewhere they begin at 16-byte boundaries and are whole 16
// bytes long).  XDT kBF16 or kF16: the rows come unquantized, and every workgroup quantizes them for itself while
// its part of the weight is on the way: a launch less than codes that another kernel leaves.
template <int XDT, bool ANY, int MT, int RT, int W, int UN>
__global__ __launch_bounds__(W * 64) void int8_gemm_few_kernel(const Int8GemmArgs g, const Int8RowsArgs rows) {
  constexpr bool kQuantize = XDT >= 0;
  static_assert(!(kQuantize && ANY), "the rows that are quantized here are whole 16 bytes");
  constexpr int kTiles = MT * RT;
  static_assert(!kQuantize || MT == 1, "at most sixteen rows are quantized here");
  __shared__ i32x4_t sums[W][kTiles][64];
  __shared__ __attribute__((aligned(16))) int8_t codes[kQuantize ? kFewCodes : 16];
  __shared__ double red[W];
  __shared__ float row_scales[16];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int r = lane & 15, k16 = (lane >> 4) * 16;
  const int n0 = xcd_local_index8(blockIdx.x, gridDim.x) * (16 * RT);
  const int w_stride = ANY ? 0 : int(g.w_stride), a_stride = ANY ? 0 : int(g.a_stride);
  // rows past the last: no access, zeros
  const auto rw = buffer_resource_2g(g.w + n0 * g.w_stride, unsigned(min(16 * RT, g.N - n0) - 1) * w_stride + g.K);
  const auto ra = buffer_resource_2g(g.a, kQuantize ? 0u : unsigned(g.M - 1) * a_stride + g.K);
  int w_at[RT], a_at[MT];
#pragma unroll
  for (int t = 0; t < RT; ++t) w_at[t] = n0 + 16 * t + r < g.N ? (16 * t + r) * w_stride + k16 : kOutOfRange;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if (kQuantize) a_at[t] = min(r, g.M - 1) * g.K + k16;  // (a column past M is not stored)
    else a_at[t] = 16 * t + r < g.M ? (16 * t + r) * a_stride + k16 : kOutOfRange;
  }
  i32x4_t acc[RT][MT];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) acc[i / MT][i % MT] = i32x4_t{0, 0, 0, 0};
  u32x4_t w[UN][2][RT], a[UN][2][MT];
  // ANY: rows past the last are the last again, not stored
  const int8_t *w_row[RT], *a_row[MT];
  if constexpr (ANY) {
#pragma unroll
    for (int t = 0; t < RT; ++t) w_row[t] = g.w + min(n0 + 16 * t + r, g.N - 1) * g.w_stride + k16;
#pragma unroll
    for (int t = 0; t < MT; ++t) a_row[t] = g.a + min(16 * t + r, g.M - 1) * g.a_stride + k16;
  }
  // (an offset with kOutOfRange's bit is past every range)
  auto past = [&](int k) __attribute__((always_inline)) { return k + k16 < g.K ? 0 : kOutOfRange; };
  auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + u * W * 128 + h * 64;
        if constexpr (ANY) {
          const bool whole = k + 64 <= g.K;
#pragma unroll
          for (int t = 0; t < RT; ++t) w[u][h][t] = whole ? any_b128(w_row[t] + k) : part_b128(w_row[t] + k, g.K - k - k16);
#pragma unroll
          for (int t = 0; t < MT; ++t) a[u][h][t] = whole ? any_b128(a_row[t] + k) : part_b128(a_row[t] + k, g.K - k - k16);
          continue;
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) w[u][h][t] = load_b128_stream(rw, (w_at[t] + k) | past(k), 0);
        if constexpr (!kQuantize) {
#pragma unroll
          for (int t = 0; t < MT; ++t) a[u][h][t] = load_b128(ra, (a_at[t] + k) | past(k), 0);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  int k0 = wave * 128;
  load(k0);
  if constexpr (kQuantize) {
    RowPointers p{};
    for (int m = 0; m < g.M; ++m) {
      p.x = rows.x + m * rows.x_stride;
      p.codes = codes + m * g.K;
      quantize_row<XDT, kRowsPlain, W * 64, 2>(rows, p, row_scales + m, threadIdx.x, red);
    }
    __syncthreads();
  }
  while (true) {
    if constexpr (kQuantize) {
#pragma unroll
      for (int u = 0; u < UN; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = k0 + u * W * 128 + h * 64;
          a[u][h][0] = *reinterpret_cast<const u32x4_t*>(codes + (past(k) ? k16 : a_at[0] + k));
        }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[i][j] = mfma_i8_16(w[u][h][i], a[u][h][j], acc[i][j]);
    k0 += W * 128 * UN;
    if (k0 >= g.K) break;
    load(k0);
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i) sums[wave][i][lane] = acc[i / MT][i % MT];
  __syncthreads();
  for (int tile = wave; tile < kTiles; tile += W) {
    i32x4_t total = sums[0][tile][lane];
#pragma unroll
    for (int v = 1; v < W; ++v) total += sums[v][tile][lane];
    const int m = (tile % MT) * 16 + r, n = n0 + (tile / MT) * 16 + (lane >> 4) * 4;
    // (their scales loaded in front of the products: 4096 x 12288 12.3 us for 11.9)
    if (m < g.M && n < g.N) store4(g, m, n, total, kQuantize ? row_scales[m & 15] : g.a_scales[m], load_columns(g, n));
  }
}

}  // namespace fx
