// Products of 8-bit rows: what the kernels share.
#pragma once
#include "int8_launch.h"

namespace fx {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

// D[i, j] += sum_k A[i, k] B[j, k] over 64 bytes of k: lane l gives bytes 16 (l / 16) .. of row
// l % 16 of A and of B, and holds D[4 (l / 16) + r, l % 16].  A is the weight, so that a lane's
// four results are neighbours in a row of the output.
__device__ __forceinline__ i32x4_t mfma_i8_16(const u32x4_t& a, const u32x4_t& b, const i32x4_t& c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ float load_value(const void* p, long long i) {
  if constexpr (DT == kF32) return static_cast<const float*>(p)[i];
  else return to_f32<DT>(static_cast<const uint16_t*>(p)[i]);
}

typedef float f32x4v_t __attribute__((ext_vector_type(4)));

// What the results of columns n .. n + 3 take besides their sums (scales 0 past the last).
struct Columns4 {
  f32x4v_t scales, bias;
};
__device__ __forceinline__ float bias_value(const Int8GemmArgs& g, int n) {
  if (g.dt == kF32) return load_value<kF32>(g.bias, n);
  return g.dt == kBF16 ? load_value<kBF16>(g.bias, n) : load_value<kF16>(g.bias, n);
}
__device__ __forceinline__ Columns4 load_columns(const Int8GemmArgs& g, int n) {
  Columns4 c{__builtin_bit_cast(f32x4v_t, load_b128(buffer_resource(g.w_scales, size_t(g.N) * 4), n * 4, 0)),
             {0.f, 0.f, 0.f, 0.f}};
  if (g.bias)
#pragma unroll
    for (int r = 0; r < 4; ++r) c.bias[r] = bias_value(g, min(n + r, g.N - 1));
  return c;
}

// Columns n .. n + 3 (those below N) of row m: one rounding of (acc a_scale) w_scale + bias in fp32.
// (sa: the row's scale.)  acc's own float is rounded once beyond 2^24 (2^-24 of it).
template <int DT>
__device__ __forceinline__ void store4_as(const Int8GemmArgs& g, int m, int n, const i32x4_t& acc, float sa,
                                          const Columns4& c) {
  float y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = fmaf(float(acc[r]) * sa, c.scales[r], c.bias[r]);
  const long long at = m * g.out_stride + n;
  if constexpr (DT == kF32) {
    float* out = static_cast<float*>(g.out) + at;
    if (n + 4 <= g.N) __builtin_memcpy(out, y, 16);
    else
#pragma unroll
      for (int r = 0; r < 3; ++r)
        if (n + r < g.N) out[r] = y[r];
  } else {
    uint16_t* out = static_cast<uint16_t*>(g.out) + at;
    if (n + 4 <= g.N) {
      const unsigned v[2] = {round_pair_bits<DT>(y[0], y[1]), round_pair_bits<DT>(y[2], y[3])};
      __builtin_memcpy(out, v, 8);
    } else {
#pragma unroll
      for (int r = 0; r < 3; ++r)
        if (n + r < g.N) out[r] = from_f32<DT>(y[r]);
    }
  }
}
__device__ __forceinline__ void store4(const Int8GemmArgs& g, int m, int n, const i32x4_t& acc, float sa,
                                       const Columns4& c) {
  if (g.dt == kBF16) store4_as<kBF16>(g, m, n, acc, sa, c);
  else if (g.dt == kF16) store4_as<kF16>(g, m, n, acc, sa, c);
  else store4_as<kF32>(g, m, n, acc, sa, c);
}

}  // namespace fx
