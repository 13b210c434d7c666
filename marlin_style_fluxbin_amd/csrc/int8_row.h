// A row of values to 8-bit codes and a scale, by the threads of a wave or of a workgroup
// (int8_rows.hip; int8_gemm_few.h quantizes its own few rows).
#pragma once
#include "int8_launch.h"

namespace fx {

constexpr float kSmall = 0x1p-100f;  // 127 / a and the codes' products are normal floats from here on
constexpr float kRounder = 12582912.f;  // 1.5 * 2^23: adding it rounds to a whole number, ties to even

template <int TPR, class T, class F>
__device__ __forceinline__ T row_reduce(T v, F f, T* red) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v = f(v, __shfl_xor(v, offset, 64));
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = f(v, red[i]);
  }
  return v;
}

// Eight 16-bit values from p, n of them there (the others 0).  Rows begin at any element: the loads
// and stores of whole chunks are 16 and 8 bytes at whatever address (1001 rows of 2077 columns 7.1 us,
// element by element 11.6).
__device__ __forceinline__ u32x4_t load8(const uint16_t* p, int n) {
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (n >= 8) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) v[e >> 1] |= unsigned(p[e]) << (16 * (e & 1));
  }
  return v;
}
__device__ __forceinline__ void store8(uint16_t* p, const u32x4_t& v, int n) {
  if (n >= 8) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = uint16_t(v[e >> 1] >> (16 * (e & 1)));
  }
}
// Eight codes, each in the low byte of c, n of them there.
__device__ __forceinline__ void store_codes(int8_t* p, const unsigned (&c)[8], int n) {
  if (n >= 8) {
    unsigned v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned lo = __builtin_amdgcn_perm(c[4 * h + 1], c[4 * h], 0x0c0c0400u);
      const unsigned hi = __builtin_amdgcn_perm(c[4 * h + 3], c[4 * h + 2], 0x0c0c0400u);
      v[h] = lo | hi << 16;
    }
    __builtin_memcpy(p, v, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = int8_t(c[e]);
  }
}
template <int DT>
__device__ __forceinline__ float at8(const u32x4_t& v, int e) {
  return to_f32<DT>(uint16_t(v[e >> 1] >> (16 * (e & 1))));
}
template <int DT>
__device__ __forceinline__ u32x4_t add8(const u32x4_t& x, const u32x4_t& r) {
  u32x4_t s;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float lo = to_f32<DT>(uint16_t(x[w])) + to_f32<DT>(uint16_t(r[w]));
    float hi = to_f32<DT>(uint16_t(x[w] >> 16)) + to_f32<DT>(uint16_t(r[w] >> 16));
    s[w] = round_pair_bits<DT>(lo, hi);
  }
  return s;
}

constexpr float kSwigluSmall = 0x1p-60f;

// silu(x) y within 2^-21 of it, or an infinity where the floats do not give it: the row is then formed
// in 64 bits.  exp(-x) = 2^(n + f) with n whole and f from a product in two parts; one Newton step on
// the reciprocal (4096 rows of 12288 columns 48 us, with expf and a division 110).  Below -87 the value
// is under 2^-119 |y| and counts as zero in a row whose largest is 2^-60 and more.
__device__ __forceinline__ float swiglu(float x, float y) {
  constexpr float kHigh = -0x1.715476p+0f, kLow = -0x1.4ae0cp-26f;  // -log2(e) in two parts
  const float n = rintf(x * kHigh);
  const float f = fmaf(x, kLow, fmaf(x, kHigh, -n));
  const float d = 1.f + ldexpf(__builtin_amdgcn_exp2f(f), int(n));
  float r = __builtin_amdgcn_rcpf(d);
  r = fmaf(fmaf(-d, r, 1.f), r, r);
  float v = x * r * y;
  if (x < -87.f) v = fabsf(y) <= 0x1p30f && x > -INFINITY ? 0.f : INFINITY;
  return v;
}

// A row's addresses; codes may lie in LDS.
struct RowPointers {
  const uint16_t *x, *second;
  uint16_t* sum;
  int8_t* codes;
};

// A row in 64 bits, read anew: rows of any length, and those whose values leave the range that the
// floats of the fast way hold (a row of zeros, magnitudes below 2^-100, sums of squares or products
// beyond 2^128, infinities, NaN).
template <int DT, int MODE, int TPR>
__device__ void row_in_64_bits(const Int8RowsArgs& a, const RowPointers& p, float* scale_out, int tl,
                               bool added, double* red) {
  const auto value = [&](int c, int e, const u32x4_t& xv, const u32x4_t& yv) __attribute__((always_inline)) {
    const double x = at8<DT>(xv, e);
    if constexpr (MODE == kRowsNorm) return x * double(at8<DT>(yv, e));
    else if constexpr (MODE == kRowsSwiglu) return x / (1. + exp(-x)) * double(at8<DT>(yv, e));
    else return x;
  };
  const auto load = [&](int c, u32x4_t& xv, u32x4_t& yv) __attribute__((always_inline)) {
    const int n = a.columns - 8 * c;
    yv = u32x4_t{0u, 0u, 0u, 0u};
    if (MODE == kRowsNorm && p.second) xv = load8(p.sum + 8 * c, n);
    else xv = load8(p.x + 8 * c, n);
    if constexpr (MODE == kRowsNorm) yv = load8(a.weight + 8 * c, n);
    if constexpr (MODE == kRowsSwiglu) yv = load8(p.second + 8 * c, n);
  };
  const int chunks = (a.columns + 7) / 8;
  double top = 0., squares = 0.;
  for (int c = tl; c < chunks; c += TPR) {
    if (MODE == kRowsNorm && p.second && !added) {  // each thread reads what it wrote itself
      const int n = a.columns - 8 * c;
      store8(p.sum + 8 * c, add8<DT>(load8(p.x + 8 * c, n), load8(p.second + 8 * c, n)), n);
    }
    u32x4_t xv, yv;
    load(c, xv, yv);
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const double v = fabs(value(c, e, xv, yv)), x = at8<DT>(xv, e);
      top = v >= top || v != v ? v : top;  // a NaN stays: no later value is >= it, and v == v
      if constexpr (MODE == kRowsNorm) squares += x * x;
    }
  }
  const auto larger = [](double u, double v) { return u != u || u >= v ? u : v; };  // a NaN is the largest
  const auto plus = [](double u, double v) { return u + v; };
  top = row_reduce<TPR>(top, larger, red);
  double inverse = 1.;
  if constexpr (MODE == kRowsNorm) {
    squares = row_reduce<TPR>(squares, plus, red);
    inverse = top > 0. ? 1. / sqrt(squares / a.columns + double(a.eps)) : 0.;
  }
  float scale = float(top * inverse / 127.);
  const bool held = scale < INFINITY;  // a row that no float scale stands for is NaN
  if (!held) scale = __uint_as_float(0x7fc00000u);
  if (tl == 0) *scale_out = scale;
  for (int c = tl; 8 * c < a.code_columns; c += TPR) {
    u32x4_t xv = {0u, 0u, 0u, 0u}, yv = xv;
    if (c < chunks) load(c, xv, yv);
    unsigned code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      code[e] = held && top > 0. ? unsigned(int(rint(value(c, e, xv, yv) * 127. / top))) : 0u;
    store_codes(p.codes + 8 * c, code, a.code_columns - 8 * c);
  }
}

// One row by TPR threads (thread tl of them), CH chunks of 8 columns a thread in registers (0: rows of
// any length).  `red`: a double for each of the workgroup's waves, in LDS.
template <int DT, int MODE, int TPR, int CH>
__device__ __forceinline__ void quantize_row(const Int8RowsArgs& a, const RowPointers& p, float* scale_out, int tl,
                                             double* red) {
  if constexpr (CH == 0) {
    row_in_64_bits<DT, MODE, TPR>(a, p, scale_out, tl, false, red);
  } else {
    u32x4_t xv[CH], yv[CH], wv[CH];
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int c = tl + q * TPR, n = a.columns - 8 * c;
      xv[q] = load8(p.x + 8 * c, n);
      if (MODE != kRowsPlain && p.second) yv[q] = load8(p.second + 8 * c, n);
      if constexpr (MODE == kRowsNorm) wv[q] = load8(a.weight + 8 * c, n);
    }
    float v[CH][8], squares = 0.f;
    unsigned top_bits = 0u;
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      if (MODE == kRowsNorm && p.second) {
        const int c = tl + q * TPR;
        xv[q] = add8<DT>(xv[q], yv[q]);
        store8(p.sum + 8 * c, xv[q], a.columns - 8 * c);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = at8<DT>(xv[q], e);
        if constexpr (MODE == kRowsNorm) {
          squares = fmaf(x, x, squares);
          v[q][e] = x * at8<DT>(wv[q], e);  // exact: 22 bits at most
        } else if constexpr (MODE == kRowsSwiglu) {
          v[q][e] = swiglu(x, at8<DT>(yv[q], e));
        } else {
          v[q][e] = x;
        }
        top_bits = max(top_bits, __float_as_uint(v[q][e]) & 0x7fffffffu);
      }
    }
    // (as bits, so that an infinity or NaN is the largest)
    top_bits = row_reduce<TPR>(top_bits, [](unsigned u, unsigned w) { return max(u, w); }, reinterpret_cast<unsigned*>(red));
    const float top = __uint_as_float(top_bits);
    float inverse = 1.f;
    bool plain = top_bits < 0x7f800000u && top >= (MODE == kRowsSwiglu ? kSwigluSmall : kSmall);
    if constexpr (MODE == kRowsNorm) {
      squares = row_reduce<TPR>(squares, [](float u, float w) { return u + w; }, reinterpret_cast<float*>(red));
      plain = plain && squares < INFINITY && squares >= kSmall;
      inverse = rsqrtf(squares / float(a.columns) + a.eps);
    }
    // Zeros (a padded batch's rows), and infinities and NaN where no product can overflow, need no second look.
    constexpr bool kBounded = MODE == kRowsPlain || (MODE == kRowsNorm && DT == kF16);
    if (top_bits == 0u || (kBounded && top_bits >= 0x7f800000u)) {
      unsigned any = 0u;
      if (top_bits == 0u) {
        const uint16_t* from = MODE == kRowsNorm && p.second ? p.sum : p.x;
        for (int c = tl; 8 * c < a.columns; c += TPR) {
          const u32x4_t x = load8(from + 8 * c, a.columns - 8 * c);
          any |= (x[0] | x[1] | x[2] | x[3]) & 0x7fff7fffu;
        }
        any = row_reduce<TPR>(any, [](unsigned u, unsigned w) { return u | w; }, reinterpret_cast<unsigned*>(red));
      }
      if (any == 0u) {
        if (tl == 0) *scale_out = top_bits == 0u ? 0.f : __uint_as_float(0x7fc00000u);
        const unsigned none[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        for (int c = tl; 8 * c < a.code_columns; c += TPR) store_codes(p.codes + 8 * c, none, a.code_columns - 8 * c);
        return;
      }
    }
    const float scale = top * inverse / 127.f;
    if (!plain || !(scale < INFINITY)) {
      row_in_64_bits<DT, MODE, TPR>(a, p, scale_out, tl, true, red);
      return;
    }
    if (tl == 0) *scale_out = scale;
    const float r = 127.f / top;
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int c = tl + q * TPR, n = a.code_columns - 8 * c;
      unsigned code[8];
      bool near = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float t = v[q][e] * r, whole = t + kRounder;
        code[e] = __float_as_uint(whole);
        // within the rounding of t (2^-15) of a border between two codes
        near = near || fabsf(t - (whole - kRounder)) > 0.4999f;
      }
      // The products w s and x are exact, so their codes can be: the quotient again in 64 bits,
      // where one of 22-bit numbers that is no border differs from every border.
      if (MODE != kRowsSwiglu && near) {
#pragma unroll
        for (int e = 0; e < 8; ++e) code[e] = unsigned(int(rint(double(v[q][e]) * 127. / double(top))));
      }
      if (n > 0) store_codes(p.codes + 8 * c, code, n);
    }
  }
}

}  // namespace fx
