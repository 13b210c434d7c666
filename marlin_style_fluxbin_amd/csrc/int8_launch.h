// Launch plumbing of the 8-bit rows (int8_rows.hip) and their products (int8_gemm*.hip).
#pragma once
#include "common.h"

namespace fx {

// What a row's values are before they are quantized.
enum : int { kRowsPlain = 0, kRowsNorm = 1, kRowsSwiglu = 2 };

struct Int8RowsArgs {
  const uint16_t* x;       // plain, norm: the rows; SwiGLU: the gate
  const uint16_t* second;  // norm: the residual, or null; SwiGLU: up
  const uint16_t* weight;  // norm: [columns]
  uint16_t* sum;           // norm with a residual: round(x + residual)
  int8_t* codes;
  float* scales;
  long long x_stride, second_stride, sum_stride, code_stride;  // elements between rows
  int rows, columns;
  int code_columns;  // columns .. code_columns of the codes become 0
  float eps;
};
bool launch_int8_rows(int dt, int mode, const Int8RowsArgs& a, hipStream_t s);

struct Int8RestoreArgs {
  const int8_t* codes;
  const float* scales;
  void* out;
  long long code_stride, out_stride;
  int rows, columns;
};
bool launch_int8_restore(int dt, const Int8RestoreArgs& a, hipStream_t s);

// out[m, n] = (sum_k a[m, k] w[n, k]) a_scales[m] w_scales[n] + bias[n]
struct Int8GemmArgs {
  const int8_t* a;
  const int8_t* w;
  const float* a_scales;
  const float* w_scales;
  const void* bias;  // [N] of out's type, or null
  void* out;
  int* partial;      // split K: [splits, M, N] sums, else null
  long long a_stride, w_stride, out_stride;
  int M, N, K;
  int dt;            // of out and bias
  int k_per_split;   // a multiple of the kernel's K step
  int any;           // few rows: a's and w's at any address, K any; else whole 16 bytes at 16-byte boundaries
};
constexpr long long kInt8RowLimit = 1LL << 22;  // bytes between rows: 256 rows stay within 31 bits
constexpr int kInt8MaxK = 131071;               // 2^14 * 131071 < 2^31: the sums are exact

struct Int8GemmPlan {
  int tile;    // which kernel
  int splits;  // workgroups along K
  int k_per_split;
};
// any: rows that do not lie at 16-byte boundaries or are not whole 16 bytes.  Few of them are read in
// place, more are copied first (launch_int8_align) and K is then whole 16.
constexpr int kInt8Few = -1;  // int8_gemm_few.h
Int8GemmPlan plan_int8_gemm(int M, int N, int K, bool any);

struct Int8AlignArgs {
  const int8_t* from[2];  // the activations, the weight
  int8_t* to[2];          // rows of `width` bytes
  long long stride[2];
  int rows[2];            // 0: none
  int columns, width;
};
void launch_int8_align(const Int8AlignArgs& a, hipStream_t s);
// Whether a Linear's rows are quantized in the product's own launch, and that launch.
bool int8_linear_fuses(int M, int N, int K);
void launch_int8_linear_few(int x_dt, const Int8RowsArgs& rows, const Int8GemmArgs& g, hipStream_t s);
bool launch_int8_gemm(const Int8GemmPlan& plan, const Int8GemmArgs& a, hipStream_t s);

}  // namespace fx
