/*
 * Products in 8-bit integers with a scale for each row of both factors, and the rows that feed
 * them (included by fluxbin_amd.h; the same library, error and stream conventions).
 *
 * A row p of values is held as codes and a scale: with a = max|p|,
 *   code = round(127 p / a), ties to even, in [-127, 127];  scale = fp32(a / 127),
 * standing for code * scale.  A row of zeros has scale 0.  A row that holds an infinity or a
 * NaN, or whose scale no finite float is, stands for NaN (codes 0, scale NaN).
 *
 * Codes are int8 rows of contiguous columns; strides count elements between rows, all
 * non-negative.  dtype: FX_F16 or FX_BF16 for the rows' inputs, also FX_F32 for the outputs of
 * fx_int8_restore and fx_int8_gemm.  rows up to 2^21 (0 launches nothing), columns up to 2^20 (codes of
 * more than 16384 columns are formed in 64 bits, at two to six times the time per value).
 * Outputs overlap no input but where it says so.
 */
#ifndef FLUXBIN_INT8_H
#define FLUXBIN_INT8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows x [rows, columns] to codes [rows, code_columns] and scales [rows].  code_columns >=
 * columns: the codes behind a row's last column become 0 (rows padded to what fx_int8_gemm
 * takes).  Rows begin at any element.  Codes of inputs as they are (quantize, rmsnorm) are the
 * exact quotient's.
 */
int fx_int8_quantize(const void *x, long long x_stride, int8_t *codes, long long code_stride, float *scales, int rows,
                     int columns, int code_columns, int dtype, void *stream);
/*
 * p = weight s / sqrt(mean(s^2) + eps), with no rounding to 16 bits in front of the codes;
 * s = x, or with a residual (not NULL) s = round(x + residual), written to residual_out, which
 * may be x or residual itself (the same address and stride).
 */
int fx_int8_rmsnorm(const void *x, long long x_stride, const void *residual, long long residual_stride,
                    void *residual_out, long long residual_out_stride, const void *weight, int8_t *codes,
                    long long code_stride, float *scales, int rows, int columns, int code_columns, float eps, int dtype,
                    void *stream);
/* p = gate / (1 + exp(-gate)) up, in fp32. */
int fx_int8_silu_mul(const void *gate, long long gate_stride, const void *up, long long up_stride, int8_t *codes,
                     long long code_stride, float *scales, int rows, int columns, int code_columns, int dtype,
                     void *stream);
/* out [rows, columns] = code * scale, in fp32, rounded to dtype. */
int fx_int8_restore(const int8_t *codes, long long code_stride, const float *scales, void *out, long long out_stride,
                    int rows, int columns, int dtype, void *stream);

/*
 * out[m, n] = (sum_k a[m, k] w[n, k]) a_scales[m] w_scales[n] + bias[n]: the sum exact, then
 * fp32, rounded once to dtype (out's and bias's; bias may be NULL).  a [M, K], w [N, K] and
 * out [M, N]; K up to 131056, M up to 2^21, N up to 2^20; strides of a and w 0 or at least K.  out
 * overlaps no input.  Rows of whole 16 bytes (K a multiple of 16) at 16-byte boundaries, at most
 * 2^22 bytes apart, are read where they are, and so are those of a product of up to 32 rows (without
 * K splits, so slower where K is long and N short); others are copied into the workspace in every call.
 * `workspace` (16-byte aligned, no initial contents, NULL when 0 bytes) also holds the partial sums
 * of a product that is split along K; calls that share one must be ordered on one stream.  `loose`: 1
 * when a's rows do not lie so, plus 2 when w's do not (3 by itself where K is no multiple of 16).
 */
size_t fx_int8_gemm_workspace_bytes(int M, int N, int K, int loose);
int fx_int8_gemm(const int8_t *a, long long a_stride, const float *a_scales, const int8_t *w, long long w_stride,
                 const float *w_scales, const void *bias, void *out, long long out_stride, void *workspace,
                 size_t workspace_bytes, int M, int N, int K, int dtype, void *stream);

/*
 * A Linear in one call: rows x [M, K] of x_dtype (fp16 or bf16) quantized (fx_int8_quantize) and
 * multiplied (fx_int8_gemm) with w [N, K padded to whole 16, zeros behind K] to out of out_dtype.
 * `workspace`: fx_int8_linear_workspace_bytes bytes (NULL when 0: few rows that the product's launch
 * quantizes), 16-byte aligned, no initial contents; it holds the codes, their scales and the
 * product's partial sums; calls that share one must be ordered on one stream.
 */
size_t fx_int8_linear_workspace_bytes(int M, int N, int K);
int fx_int8_linear(const void *x, long long x_stride, int x_dtype, const int8_t *w, long long w_stride,
                   const float *w_scales, const void *bias, void *out, long long out_stride, void *workspace,
                   size_t workspace_bytes, int M, int N, int K, int out_dtype, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* FLUXBIN_INT8_H */
