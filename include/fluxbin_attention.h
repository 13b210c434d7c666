/*
 * Cached attention with a sliding window and sinks, and the 4-bit key/value cache
 * (included by fluxbin_amd.h; the same library, error and stream conventions).
 *
 * One call serves `batch` sequences of up to `tokens` queries each.  Sequence b holds
 * n = lengths[b] keys (clamped to [0, max_len]; lengths NULL: max_len), the last
 * m = query_lengths[b] of which (clamped to [0, tokens]; NULL: tokens) belong to its
 * queries: query t < m sits at position p = n - m + t and sees the keys j <= p with
 * j > p - window or j < sinks (window 0: every key j <= p).  Query head h reads KV head
 * h / (n_q_heads / n_kv_heads):
 *   out = sum_j softmax_j(scale q . k_j) v_j
 * with fp32 scores, softmax and accumulation, p rounded to 16 bits as the matrix cores take
 * it (fp16: weights below 2^-32 of a row's largest count as zero), out rounded once.  A query
 * that sees no key (p < 0) gives zeros; rows t >= m of out are left as they are.  Keys that a
 * query does not see never reach its row, whatever they hold; an infinity or NaN that it sees
 * does.  lengths and query_lengths are int32 arrays in device memory, read by the kernels:
 * a captured call follows their contents on every replay.
 *
 * The launches are chosen from the sizes alone (never from the lengths); a call takes one or
 * two, the second joining key splits through `workspace`
 * (fx_cached_attention_workspace_bytes bytes, 16-byte aligned, no initial contents; NULL
 * when 0).  Calls that share a workspace must be ordered on one stream.
 */
#ifndef FLUXBIN_ATTENTION_H
#define FLUXBIN_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* kv4 0: for fx_window_attention, else for fx_kv4_attention. */
size_t fx_cached_attention_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int tokens, int max_len,
                                           int head_dim, int window, int sinks, int dtype, int kv4);
/*
 * q [batch, n_q_heads, tokens, head_dim], k and v [batch, n_kv_heads, max_len, head_dim],
 * out as q, all of `dtype` (fp16 or bf16), the last axis contiguous; strides[12]: the
 * (batch, head, token or position) element strides of q, k, v and out, non-negative
 * multiples of 8, those of positions at most 2^22.  All four 16-byte aligned.  head_dim 64,
 * 128 or 256; n_q_heads a multiple of n_kv_heads; window and sinks >= 0, scale positive
 * and finite.
 */
int fx_window_attention(const void *q, const void *k, const void *v, void *out, const long long *strides,
                        const int *lengths, const int *query_lengths, void *workspace, size_t workspace_bytes,
                        int batch, int n_q_heads, int n_kv_heads, int tokens, int max_len, int head_dim, int window,
                        int sinks, float scale, int dtype, void *stream);
/*
 * The same over a 4-bit cache (format below); strides[6]: q's and out's.
 */
int fx_kv4_attention(const void *q, const void *k_codes, const void *k_scales, const void *v_codes,
                     const void *v_scales, void *out, const long long *strides, const int *lengths,
                     const int *query_lengths, void *workspace, size_t workspace_bytes, int batch, int n_q_heads,
                     int n_kv_heads, int tokens, int max_len, int head_dim, int window, int sinks, float scale,
                     int dtype, void *stream);
/*
 * The 4-bit cache.  Per sequence, KV head and position, for each group of 64 columns (lo
 * and hi its extremes):
 *   minimum = fp16(lo), scale = fp16(fp32(hi - lo) * fp32(1 / 15)),
 *   code = clamp(round(fp32(fp32(x - minimum) * fp32(1 / scale))), 0, 15), ties to even
 *   (scale 0: code 0), standing for code * scale + minimum.
 * A group that holds an infinity, a NaN or a magnitude above 32768 stands for NaN (scale 0,
 * minimum NaN).
 * codes uint16 [batch, n_kv_heads, max_len, 16, head_dim / 64]: word [c, g] holds columns
 * 64 g + 4 c + k, k < 4, in bits 4 k .. 4 k + 3; scales fp16 [batch, n_kv_heads, max_len,
 * head_dim / 64, 2]: (scale, minimum).  All contiguous and 16-byte aligned.
 *
 * fx_kv4_append writes tokens t < counts[b] (clamped to [0, tokens]; counts NULL: tokens) of
 * k and v [batch, n_kv_heads, tokens, head_dim] to positions start[b] + t (start NULL:
 * start_all + t); positions outside [0, max_len) are dropped.  strides[6]: k's and v's.
 */
int fx_kv4_append(const void *k, const void *v, const long long *strides, const int *start, int start_all,
                  const int *counts, void *k_codes, void *k_scales, void *v_codes, void *v_scales, int batch,
                  int n_kv_heads, int tokens, int max_len, int head_dim, int dtype, void *stream);
/* The values that the first `rows` positions stand for, rounded once to `dtype`: k_out and
 * v_out [batch, n_kv_heads, rows, head_dim], contiguous, 16-byte aligned. */
int fx_kv4_restore(const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales, void *k_out,
                   void *v_out, int batch, int n_kv_heads, int max_len, int rows, int head_dim, int dtype,
                   void *stream);

#ifdef __cplusplus
}
#endif

#endif /* FLUXBIN_ATTENTION_H */
