/*
 * rxmet_decoder.h — C ABI of the 8-bit decoder operators: root-mean-square norm with residual
 * and int8 output, int8 matrix product with an epilogue, a paged cache of int8 keys and values,
 * and the attention over it.  No counterpart in the reference: they carry its symmetric int8
 * grids into the layers of a language model.
 *
 * Every entry point takes device pointers and a hipStream_t (as void*), queues its kernels there
 * and returns 0 or a negative status (rxmet_last_error() has the message).  Nothing allocates
 * device memory.  Element types are RXMET_QDQ_F32 / F16 / BF16 of rxmet_qdq.h.  Strides count
 * elements; the last axis of every tensor is dense.
 *
 * A grid is symmetric: value = code * scale, codes -127..127, rounding half to even.  Scales are
 * made from max(largest magnitude, 2^-112); a group with a NaN or an infinity has scale NaN and
 * codes 0, so that all of its values are NaN.
 */
#ifndef RXMET_DECODER_H_
#define RXMET_DECODER_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Widest row of the row operators. */
#define RXMET_ROW_MAX 65536
/* Longest contraction of rxmet_linear_int8 (the int32 sum of 2^14 * K stays in range). */
#define RXMET_LINEAR_INT8_K_MAX 131071

/*
 * Rows to int8.  With a weight: h = round_dtype(x + residual) (h = x without a residual),
 * rstd = 1 / sqrt(mean(h^2) + eps), u = h * weight (fp32; a product beyond it is an infinity),
 * a = max(max|u|, 2^-112),
 * codes = rint(u * (127 / a)), scales = a / 127 * rstd.  The codes do not go by rstd, so they do not go by the
 * order of the mean's sum.  Without a weight (NULL): u = x, rstd = 1.
 *   x, residual   [rows, cols], row strides x_stride / residual_stride
 *   weight        [cols], of `dtype` or (weight_f32 != 0) fp32
 *   h             [rows, cols] out, needed with a residual, else NULL
 *   codes         [rows, cols] int8 out, or NULL
 *   y             [rows, cols] out: codes * scale in dtype (the training form), or NULL
 *   scales, rstd  [rows] fp32 out; rstd may be NULL
 */
int rxmet_rms_quantize_forward(const void *x, int64_t x_stride, const void *residual,
                               int64_t residual_stride, const void *weight, int32_t weight_f32,
                               void *h, int8_t *codes, void *y, float *scales, float *rstd,
                               int64_t rows, int64_t cols, int32_t dtype, float eps, void *stream);

/*
 * Gradient of the training form, straight through the rounding: with n = h * rstd and
 * dn = dy * weight, dx = rstd * (dn - n * mean(dn * n)) + dh; d_weight = sum over rows of dy * n,
 * in a fixed order.  dx is the gradient of x and of the residual.  dh (the gradient that reaches
 * h by itself) and d_weight may be NULL.  d_weight has the weight's type.
 */
int64_t rxmet_rms_quantize_backward_workspace_bytes(int64_t rows, int64_t cols);
int rxmet_rms_quantize_backward(const void *dy, int64_t dy_stride, const void *dh,
                                int64_t dh_stride, const void *h, int64_t h_stride,
                                const void *weight, int32_t weight_f32, const float *rstd,
                                void *dx, void *d_weight, int64_t rows, int64_t cols,
                                int32_t dtype, void *workspace, void *stream);

/* Activations of rxmet_linear_int8 (gelu: with the error function). */
enum {
  RXMET_ACT_NONE = 0,
  RXMET_ACT_RELU = 1,
  RXMET_ACT_SILU = 2,
  RXMET_ACT_GELU = 3,
};

/*
 * y[m, n] = act(sum_k codes[m, k] * weight[n, k] * scales[m] * weight_scales[n] + bias[n])
 *           + residual[m, n]
 * The sum is exact (int32); the rest is fp32, rounded once to dtype.  codes [M, K] and weight
 * [N, K] int8 with row strides in bytes; bias [N] and residual [M, N] in dtype, may be NULL;
 * y [M, N] dense.  The workspace (aligned to 16 bytes) may be NULL where its size is 0.  Rows that do not all
 * start on 16 bytes are copied into it for more than 16 rows of x; a weight laid out with such
 * a row stride once saves that.
 */
int64_t rxmet_linear_int8_workspace_bytes(const int8_t *codes, int64_t codes_stride,
                                          const int8_t *weight, int64_t weight_stride, int64_t M,
                                          int64_t N, int64_t K);
int rxmet_linear_int8(const int8_t *codes, int64_t codes_stride, const float *scales,
                      const int8_t *weight, int64_t weight_stride, const float *weight_scales,
                      const void *bias, const void *residual, int64_t residual_stride, void *y,
                      int64_t M, int64_t N, int64_t K, int32_t activation, int32_t dtype,
                      void *workspace, void *stream);

/*
 * A cache of int8 keys and values in pages of 16, 32, 64 or 128 tokens, with one scale for each
 * page and head.  Keys lie [pages, heads, page_size, dim], values [pages, heads, dim, page_size]
 * (the order in which the attention's second product reads them).  Sequence b's token t is in
 * page block_table[b, t / page_size] at t % page_size.  An id outside the cache, or a token past
 * the table's width, is never dereferenced: append leaves the token out, read and attention
 * give NaN for it.
 */
typedef struct rxmet_kv_cache {
  int8_t *k, *v;
  float *k_scale, *v_scale; /* [pages, heads], positive as append makes them */
  int64_t pages;
  int32_t heads, page_size, dim, reserved; /* dim: 64, 128, 192 or 256; reserved 0 */
} rxmet_kv_cache;

/* Where the sequences lie: block_table [seqs, table_cols] int32 with row stride table_stride. */
typedef struct rxmet_kv_table {
  const int32_t *ids;
  int64_t stride;
  int32_t seqs, cols;
} rxmet_kv_table;

/*
 * Puts new tokens behind `lengths[b]` tokens of each sequence: rows cu_new[b]..cu_new[b+1] of key
 * and value ([tokens, heads, dim], strides of the first two axes), or row b alone where cu_new is
 * NULL.  A page's scale becomes max(largest new magnitude / 127, its scale if it holds older
 * tokens of the sequence); where it grows, the older codes become rint(code * old / new).
 * max_new: the most new tokens of a sequence (a larger count is taken too, more slowly).
 */
int rxmet_kv_append(const rxmet_kv_cache *cache, const rxmet_kv_table *table,
                    const int32_t *lengths, const int32_t *cu_new, int64_t tokens,
                    int64_t max_new, const void *key, int64_t key_stride_t, int64_t key_stride_h,
                    const void *value, int64_t value_stride_t, int64_t value_stride_h,
                    int32_t dtype, void *stream);

/*
 * Values of the tokens first[b] + i, i < cu[b+1] - cu[b], to rows cu[b] + i of key and value
 * ([tokens, heads, dim] dense, in dtype).
 */
int rxmet_kv_read(const rxmet_kv_cache *cache, const rxmet_kv_table *table, const int32_t *first,
                  const int32_t *cu, int64_t tokens, int64_t max_tokens, void *key, void *value,
                  int32_t dtype, void *stream);

/*
 * out[i, g] = softmax(q . k * scale) v over the cached tokens that query i sees.  Rows
 * cu_query[b]..cu_query[b+1] of query ([queries, q_heads, dim], strides of the first two axes; row b alone
 * where cu_query is NULL) are the last ones of sequence b's lengths[b] tokens: query j of n stands
 * at p = lengths[b] - n + j and sees tokens t <= p (causal) or all (causal == 0), and
 * t > p - window where window > 0.  A query that sees nothing gives 0.  q_heads is a multiple of
 * the cache's heads; query head g reads head g / (q_heads / heads).
 * max_query, max_length: the most queries and tokens of a sequence; they size the launch (longer
 * ones are taken too).  dtype: F16 or BF16.
 */
int64_t rxmet_kv_attention_workspace_bytes(const rxmet_kv_cache *cache, int32_t seqs,
                                           int64_t queries, int32_t q_heads, int64_t max_query,
                                           int64_t max_length, int64_t window);
int rxmet_kv_attention(const rxmet_kv_cache *cache, const rxmet_kv_table *table,
                       const int32_t *lengths, const int32_t *cu_query, int64_t queries,
                       int64_t max_query, int64_t max_length, const void *query,
                       int64_t query_stride_t, int64_t query_stride_h, int32_t q_heads,
                       float scale, int32_t causal, int64_t window, void *out, int32_t dtype,
                       void *workspace, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RXMET_DECODER_H_ */
