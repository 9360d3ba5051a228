/*
 * rxmet_experts.h — C ABI of the expert layers' operators: routing of tokens to experts with its
 * gradient, the entries' order by expert, the int8 product with a weight for each expert, and the
 * weighted sum of a token's rows with its gradient.  No counterpart in the reference: they carry
 * the int8 product of rxmet_decoder.h into feed-forwards of experts.
 *
 * Every entry point takes device pointers and a hipStream_t (as void*), queues its kernels there
 * and returns 0 or a negative status (rxmet_last_error() has the message).  Nothing allocates
 * device memory.  Element types are RXMET_QDQ_F32 / F16 / BF16 of rxmet_qdq.h, activations
 * RXMET_ACT_* of rxmet_decoder.h.  Strides count elements; the last axis of every tensor is dense.
 *
 * An entry is one of the top_k experts of a token: entry t * top_k + j is token t's j-th.  Places
 * count the entries in the experts' order.
 */
#ifndef RXMET_EXPERTS_H_
#define RXMET_EXPERTS_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Most experts, experts of a token and groups of experts. */
#define RXMET_EXPERTS_MAX 1024
#define RXMET_TOP_K_MAX 64
#define RXMET_EXPERT_GROUPS_MAX 64

/* Scores s of a token's logits l. */
enum {
  RXMET_SCORE_SOFTMAX = 0, /* exp(l_e) / sum over all experts */
  RXMET_SCORE_SIGMOID = 1, /* 1 / (1 + exp(-l_e)) */
};

/*
 * How a token's experts are chosen.  With a bias the experts are ordered by c_e = fl32(s_e) + bias_e
 * (the score, computed in 64 bits to a few 2^-53 and rounded to fp32; one fp32 addition), without one by
 * their logits; NaN counts as -infinity and ties go to the lowest index.  The `experts` fall into `groups`
 * runs of equal length: a group's value is the sum (fp32) of its `group_best` (1 or 2) largest c (without a
 * bias: of fl32(s_e); of the logit alone where group_best is 1), and only the `top_groups` groups of the
 * largest values are chosen from.
 * Weights are the scores without the bias, over their sum (renormalize != 0), times `scale`.
 */
typedef struct rxmet_router {
  int32_t experts, top_k, score, renormalize;
  int32_t groups, top_groups, group_best;
  float scale;
} rxmet_router;

/*
 * experts, weights [tokens, top_k]: the chosen experts in their order (int32) and their weights
 * (fp32).  logits [tokens, experts] with a row stride; bias [experts] fp32 or NULL.  A softmax row
 * with a NaN or +infinity has NaN weights, a sigmoid one where a NaN is chosen; chosen experts whose
 * logits are all -infinity have the weights 0.  At most 2^24 tokens.
 */
int rxmet_route_forward(const rxmet_router *router, const void *logits, int64_t stride,
                        const float *bias, int32_t *experts, float *weights, int64_t tokens,
                        int32_t dtype, void *stream);

/*
 * d_logits [tokens, experts] (dense, in dtype) of d_weights [tokens, top_k]: the derivative of the
 * weights for fixed `experts`; the choice and the bias have none.  Experts that weigh nothing get 0.
 */
int rxmet_route_backward(const rxmet_router *router, const void *logits, int64_t stride,
                         const int32_t *experts, const float *d_weights, void *d_logits,
                         int64_t tokens, int32_t dtype, void *stream);

/*
 * Order of `count` entries (at most 2^26) by expert, entries of the same expert in their order.  experts [count]
 * int32; ids outside 0..num_experts-1 belong to no expert.
 *   offsets  [num_experts + 1] out: expert e's places are offsets[e]..offsets[e + 1]
 *   entries  [count] out: the entry of each place; behind offsets[num_experts] stand those of no expert
 *   places   [count] out: the place of each entry, -1 for those of no expert
 * The workspace (aligned to 4 bytes) may be NULL where its size is 0.
 */
int64_t rxmet_group_experts_workspace_bytes(int64_t count, int32_t num_experts);
int rxmet_group_experts(const int32_t *experts, int64_t count, int32_t num_experts,
                        int32_t *offsets, int32_t *entries, int32_t *places, void *workspace,
                        void *stream);

/*
 * What rxmet_group_experts gave for tokens * top_k entries.  Places may have been set to -1 since: entries without
 * one add nothing in rxmet_experts_combine (rxmet_experts_linear_int8 goes by offsets and entries).
 */
typedef struct rxmet_expert_groups {
  const int32_t *offsets, *entries, *places;
  int64_t tokens;
  int32_t top_k, experts;
} rxmet_expert_groups;

/*
 * For each place i of expert e:
 *   y[i, n] = act(acc[n]) with acc[n] = sum_k codes[r, k] * weight[e, n, k] * scales[r]
 *             * weight_scales[e, n] + bias[e, n],
 *   gated: y[i, n] = act(acc[n]) * acc[N + n].
 * r = i where `grouped` is set (codes [tokens * top_k, K]), else entries[i] / top_k (codes [tokens,
 * K]).  weight [experts, N or 2 N, K] int8 with strides of the first two axes in bytes;
 * weight_scales and bias [experts, N or 2 N] dense, bias in dtype or NULL; y [tokens * top_k, N] dense.
 * The sum is exact (int32), the rest fp32, rounded once to dtype.  Rows behind offsets[experts]
 * are not written.  Offsets and entries out of their range lead to no access out of bounds.
 * At most 2^24 tokens, fewer than 2^26 rows (tokens * top_k), N up to 2^24, K up to 131071; and the grid has to hold
 * what the rows may need: ceil(N / 128) (gated: / 64) * (rows / 64 + experts) and ceil(N / 32) (gated: / 16) * experts
 * are below 2^22.
 */
int rxmet_experts_linear_int8(const rxmet_expert_groups *groups, int32_t grouped,
                              const int8_t *codes, int64_t codes_stride, const float *scales,
                              const int8_t *weight, int64_t weight_stride, int64_t expert_stride,
                              const float *weight_scales, const void *bias, void *y, int64_t N,
                              int64_t K, int32_t gated, int32_t activation, int32_t dtype,
                              void *stream);

/*
 * out[t] = sum_j weights[t, j] * y[places[t, j]] + residual[t], in fp32 in the order of j, rounded
 * once.  Entries without a place add nothing.  y [tokens * top_k, N] and residual [tokens, N] (or NULL)
 * in dtype with row strides; weights [tokens, top_k] fp32; out [tokens, N] dense.  At most 2^23 tokens, N up to
 * 2^24, in the gradient too.
 */
int rxmet_experts_combine(const rxmet_expert_groups *groups, const void *y, int64_t y_stride,
                          const float *weights, const void *residual, int64_t residual_stride,
                          void *out, int64_t N, int32_t dtype, void *stream);

/*
 * Its gradient for d_out [tokens, N]: d_y[places[t, j]] = weights[t, j] * d_out[t], 0 in the rows that no entry
 * has as its place, and d_weights[t, j] = sum_n d_out[t, n] * y[places[t, j], n] in a fixed order, 0 without a
 * place.  No two entries may have the same place.  d_y (dense) or d_weights may be NULL; d_y needs the groups'
 * entries, d_weights needs y.  The residual's gradient is d_out.
 */
int rxmet_experts_combine_backward(const rxmet_expert_groups *groups, const void *d_out,
                                   int64_t d_out_stride, const void *y, int64_t y_stride,
                                   const float *weights, void *d_y, float *d_weights, int64_t N,
                                   int32_t dtype, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RXMET_EXPERTS_H_ */
