/*
 * hsn_score.h -- log probabilities of given tokens on MI355X (gfx950), with the entropy and the most
 * probable alternatives, and the gradient. For each of n rows of V logits l and the row's token t:
 *   m = max l,  x_j = l_j - m,  S = sum_j e^x_j,  p_j = e^x_j / S,  log p_j = x_j - log S
 *   logprob = log p_t,  entropy = -sum_j p_j log p_j = log S - (sum_j e^x_j x_j) / S
 * - A token outside [0, V) is skipped: logprob 0 and no gradient from it; the entropy is the row's.
 * - A logit of -inf has no mass. A row of nothing else has logprob -inf, entropy 0 and no gradient.
 * - A row with a NaN or +inf has NaN for its values and its whole gradient.
 * - The alternatives are the `top` largest logits that are neither NaN nor -inf, the largest first and
 *   equal ones by token; where there are fewer, the token is -1 and its log probability -inf.
 * logits [n, V] in `dtype` (HSN_DTYPE_F32, _F16 or _BF16), rows `row` elements apart, any multiple of
 * the type's size as address. tokens[i * token_stride], int64 (token_bytes 8) or int32 (4).
 * Everything is computed in fp32, but for the sums over a thread's logits, which are float64 beyond 16
 * or 32 of them: a log probability is right to about 2^-22 of max(1, |x|, log S) and the entropy to
 * 2^-21 of max(1, log S), whatever the logits are. An exponential's argument is rounded, so a probability
 * is right to about 2^-21 + 2^-23 |x| of itself (and to 2^-126); a 16-bit gradient is rounded once. Sums
 * are taken in an order that depends on n, V, the type and the rows' addresses modulo 16 alone.
 * 1 <= V <= 2^24, n V < 2^40, n < 2^24, top <= 32.
 *
 * Nothing is allocated and nothing is kept between calls, so a call may be captured in a graph.
 * `stream` is a hipStream_t (NULL: the default stream). The call returns once the work is enqueued,
 * with the status codes of hsn_ops.h and the message in hsn_win_last_error().
 */
#ifndef HSN_SCORE_H
#define HSN_SCORE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSN_SCORE_MAX_TOP 32
#define HSN_SCORE_MAX_TOKENS (1 << 24)

/* Bytes of device workspace hsn_score_forward needs, 16-byte aligned; 0 where it needs none. Its
 * contents do not matter before the call. */
int hsn_score_workspace(int n, int V, int dtype, int top, int64_t* bytes);

/*
 * logprob, entropy [n] (fp32); top_tokens (int64), top_logprobs (fp32) [n, top], NULL where top is 0;
 * stats [n, 4] (fp32, 16-byte aligned; may be NULL): m, 1 / S (0 for a row without mass), log S and the
 * entropy, for the backward.
 */
int hsn_score_forward(const void* logits, int64_t row, int dtype, const void* tokens,
                      int64_t token_stride, int token_bytes, float* logprob, float* entropy,
                      int64_t* top_tokens, float* top_logprobs, float* stats, int n, int V, int top,
                      void* workspace, int64_t workspace_bytes, void* stream);

/*
 * d_logits [n, V] (dense, `dtype`) from the forward's inputs and stats, and the cotangents g =
 * d_logprob and h = d_entropy [n] (fp32, strides in elements; either may be NULL: zero):
 *   d_j = g ([j = t] - p_j) - h p_j (log p_j + entropy)
 * d_logits must not overlap the inputs.
 */
int hsn_score_backward(const void* logits, int64_t row, int dtype, const void* tokens,
                       int64_t token_stride, int token_bytes, const float* stats,
                       const float* d_logprob, int64_t g_stride, const float* d_entropy,
                       int64_t h_stride, void* d_logits, int n, int V, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSN_SCORE_H */
