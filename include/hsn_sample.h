/*
 * hsn_sample.h -- the choice of a token from logits on MI355X (gfx950), from given random numbers.
 *
 * For each of n rows of V logits, with the row's settings temperature t, top_k, top_p, min_p and
 * its random number u in [0, 1):
 *   - NaN counts as -inf. Tokens are ordered by logit, descending; equal logits by token, ascending.
 *     A row without a logit above -inf gives -1; t <= 0 (or NaN) gives the order's first token.
 *   - x = (l - max l) / t (0 for l = max l) and e = exp(x), each rounded to fp32; the weight is the
 *     integer w = floor(2^40 e). Weights are whole numbers, so every order of adding them gives
 *     the same sums, and the same token on every run.
 *   - kept: the first top_k tokens of the order (top_k <= 0: all); of these the shortest prefix
 *     whose mass is at least top_p of their mass (top_p >= 1: all); of these the ones with e >=
 *     min_p (min_p <= 0: all). The order's first token is always kept.
 *   - the result is the first kept token, in the order of tokens, at which the running sum of
 *     weights exceeds floor(u W), W the kept weights' sum.
 * logits [n, V] in `dtype` (HSN_DTYPE_F32, _F16 or _BF16), rows `row` elements apart. u, temperature,
 * top_k, top_p and min_p are arrays of n on the device; each of the four settings may be NULL, and
 * then `settings` holds it for every row. tokens [n] is int64. 1 <= V <= 2^18, n < 2^22.
 *
 * Nothing is allocated and nothing is kept between calls, so the call may be captured in a graph.
 * `stream` is a hipStream_t (NULL: the default stream). The call returns once the work is
 * enqueued, with the status codes of hsn_ops.h and the message in hsn_win_last_error().
 */
#ifndef HSN_SAMPLE_H
#define HSN_SAMPLE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSN_SAMPLE_MAX_TOKENS 262144

typedef struct hsn_sample_settings {
    float temperature;
    int32_t top_k;
    float top_p;
    float min_p;
} hsn_sample_settings;

/* Bytes of device workspace hsn_sample needs, 16-byte aligned; 0 where it needs none. Its contents do
 * not matter before the call. */
int hsn_sample_workspace(int n, int V, int dtype, int64_t* bytes);

int hsn_sample(const void* logits, int64_t row, int dtype, const float* u,
               const float* temperature, const int32_t* top_k, const float* top_p,
               const float* min_p, const hsn_sample_settings* settings, int64_t* tokens, int n,
               int V, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSN_SAMPLE_H */
