/*
 * hsn_unit_router.h -- the choice of units in training on MI355X (gfx950): the k largest of each
 * token's M logits, their shares, the units' load with its balance loss, and the gradient. For each of n
 * tokens, where valid[i] (NULL: all) and some logit is above -inf (a live token):
 *   units = the k largest logits, the largest first, equal ones by unit; -inf is never chosen
 *   shares = softmax of the chosen logits (in fp32)
 *   p = softmax of all M logits
 * and over all tokens, with c_e the number of times unit e is chosen and R the live tokens:
 *   load_e = c_e / sum c,  prob_e = (sum over live tokens of p_e) / R,  balance = M sum_e load_e prob_e
 * (1 where the units are chosen alike; 0 without a live token). An empty slot has unit -1 and share 0; a
 * token that is not live has k of them, and no gradient.
 * - A NaN logit is chosen first. A token with a NaN or +inf has NaN shares and a NaN gradient, and makes
 *   the probs and the balance NaN; the other tokens' gradients are not touched by it.
 * logits [n, M] in `dtype` (HSN_DTYPE_F32, _F16 or _BF16), rows `row` elements apart; valid is uint8.
 * Everything is computed in fp32; the sums over tokens are fp32 over at most a few hundred tokens and
 * float64 above, in an order that depends on n, M and the type alone.
 * 1 <= M <= 256, 1 <= k <= min(M, 16), n < 2^30.
 *
 * Nothing is allocated and nothing is kept between calls, so a call may be captured in a graph.
 * `stream` is a hipStream_t (NULL: the default stream). The call returns once the work is enqueued,
 * with the status codes of hsn_ops.h and the message in hsn_win_last_error().
 */
#ifndef HSN_UNIT_ROUTER_H
#define HSN_UNIT_ROUTER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSN_ROUTER_MAX_UNITS 256
#define HSN_ROUTER_MAX_CHOSEN 16

/* Bytes of device workspace hsn_unit_router_forward needs, 16-byte aligned. Its contents do not matter
 * before the call. */
int hsn_unit_router_workspace(int n, int M, int dtype, int64_t* bytes);

/*
 * units (int64), shares (fp32) [n, k]; tally [M + 1] (int64): c, then R; probs [M], balance [1] (fp32).
 */
int hsn_unit_router_forward(const void* logits, int64_t row, int dtype, const uint8_t* valid,
                            int64_t* units, float* shares, int64_t* tally, float* probs,
                            float* balance, int n, int M, int k, void* workspace,
                            int64_t workspace_bytes, void* stream);

/*
 * d_logits [n, M] (dense, `dtype`) from the forward's logits, valid, units and tally, and the cotangents
 * g = d_shares [n, k] (rows g_row elements apart) and b = d_balance [1] (fp32, either NULL: zero). For a
 * live token, with s its shares and c' = b M / R:
 *   d_j = s_j (g_j - sum s g) where j is chosen, + c' p_j (load_j - sum p load)
 * A unit outside [0, M) is an empty slot. d_logits must not overlap the inputs.
 */
int hsn_unit_router_backward(const void* logits, int64_t row, int dtype, const uint8_t* valid,
                             const int64_t* units, const int64_t* tally, const float* d_shares,
                             int64_t g_row, const float* d_balance, void* d_logits, int n, int M,
                             int k, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSN_UNIT_ROUTER_H */
