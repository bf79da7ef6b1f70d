/*
 * hsn_units_layer.h -- a whole layer of routed units for a few tokens on MI355X (gfx950): the
 * router's products, the choice, the units and their weighted sum. For each of n tokens x[i]:
 *   l = router x[i] (fp32); S = the K units with the largest l (ties: the lowest unit);
 *   p = softmax of l over S;
 *   z = x[i] W1[e] + b1[e],  v = gelu(z) (HSN_UNITS_GELU: z/2 (1 + erf(z / sqrt 2)), H1 = H) or
 *   silu(z[:H]) z[H:] (HSN_UNITS_SWIGLU, H1 = 2 H);
 *   y[i] = sum over e in S of p[e] (v W2[e] + b2[e]).
 * x [n, d_in], router [M, d_in], W1 [M, d_in, H1], b1 [M, H1], W2 [M, H, d_out], b2 [M, d_out] and
 * y [n, d_out] are in `dtype` (HSN_DTYPE_F32, _F16 or _BF16), dense and row-major but for x, whose
 * rows are x_row elements apart; b1 and b2 may be NULL. The weights have the unit bank's layout
 * ([in, out], hsn_ops.h). Products are summed in fp32 and nothing is rounded to 16 bits before y.
 * 1 <= K <= min(M, HSN_UNITS_MAX_CHOSEN), M <= HSN_UNITS_MAX, n <= HSN_UNITS_MAX_TOKENS.
 *
 * workspace: hsn_units_layer_workspace() bytes of device memory, 16-byte aligned; its contents do
 * not matter before the call. Nothing is allocated and nothing is kept between calls, so the call
 * may be captured in a graph. Every sum has a fixed order. `stream` is a hipStream_t (NULL: the
 * default stream). The call returns once the work is enqueued, with the status codes of hsn_ops.h
 * and the message in hsn_win_last_error(). y must not overlap an input.
 */
#ifndef HSN_UNITS_LAYER_H
#define HSN_UNITS_LAYER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSN_UNITS_GELU 0
#define HSN_UNITS_SWIGLU 1
#define HSN_UNITS_MAX 256
#define HSN_UNITS_MAX_CHOSEN 16
#define HSN_UNITS_MAX_TOKENS 64

int hsn_units_layer_workspace(int n, int M, int K, int d_in, int H, int d_out, int dtype,
                              int activation, int64_t* bytes);
int hsn_units_layer(const void* x, int64_t x_row, const void* router, const void* W1,
                    const void* b1, const void* W2, const void* b2, void* y, int n, int M, int K,
                    int d_in, int H, int d_out, int dtype, int activation, void* workspace,
                    int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSN_UNITS_LAYER_H */
