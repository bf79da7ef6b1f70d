/*
 * hsn_embed.h -- the embedding of tokens and its gradient on MI355X (gfx950).
 *   out[i] = scale table[t_i],     d_table[v] = scale (sum over t_i = v of d_out[i])
 * for the B T tokens t[b, t] of a batch (B = 1 for a plain list). A token outside [0, V) is padding: its
 * row is zero and it has no gradient. A table row that no token names has gradient zero.
 * Types: HSN_DTYPE_F32, _F16 or _BF16, each of the table (and its gradient) and the rows (and their
 * cotangents) its own. Products are taken and sums held in fp32 and rounded once; the sum of a token's
 * cotangents is taken in the order of its positions, a span of them after the other, so the same call
 * gives the same bits.
 * Strides are counted in elements; the last dimension of table, out, d_out and d_table is contiguous.
 * tokens are int64 (token_bytes 8) or int32 (4). 1 <= V <= 2^24, 1 <= D <= 65536, B T < 2^26.
 *
 * Nothing is allocated and nothing is kept between calls, so a call may be captured in a graph.
 * `stream` is a hipStream_t (NULL: the default stream). The call returns once the work is enqueued,
 * with the status codes of hsn_ops.h and the message in hsn_win_last_error(). Outputs must not overlap
 * inputs.
 */
#ifndef HSN_EMBED_H
#define HSN_EMBED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSN_EMBED_MAX_TOKENS (1 << 24)
#define HSN_EMBED_MAX_WIDTH 65536

/* out [B, T, D], dense. */
int hsn_embed_forward(const void* tokens, int64_t token_b, int64_t token_t, int token_bytes,
                      const void* table, int64_t table_row, int table_dtype, float scale, void* out,
                      int out_dtype, int B, int T, int V, int D, void* stream);

/* Bytes of device workspace hsn_embed_backward needs, 16-byte aligned. Its contents do not matter before
 * the call. */
int hsn_embed_workspace(int B, int T, int V, int D, int d_out_dtype, int64_t* bytes);

/* d_table [V, D], dense. */
int hsn_embed_backward(const void* tokens, int64_t token_b, int64_t token_t, int token_bytes,
                       const void* d_out, int64_t d_out_b, int64_t d_out_t, int d_out_dtype,
                       float scale, void* d_table, int table_dtype, int B, int T, int V, int D,
                       void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSN_EMBED_H */
