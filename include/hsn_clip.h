/*
 * hsn_clip.h -- the global norm of many gradients, and clipping by it, on MI355X (gfx950).
 *   norm = sqrt(sum of g^2 over every element of every tensor), in float64
 *   coefficient = min(1, max_norm / (norm + 1e-6)); 1 where the norm is infinite or NaN
 *   out_j = coefficient * grad_j (the product in float64, rounded to fp32 and then to the type)
 * The tensors are n lists of elements side by side in memory, each of its own type (HSN_DTYPE_F32,
 * _F16 or _BF16) and at any address that its type allows; a tensor may hold no element. Sums are taken
 * in an order that depends on the counts alone, so the same lists give the same bits.
 *
 * Nothing is allocated and nothing is kept between calls, so a call may be captured in a graph.
 * `stream` is a hipStream_t (NULL: the default stream). The call returns once the work is enqueued,
 * with the status codes of hsn_ops.h and the message in hsn_win_last_error().
 */
#ifndef HSN_CLIP_H
#define HSN_CLIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of device workspace hsn_clip needs for tensors of these element counts, 8-byte aligned. Its
 * contents do not matter before the call. */
int hsn_clip_workspace(const int64_t* numels, int n, int64_t* bytes);

/*
 * result: two float64 on the device, the norm and the coefficient. grads[j], outs[j] (device addresses)
 * hold numels[j] elements of type dtypes[j] each; the four lists are on the host. outs[j] may be
 * grads[j] (in place); otherwise no tensor written may overlap another one written or read. Where every
 * outs[j] is grads[j], a coefficient of 1 leaves the memory untouched. outs may be NULL: the norm and
 * the coefficient alone. max_norm >= 0 (infinity: no limit).
 */
int hsn_clip(const void* const* grads, void* const* outs, const int64_t* numels, const int* dtypes,
             int n, double max_norm, double* result, void* workspace, int64_t workspace_bytes,
             void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSN_CLIP_H */
