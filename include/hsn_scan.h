/*
 * hsn_scan.h -- the gated linear recurrence over whole sequences on MI355X (gfx950): the window's
 * update h' = h + b (c - h) where every channel is written at every position, so that the time
 * axis can be split and joined. With g = gate[r,t,:], y = y[r,t,:], and the state before the
 * position m h[t-1] (m = 0 where reset[r,t], else 1; h[-1] = h0):
 *   b = sigmoid(g), c = tanh(y) or y,   h[t] = (1 - b) (m h[t-1]) + b c
 * Shapes: B rows, T positions, D channels. y and gate are [B, T, D] in `dtype` (HSN_DTYPE_F32,
 * _F16 or _BF16) with the last index contiguous and any row and position strides, counted in
 * elements; every other tensor is dense and row-major. reset holds 0 or 1. States (h0, h_T, marks,
 * state and their cotangents) are fp32. T and D are at most 2^30, and a call whose rows, channels and
 * spans of time need more workgroups than one grid holds is refused.
 *
 * Everything is computed in fp32: a share b or 1 - b is right to about (1.25 |g| + 8) 2^-24 of
 * itself, a tanh to 2.7e-7 and to 3e-6 of itself (fp32 inputs) or 4e-5 (16-bit ones). A state that is
 * not finite ends at the next reset; until then a NaN stays one, and an infinity stays one or, where
 * spans are joined, becomes a NaN.
 *
 * Caller-allocated outputs; nothing is allocated and nothing is kept between calls, so every call
 * may be captured in a graph. `stream` is a hipStream_t (NULL: the default stream). Functions
 * return once the work is enqueued, with the status codes of hsn_ops.h and the message in
 * hsn_win_last_error(). Outputs must not overlap inputs, except the step's state.
 */
#ifndef HSN_SCAN_H
#define HSN_SCAN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSN_SCAN_TANH 0
#define HSN_SCAN_LINEAR 1

/* Positions between two kept states: marks is [B, ceil(T / HSN_SCAN_SPAN), D], the state before
 * every position that is a multiple of it (before that position's own reset). */
#define HSN_SCAN_SPAN 128

/* Bytes of device workspace hsn_scan_forward (backward = 0) or hsn_scan_backward (1) needs for
 * the shape; 0 where it needs none. Its contents do not matter before the call. */
int hsn_scan_workspace(int B, int T, int D, int dtype, int backward, int64_t* bytes);

/*
 * h [B, T, D] (dtype), the end state h_T [B, D] and, where marks is not NULL, the states the
 * backward starts from. reset [B, T] (uint8) and h0 [B, D] may be NULL (no resets; zero).
 * T may be 0: h_T = h0.
 */
int hsn_scan_forward(const void* y, int64_t y_row, int64_t y_pos, const void* gate,
                     int64_t gate_row, int64_t gate_pos, int dtype, int candidate,
                     const uint8_t* reset, const float* h0, void* h, float* h_T, float* marks,
                     int B, int T, int D, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * From the forward's inputs and marks, and the cotangents d_h [B, T, D] (dtype, strided as y; may
 * be NULL: zero) and d_h_T [B, D] (may be NULL), with l[t] the whole cotangent of h[t]:
 *   l[t] = d_h[t] + (1 - b[t+1]) m[t+1] l[t+1]   (d_h[T-1] takes d_h_T on top)
 *   d_y = b l c'(y),  d_gate = l b (1 - b) (c - m h[t-1]),  d_h0 = (1 - b[0]) m[0] l[0]
 * d_y and d_gate are dense [B, T, D] (dtype), d_h0 [B, D]. T may be 0: d_h0 = d_h_T.
 */
int hsn_scan_backward(const void* y, int64_t y_row, int64_t y_pos, const void* gate,
                      int64_t gate_row, int64_t gate_pos, int dtype, int candidate,
                      const uint8_t* reset, const float* marks, const void* d_h, int64_t d_row,
                      int64_t d_pos, const float* d_h_T, void* d_y, void* d_gate, float* d_h0,
                      int B, int T, int D, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * One position of n sequences whose states lie in a pool: sequence i reads and writes row rows[i]
 * of state [S, D] in place (rows NULL: row i, n <= S) from y, gate [n, D] (row strides in
 * elements) and reset [n] (may be NULL), and its new state is also h [n, D] in `dtype`. A row
 * outside [0, S) is padding: h is 0 there and no state is touched. The rows in range must be
 * distinct.
 */
int hsn_scan_step(const void* y, int64_t y_row, const void* gate, int64_t gate_row, int dtype,
                  int candidate, const int32_t* rows, const uint8_t* reset, float* state, void* h,
                  int n, int S, int D, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSN_SCAN_H */
