// What the gated linear recurrence's kernels share: a position's share kept, share written and
// candidate, in fp32.
#pragma once

#include "../../include/hsn_scan.h"
#include "common.cuh"
#include "dpp.cuh"

namespace hsn {
namespace scan {

// a = sigmoid(-g) (the share of the old state kept) and b = sigmoid(g) (the share written), each
// to a few ulps of itself: e = exp(-|g|) never overflows, and of 1/(1+e) and e/(1+e) neither is a
// difference from 1 (1 - b would leave nothing of a small a).
__device__ __forceinline__ void gates(float g, float& a, float& b) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * __builtin_fabsf(g));
    const float big = __builtin_amdgcn_rcpf(1.0f + e);
    const float small = e * big;
    a = g >= 0.0f ? small : big;
    b = g >= 0.0f ? big : small;
}

// tanh(y) to a few ulps of itself: (1 - e) / (1 + e) with e = exp(-2|y|), and the series
// y - y^3/3 + 2 y^5/15 below |y| = 1/16, where 1 - e cancels (the next term, 17 y^7 / 315, is
// under 4e-9 of y there).
__device__ __forceinline__ float tanh_exact(float y) {
    const float e = __builtin_amdgcn_exp2f(-2.0f * kLog2e * __builtin_fabsf(y));
    const float t = __builtin_copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), y);
    const float y2 = y * y;
    const float s = __builtin_fmaf(y2 * y, __builtin_fmaf(y2, 2.0f / 15.0f, -1.0f / 3.0f), y);
    return __builtin_fabsf(y) < 0.0625f ? s : t;
}

__device__ __forceinline__ float candidate(float y, int kind) {
    return kind == HSN_SCAN_TANH ? tanh_exact(y) : y;
}

}  // namespace scan
}  // namespace hsn
