// The gated linear recurrence over whole sequences (include/hsn_scan.h): forward, backward and
// the single position.
//
// Forward and backward: a lane walks one channel of one row through the positions. The backward
// makes a span's states again from the mark before it (the state itself is not read: 5 elements a
// position and channel instead of 6, and no rounding of h to the storage type in the gradient).
#include "abi_util.h"
#include "scan.cuh"

namespace hsn {
namespace scan {
namespace {

constexpr int kSpan = HSN_SCAN_SPAN;
constexpr int kThreads = 64;

struct Args {
    const void *y, *gate, *d_h;
    int64_t y_row, y_pos, gate_row, gate_pos, d_row, d_pos;
    const uint8_t* reset;
    const float *h0, *d_h_T;
    float *h_T, *marks, *d_h0;
    void *h, *d_y, *d_gate;
    int B, T, D, candidate;
};

template <typename E>
__global__ __launch_bounds__(kThreads) void walk_forward(Args p) {
    const int ch = blockIdx.x * kThreads + threadIdx.x, r = blockIdx.y;
    if (ch >= p.D) return;
    const E* y = static_cast<const E*>(p.y) + r * p.y_row + ch;
    const E* g = static_cast<const E*>(p.gate) + r * p.gate_row + ch;
    E* out = static_cast<E*>(p.h) + int64_t(r) * p.T * p.D + ch;
    float h = p.h0 ? p.h0[int64_t(r) * p.D + ch] : 0.0f;
    const int spans = (p.T + kSpan - 1) / kSpan;
    for (int t = 0; t < p.T; ++t) {
        if (p.marks && t % kSpan == 0) p.marks[(int64_t(r) * spans + t / kSpan) * p.D + ch] = h;
        if (p.reset && p.reset[int64_t(r) * p.T + t]) h = 0.0f;
        float a, b;
        gates(to_f32(g[t * p.gate_pos]), a, b);
        h = __builtin_fmaf(a, h, b * candidate(to_f32(y[t * p.y_pos]), p.candidate));
        out[int64_t(t) * p.D] = from_f32<E>(h);
    }
    p.h_T[int64_t(r) * p.D + ch] = h;
}

template <typename E>
__global__ __launch_bounds__(kThreads) void walk_backward(Args p) {
    const int ch = blockIdx.x * kThreads + threadIdx.x, r = blockIdx.y;
    if (ch >= p.D) return;
    const E* y = static_cast<const E*>(p.y) + r * p.y_row + ch;
    const E* g = static_cast<const E*>(p.gate) + r * p.gate_row + ch;
    const E* d = static_cast<const E*>(p.d_h) + r * p.d_row + ch;
    E* dy = static_cast<E*>(p.d_y) + int64_t(r) * p.T * p.D + ch;
    E* dg = static_cast<E*>(p.d_gate) + int64_t(r) * p.T * p.D + ch;
    const int spans = (p.T + kSpan - 1) / kSpan;
    float mu = p.d_h_T ? p.d_h_T[int64_t(r) * p.D + ch] : 0.0f;  // the cotangent from later on
    for (int s = spans - 1; s >= 0; --s) {
        float q[kSpan];  // d_gate is l q, with q = a b (c - m h[t-1])
        float h = p.marks[(int64_t(r) * spans + s) * p.D + ch];
#pragma unroll
        for (int i = 0; i < kSpan; ++i) {
            const int t = s * kSpan + i;
            q[i] = 0.0f;
            if (t >= p.T) continue;
            if (p.reset && p.reset[int64_t(r) * p.T + t]) h = 0.0f;
            float a, b;
            gates(to_f32(g[t * p.gate_pos]), a, b);
            const float c = candidate(to_f32(y[t * p.y_pos]), p.candidate);
            q[i] = a * b * (c - h);
            h = __builtin_fmaf(a, h, b * c);
        }
#pragma unroll
        for (int i = kSpan - 1; i >= 0; --i) {
            const int t = s * kSpan + i;
            if (t >= p.T) continue;
            float a, b;
            gates(to_f32(g[t * p.gate_pos]), a, b);
            const float c = candidate(to_f32(y[t * p.y_pos]), p.candidate);
            const float l = (p.d_h ? to_f32(d[t * p.d_pos]) : 0.0f) + mu;
            dy[int64_t(t) * p.D] =
                from_f32<E>(l * b * (p.candidate == HSN_SCAN_TANH ? 1.0f - c * c : 1.0f));
            dg[int64_t(t) * p.D] = from_f32<E>(l * q[i]);
            mu = p.reset && p.reset[int64_t(r) * p.T + t] ? 0.0f : a * l;
        }
    }
    p.d_h0[int64_t(r) * p.D + ch] = mu;
}

template <typename E>
__global__ __launch_bounds__(256) void step(const E* y, int64_t y_row, const E* gate,
                                            int64_t gate_row, int candidate_kind,
                                            const int32_t* rows, const uint8_t* reset,
                                            float* state, E* h, int S, int D) {
    const int ch = blockIdx.x * 256 + threadIdx.x, i = blockIdx.y;
    if (ch >= D) return;
    const int row = rows ? rows[i] : i;
    float v = 0.0f;
    if (row >= 0 && row < S) {
        float* at = state + int64_t(row) * D + ch;
        float a, b;
        gates(to_f32(gate[i * gate_row + ch]), a, b);
        const float old = reset && reset[i] ? 0.0f : *at;
        v = __builtin_fmaf(a, old, b * candidate(to_f32(y[i * y_row + ch]), candidate_kind));
        *at = v;
    }
    h[int64_t(i) * D + ch] = from_f32<E>(v);
}

template <typename F>
void by_dtype(int dtype, F&& f) {
    if (dtype == HSN_DTYPE_F32) return f(float{});
    if (dtype == HSN_DTYPE_F16) return f(_Float16{});
    return f(bf16_t{});
}

void check(int B, int T, int D, int dtype, int candidate_kind) {
    HSN_REQUIRE(dtype == HSN_DTYPE_F32 || dtype == HSN_DTYPE_F16 || dtype == HSN_DTYPE_BF16,
                HSN_ERR_UNSUPPORTED_DTYPE, "dtype must be F32, F16 or BF16");
    HSN_REQUIRE(candidate_kind == HSN_SCAN_TANH || candidate_kind == HSN_SCAN_LINEAR,
                HSN_ERR_INVALID_ARGUMENT, "unknown candidate");
    HSN_REQUIRE(B >= 0 && T >= 0 && D >= 1, HSN_ERR_INVALID_ARGUMENT, "B, T >= 0 and D >= 1");
    HSN_REQUIRE(B <= 65535, HSN_ERR_SIZE_OVERFLOW, "at most 65535 rows");
}

}  // namespace
}  // namespace scan
}  // namespace hsn

using namespace hsn;
using namespace hsn::scan;

extern "C" int hsn_scan_workspace(int B, int T, int D, int dtype, int backward, int64_t* bytes) {
    HSN_ABI_BEGIN
    (void)backward;
    check(B, T, D, dtype, HSN_SCAN_TANH);
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    *bytes = 0;
    HSN_ABI_END
}

extern "C" int hsn_scan_forward(const void* y, int64_t y_row, int64_t y_pos, const void* gate,
                                int64_t gate_row, int64_t gate_pos, int dtype, int candidate_kind,
                                const uint8_t* reset, const float* h0, void* h, float* h_T,
                                float* marks, int B, int T, int D, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    (void)workspace, (void)workspace_bytes;
    check(B, T, D, dtype, candidate_kind);
    if (B == 0) return HSN_OK;
    HSN_REQUIRE(h_T && (T == 0 || (y && gate && h)), HSN_ERR_INVALID_ARGUMENT,
                "a required pointer is NULL");
    Args p{};
    p.y = y, p.gate = gate, p.y_row = y_row, p.y_pos = y_pos, p.gate_row = gate_row;
    p.gate_pos = gate_pos, p.reset = reset, p.h0 = h0, p.h = h, p.h_T = h_T, p.marks = marks;
    p.B = B, p.T = T, p.D = D, p.candidate = candidate_kind;
    by_dtype(dtype, [&](auto e) {
        walk_forward<decltype(e)><<<dim3((D + kThreads - 1) / kThreads, B), kThreads, 0, as_stream(stream)>>>(p);
    });
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}

extern "C" int hsn_scan_backward(const void* y, int64_t y_row, int64_t y_pos, const void* gate,
                                 int64_t gate_row, int64_t gate_pos, int dtype, int candidate_kind,
                                 const uint8_t* reset, const float* marks, const void* d_h,
                                 int64_t d_row, int64_t d_pos, const float* d_h_T, void* d_y,
                                 void* d_gate, float* d_h0, int B, int T, int D, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    (void)workspace, (void)workspace_bytes;
    check(B, T, D, dtype, candidate_kind);
    if (B == 0) return HSN_OK;
    HSN_REQUIRE(d_h0 && (T == 0 || (y && gate && marks && d_y && d_gate)),
                HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    Args p{};
    p.y = y, p.gate = gate, p.d_h = d_h, p.y_row = y_row, p.y_pos = y_pos, p.gate_row = gate_row;
    p.gate_pos = gate_pos, p.d_row = d_row, p.d_pos = d_pos, p.reset = reset, p.d_h_T = d_h_T;
    p.marks = const_cast<float*>(marks), p.d_y = d_y, p.d_gate = d_gate, p.d_h0 = d_h0;
    p.B = B, p.T = T, p.D = D, p.candidate = candidate_kind;
    by_dtype(dtype, [&](auto e) {
        walk_backward<decltype(e)><<<dim3((D + kThreads - 1) / kThreads, B), kThreads, 0, as_stream(stream)>>>(p);
    });
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}

extern "C" int hsn_scan_step(const void* y, int64_t y_row, const void* gate, int64_t gate_row,
                             int dtype, int candidate_kind, const int32_t* rows,
                             const uint8_t* reset, float* state, void* h, int n, int S, int D,
                             void* stream) {
    HSN_ABI_BEGIN
    check(n, 1, D, dtype, candidate_kind);
    HSN_REQUIRE(S >= 0 && (rows || n <= S), HSN_ERR_INVALID_ARGUMENT,
                "without rows the pool holds a state for every sequence");
    if (n == 0) return HSN_OK;
    HSN_REQUIRE(y && gate && h && (state || S == 0), HSN_ERR_INVALID_ARGUMENT,
                "a required pointer is NULL");
    by_dtype(dtype, [&](auto e) {
        using E = decltype(e);
        step<E><<<dim3((D + 255) / 256, n), 256, 0, as_stream(stream)>>>(
            static_cast<const E*>(y), y_row, static_cast<const E*>(gate), gate_row, candidate_kind,
            rows, reset, state, static_cast<E*>(h), S, D);
    });
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
