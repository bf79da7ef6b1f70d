// The gated linear recurrence over whole sequences (include/hsn_scan.h): the entry points and the
// single position. The kernels over tiles are in scan.cuh.
#include "abi_util.h"
#include "scan.cuh"

namespace hsn {
namespace scan {
namespace {

// One position of n sequences: a lane a channel, `blocks` workgroups a sequence.
template <typename E>
__global__ __launch_bounds__(256) void step(const E* y, int64_t y_row, const E* gate,
                                            int64_t gate_row, int candidate_kind,
                                            const int32_t* rows, const uint8_t* reset,
                                            float* state, E* h, int S, int D, int blocks) {
    const int i = blockIdx.x / blocks, ch = blockIdx.x % blocks * 256 + threadIdx.x;
    if (ch >= D) return;
    const int row = rows ? rows[i] : i;
    float v = 0.0f;
    if (row >= 0 && row < S) {
        float* at = state + int64_t(row) * D + ch;
        float a, b;
        gates(to_f32(gate[i * gate_row + ch]), a, b);
        const float old = reset && reset[i] ? 0.0f : *at;
        const float in = to_f32(y[i * y_row + ch]);
        v = __builtin_fmaf(a, old, candidate_kind == HSN_SCAN_TANH ? b * tanh_of<E>(in) : linear_share(b) * in);
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

int size_of(int dtype) { return dtype == HSN_DTYPE_F32 ? 4 : 2; }

void check(int B, int T, int D, int dtype, int candidate_kind) {
    HSN_REQUIRE(dtype == HSN_DTYPE_F32 || dtype == HSN_DTYPE_F16 || dtype == HSN_DTYPE_BF16,
                HSN_ERR_UNSUPPORTED_DTYPE, "dtype must be F32, F16 or BF16");
    HSN_REQUIRE(candidate_kind == HSN_SCAN_TANH || candidate_kind == HSN_SCAN_LINEAR,
                HSN_ERR_INVALID_ARGUMENT, "unknown candidate");
    HSN_REQUIRE(B >= 0 && T >= 0 && D >= 1, HSN_ERR_INVALID_ARGUMENT, "B, T >= 0 and D >= 1");
    HSN_REQUIRE(T <= 1 << 30 && D <= 1 << 30, HSN_ERR_SIZE_OVERFLOW, "T, D <= 2^30");
}

// A grid's dimension holds fewer than 2^32 threads.
uint32_t grid(int64_t blocks, int threads) {
    HSN_REQUIRE(blocks < (int64_t(1) << 32) / threads, HSN_ERR_SIZE_OVERFLOW,
                "too many rows and channels for one grid");
    return static_cast<uint32_t>(blocks);
}

// Every word of the exchange starts at 0 (a kernel, so that the call may be captured).
__global__ __launch_bounds__(256) void clear(uint4* box, int64_t n) {
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i < n) box[i] = uint4{};
}

// No positions: the state is carried over.
__global__ __launch_bounds__(256) void carry_over(const float* from, float* to, int64_t n) {
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : 0.0f;
}

// How a pass runs: the tiles of a row, and whether each is a workgroup of its own.
struct Plan {
    int strips_a_row, tiles;
    int64_t strips, words;
    bool split;
};

Plan plan(int B, int T, int D, int tile) {
    Plan q;
    q.strips_a_row = (D + kChannels - 1) / kChannels;
    q.strips = int64_t(B) * q.strips_a_row;
    q.tiles = (T + tile - 1) / tile;
    // 256 strips fill the GPU's compute units. Up to 8 tiles a walk is then no slower than the split
    // (backward, 256 strips in fp32: 4 tiles 34 against 40 us), from 16 on the split is faster
    // (backward in bf16: 32 tiles 187 against 170 us). With fewer strips the split is faster from two
    // tiles on, with the launch that clears its words (6 strips, two tiles: forward 12.3 against 10.0
    // us, backward 11.2 against 9.8 us). Neither way is timed between 6 and 256 strips, nor between 4 and
    // 32 tiles but for these.
    q.split = q.tiles > 1 && (q.strips < 256 || q.tiles > 8);
    const int64_t groups = (q.tiles + kGroup - 1) / kGroup;
    q.words = q.split ? 64 + (q.tiles + groups) * q.strips * kChannels : 0;
    grid(q.strips * (q.split ? q.tiles : 1), kThreads);
    return q;
}

// Two elements a load where the row length, the strides and the addresses allow, else one.
int vector_of(int size, int D, std::initializer_list<const void*> at,
              std::initializer_list<int64_t> strides) {
    bool fits = D % 2 == 0;
    for (const void* p : at) fits &= reinterpret_cast<uintptr_t>(p) % (2 * size) == 0;
    for (int64_t s : strides) fits &= s % 2 == 0;
    return fits ? 2 : 1;
}

void run(Args& p, const Plan& q, int dtype, int vec, bool back, void* workspace,
         int64_t workspace_bytes, hipStream_t st) {
    p.strips_a_row = q.strips_a_row, p.strips = static_cast<int>(q.strips), p.tiles = q.tiles;
    p.reset_words = p.T % 4 == 0 && reinterpret_cast<uintptr_t>(p.reset) % 4 == 0;
    if (q.split) {
        HSN_REQUIRE(workspace && workspace_bytes >= 8 * q.words, HSN_ERR_INVALID_ARGUMENT,
                    "the workspace is too small");
        HSN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                    "the workspace must be aligned to 16 bytes");
        p.box = static_cast<uint64_t*>(workspace);
        const int64_t n = q.words / 2;
        clear<<<grid((n + 255) / 256, 256), 256, 0, st>>>(
            reinterpret_cast<uint4*>(p.box), n);
    }
    by_dtype(dtype, [&](auto e) {
        using E = decltype(e);
        back ? launch_backward<E>(p, vec, q.split, st) : launch_forward<E>(p, vec, q.split, st);
    });
    HSN_HIP(hipGetLastError());
}

void run_empty(const float* from, float* to, int64_t n, hipStream_t st) {
    carry_over<<<grid((n + 255) / 256, 256), 256, 0, st>>>(from, to, n);
    HSN_HIP(hipGetLastError());
}

}  // namespace
}  // namespace scan
}  // namespace hsn

using namespace hsn;
using namespace hsn::scan;

extern "C" int hsn_scan_workspace(int B, int T, int D, int dtype, int backward, int64_t* bytes) {
    HSN_ABI_BEGIN
    check(B, T, D, dtype, HSN_SCAN_TANH);
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    *bytes = 8 * plan(B, T, D, backward ? backward_tile() : forward_tile(size_of(dtype))).words;
    HSN_ABI_END
}

extern "C" int hsn_scan_forward(const void* y, int64_t y_row, int64_t y_pos, const void* gate,
                                int64_t gate_row, int64_t gate_pos, int dtype, int candidate_kind,
                                const uint8_t* reset, const float* h0, void* h, float* h_T,
                                float* marks, int B, int T, int D, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    check(B, T, D, dtype, candidate_kind);
    if (B == 0) return HSN_OK;
    HSN_REQUIRE(h_T && (T == 0 || (y && gate && h)), HSN_ERR_INVALID_ARGUMENT,
                "a required pointer is NULL");
    if (T == 0) {
        run_empty(h0, h_T, int64_t(B) * D, as_stream(stream));
        return HSN_OK;
    }
    Args p{};
    p.y = y, p.gate = gate, p.y_row = y_row, p.y_pos = y_pos, p.gate_row = gate_row;
    p.gate_pos = gate_pos, p.reset = reset, p.h0 = h0, p.h = h, p.h_T = h_T, p.marks = marks;
    p.T = T, p.D = D, p.candidate = candidate_kind;
    const int vec = vector_of(size_of(dtype), D, {y, gate, h},
                              {y_row, y_pos, gate_row, gate_pos});
    run(p, plan(B, T, D, forward_tile(size_of(dtype))), dtype, vec, false, workspace, workspace_bytes,
        as_stream(stream));
    HSN_ABI_END
}

extern "C" int hsn_scan_backward(const void* y, int64_t y_row, int64_t y_pos, const void* gate,
                                 int64_t gate_row, int64_t gate_pos, int dtype, int candidate_kind,
                                 const uint8_t* reset, const float* marks, const void* d_h,
                                 int64_t d_row, int64_t d_pos, const float* d_h_T, void* d_y,
                                 void* d_gate, float* d_h0, int B, int T, int D, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    check(B, T, D, dtype, candidate_kind);
    if (B == 0) return HSN_OK;
    HSN_REQUIRE(d_h0 && (T == 0 || (y && gate && marks && d_y && d_gate)),
                HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    if (T == 0) {
        run_empty(d_h_T, d_h0, int64_t(B) * D, as_stream(stream));
        return HSN_OK;
    }
    Args p{};
    p.y = y, p.gate = gate, p.d_h = d_h, p.y_row = y_row, p.y_pos = y_pos, p.gate_row = gate_row;
    p.gate_pos = gate_pos, p.d_row = d_row, p.d_pos = d_pos, p.reset = reset, p.d_h_T = d_h_T;
    p.marks = const_cast<float*>(marks), p.d_y = d_y, p.d_gate = d_gate, p.d_h0 = d_h0;
    p.T = T, p.D = D, p.candidate = candidate_kind;
    const int vec = vector_of(size_of(dtype), D, {y, gate, d_h, d_y, d_gate},
                              {y_row, y_pos, gate_row, gate_pos, d_row, d_pos});
    run(p, plan(B, T, D, backward_tile()), dtype, vec, true, workspace, workspace_bytes,
        as_stream(stream));
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
    const int64_t blocks = (int64_t(D) + 255) / 256;
    const uint32_t all = grid(n * blocks, 256);
    by_dtype(dtype, [&](auto e) {
        using E = decltype(e);
        step<E><<<all, 256, 0, as_stream(stream)>>>(
            static_cast<const E*>(y), y_row, static_cast<const E*>(gate), gate_row, candidate_kind,
            rows, reset, state, static_cast<E*>(h), S, D, static_cast<int>(blocks));
    });
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
