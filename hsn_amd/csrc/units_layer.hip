// A whole layer of routed units for a few tokens (include/hsn_units_layer.h), in three launches:
// the router's products and the choice (a workgroup a token), the hidden units (a lane a column of
// one chosen unit of one token), the outputs (a lane a column of one token, over its K units).
#include "../../include/hsn_units_layer.h"
#include "abi_util.h"
#include "common.cuh"
#include "unit_math.cuh"

namespace hsn {
namespace units_layer {
namespace {

constexpr int kMaxUnits = HSN_UNITS_MAX, kMaxChosen = HSN_UNITS_MAX_CHOSEN;

struct Args {
    const void *x, *router, *W1, *b1, *W2, *b2;
    void* y;
    int64_t x_row;
    int* unit;      // [n, K] the choice
    float* share;   // [n, K]
    float* hidden;  // [n, K, H]
    int n, M, K, d_in, H, d_out, activation;
};

template <typename E>
__global__ __launch_bounds__(256) void route(Args a) {
    __shared__ float logit[kMaxUnits];
    const int i = blockIdx.x, lane = threadIdx.x % kWave;
    const E* x = static_cast<const E*>(a.x) + i * a.x_row;
    for (int m = threadIdx.x / kWave; m < a.M; m += 4) {
        const E* w = static_cast<const E*>(a.router) + int64_t(m) * a.d_in;
        float sum = 0.0f;
        for (int k = lane; k < a.d_in; k += kWave) sum = __builtin_fmaf(to_f32(x[k]), to_f32(w[k]), sum);
        for (int d = 1; d < kWave; d *= 2) sum += wave_shfl_xor(sum, d);
        if (lane == 0) logit[m] = sum;
    }
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    // the K largest by (key, lowest unit), one a round
    float top = 0.0f, sum = 0.0f, mine = 0.0f;
    bool taken[kMaxUnits / kWave] = {};
    for (int k = 0; k < a.K; ++k) {
        uint64_t best = 0;
        for (int j = 0; j < kMaxUnits / kWave; ++j) {
            const int m = j * kWave + lane;
            if (m < a.M && !taken[j])
                best = max(best, uint64_t(score_key(logit[m])) << 32 | uint32_t(~m));
        }
        for (int d = 1; d < kWave; d *= 2)
            best = max(best, uint64_t(__shfl_xor(static_cast<unsigned long long>(best), d, kWave)));
        const int m = static_cast<int>(~static_cast<uint32_t>(best));
        for (int j = 0; j < kMaxUnits / kWave; ++j) taken[j] |= m == j * kWave + lane;
        if (k == 0) top = logit[m];
        const float e = expf(logit[m] - top);
        sum += e;
        if (lane == k) mine = e;
        if (lane == 0) a.unit[i * a.K + k] = m;
    }
    if (lane < a.K) a.share[i * a.K + lane] = mine / sum;
}

template <typename E>
__global__ __launch_bounds__(64) void up(Args a) {
    const int col = blockIdx.x * 64 + threadIdx.x, pair = blockIdx.y;
    if (col >= a.H) return;
    const bool gated = a.activation == HSN_UNITS_SWIGLU;
    const int H1 = gated ? 2 * a.H : a.H;
    const int64_t unit = a.unit[pair];
    const E* x = static_cast<const E*>(a.x) + (pair / a.K) * a.x_row;
    const E* w = static_cast<const E*>(a.W1) + unit * a.d_in * H1 + col;
    const E* b = static_cast<const E*>(a.b1) + unit * H1 + col;
    float z = a.b1 ? to_f32(b[0]) : 0.0f, g = a.b1 && gated ? to_f32(b[a.H]) : 0.0f;
    for (int k = 0; k < a.d_in; ++k) {
        const float v = to_f32(x[k]);
        z = __builtin_fmaf(v, to_f32(w[int64_t(k) * H1]), z);
        if (gated) g = __builtin_fmaf(v, to_f32(w[int64_t(k) * H1 + a.H]), g);
    }
    a.hidden[int64_t(pair) * a.H + col] = gated ? z * act_sigmoid(z) * g : units::gelu(z);
}

template <typename E>
__global__ __launch_bounds__(64) void down(Args a) {
    const int col = blockIdx.x * 64 + threadIdx.x, i = blockIdx.y;
    if (col >= a.d_out) return;
    float y = 0.0f;
    for (int k = 0; k < a.K; ++k) {
        const int pair = i * a.K + k;
        const int64_t unit = a.unit[pair];
        const E* w = static_cast<const E*>(a.W2) + unit * a.H * a.d_out + col;
        const float* v = a.hidden + int64_t(pair) * a.H;
        float z = a.b2 ? to_f32(static_cast<const E*>(a.b2)[unit * a.d_out + col]) : 0.0f;
        for (int j = 0; j < a.H; ++j) z = __builtin_fmaf(v[j], to_f32(w[int64_t(j) * a.d_out]), z);
        y = __builtin_fmaf(a.share[pair], z, y);
    }
    static_cast<E*>(a.y)[int64_t(i) * a.d_out + col] = from_f32<E>(y);
}

void check(int n, int M, int K, int d_in, int H, int d_out, int dtype, int activation) {
    HSN_REQUIRE(dtype == HSN_DTYPE_F32 || dtype == HSN_DTYPE_F16 || dtype == HSN_DTYPE_BF16,
                HSN_ERR_UNSUPPORTED_DTYPE, "dtype must be F32, F16 or BF16");
    HSN_REQUIRE(activation == HSN_UNITS_GELU || activation == HSN_UNITS_SWIGLU,
                HSN_ERR_INVALID_ARGUMENT, "unknown activation");
    HSN_REQUIRE(n >= 0 && M >= 1 && K >= 1 && d_in >= 1 && H >= 1 && d_out >= 1,
                HSN_ERR_INVALID_ARGUMENT, "n >= 0 and every other size >= 1");
    HSN_REQUIRE(K <= M, HSN_ERR_INVALID_ARGUMENT, "K <= M");
    HSN_REQUIRE(n <= HSN_UNITS_MAX_TOKENS && M <= kMaxUnits && K <= kMaxChosen,
                HSN_ERR_SIZE_OVERFLOW, "at most 64 tokens, 256 units and 16 chosen");
    HSN_REQUIRE(d_in <= 65536 && H <= 65536 && d_out <= 65536, HSN_ERR_SIZE_OVERFLOW,
                "widths of at most 65536");
}

int64_t layout(Args* a, char* base, int n, int K, int H) {
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char* p = base + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    char* unit = take(4LL * n * K);
    char* share = take(4LL * n * K);
    char* hidden = take(4LL * n * K * H);
    if (a) {
        a->unit = reinterpret_cast<int*>(unit);
        a->share = reinterpret_cast<float*>(share);
        a->hidden = reinterpret_cast<float*>(hidden);
    }
    return at;
}

template <typename E>
void launch(const Args& a, hipStream_t st) {
    route<E><<<a.n, 256, 0, st>>>(a);
    up<E><<<dim3((a.H + 63) / 64, a.n * a.K), 64, 0, st>>>(a);
    down<E><<<dim3((a.d_out + 63) / 64, a.n), 64, 0, st>>>(a);
}

}  // namespace
}  // namespace units_layer
}  // namespace hsn

using namespace hsn;
using namespace hsn::units_layer;

extern "C" int hsn_units_layer_workspace(int n, int M, int K, int d_in, int H, int d_out, int dtype,
                                         int activation, int64_t* bytes) {
    HSN_ABI_BEGIN
    check(n, M, K, d_in, H, d_out, dtype, activation);
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    *bytes = layout(nullptr, nullptr, n, K, H);
    HSN_ABI_END
}

extern "C" int hsn_units_layer(const void* x, int64_t x_row, const void* router, const void* W1,
                               const void* b1, const void* W2, const void* b2, void* y, int n,
                               int M, int K, int d_in, int H, int d_out, int dtype, int activation,
                               void* workspace, int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    check(n, M, K, d_in, H, d_out, dtype, activation);
    if (n == 0) return HSN_OK;
    HSN_REQUIRE(x && router && W1 && W2 && y && workspace, HSN_ERR_INVALID_ARGUMENT,
                "a required pointer is NULL");
    Args a{x, router, W1, b1, W2, b2, y, x_row, nullptr, nullptr, nullptr, n, M, K, d_in, H, d_out,
           activation};
    HSN_REQUIRE(workspace_bytes >= layout(&a, static_cast<char*>(workspace), n, K, H),
                HSN_ERR_INVALID_ARGUMENT, "the workspace is too small");
    if (dtype == HSN_DTYPE_F32)
        launch<float>(a, as_stream(stream));
    else if (dtype == HSN_DTYPE_F16)
        launch<_Float16>(a, as_stream(stream));
    else
        launch<bf16_t>(a, as_stream(stream));
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
