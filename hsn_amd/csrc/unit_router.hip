// The choice of units in training, their load with its balance loss, and the gradient
// (include/hsn_unit_router.h).
//
// A token is a group of G lanes with four units each (G the power of two that holds M), so a wave takes
// 64 / G tokens at a time, and maxima and sums over a token are lane steps. The k units are chosen one after
// the other: the group's largest key, its first lane, that lane's first unit. Each lane adds the
// probabilities and counts of its own units over all tokens that it meets; lanes, waves and at last
// workgroups are added in a fixed order, so the sums repeat, and a second launch makes the balance of them.
//
// The backward takes the probabilities again from the logits. The chosen slots of a wave's tokens go through
// LDS to the lanes that hold their units.
#include <algorithm>

#include "../../include/hsn_unit_router.h"
#include "abi_util.h"
#include "packs.cuh"

namespace hsn {
namespace router {
namespace {

constexpr int kEach = 4;  // units a lane
constexpr int kWaves = 8, kThreads = kWaves * kWave;
constexpr int kMostGroups = 512;        // workgroups of the forward: two a compute unit
constexpr int kMostBackward = 2048;
constexpr int kFlush = 128;             // tokens that a lane adds in fp32
constexpr int kFinish = 1024, kFinishUnits = 16, kFinishSlices = kFinish / kFinishUnits;
constexpr float kLog2 = 1.4426950408889634f;
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // score_key(-inf)

struct Args {
    const void* logits;
    int64_t row;
    const uint8_t* valid;
    int64_t* units;
    float* shares;
    int64_t* tally;
    float *probs, *balance;
    int n, M, k;
    // workspace: of each forward workgroup; of each workgroup that finishes
    double* part_probs;     // [groups, M]
    uint32_t* part_counts;  // [groups, M + 1], the live tokens last
    double* part_dot;       // [finishing]: sum of c_e prob_e
    int64_t* part_chosen;   // [finishing]: sum of c_e
    uint32_t* arrived;
    int groups;
    // backward
    const float *g, *d_balance;
    int64_t g_row;
    void* d_logits;
};

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2); }

template <int G>
__device__ __forceinline__ float group_largest(float v) {
    if constexpr (G >= 2) v = fmaxf(v, dpp_f32<dpp::kXor1>(v));
    if constexpr (G >= 4) v = fmaxf(v, dpp_f32<dpp::kXor2>(v));
    if constexpr (G >= 8) v = fmaxf(v, dpp_f32<dpp::kHalfMirror>(v));
    if constexpr (G >= 16) v = fmaxf(v, dpp_f32<dpp::kRor8>(v));
    if constexpr (G >= 32) {
        const RowPair r = pair16(__float_as_uint(v));
        v = fmaxf(__uint_as_float(r.lo), __uint_as_float(r.hi));
    }
    if constexpr (G >= 64) {
        const RowPair r = pair32(__float_as_uint(v));
        v = fmaxf(__uint_as_float(r.lo), __uint_as_float(r.hi));
    }
    return v;
}

// The bits of a ballot that are this lane's group's, from bit 0 on.
template <int G>
__device__ __forceinline__ uint64_t of_group(uint64_t lanes) {
    if constexpr (G == kWave) return lanes;
    return lanes >> (lane_id() / G * G) & ((uint64_t(1) << (G % kWave)) - 1);
}

// A lane's four logits of a token; -inf behind the last unit and where there is no token.
template <typename E>
__device__ __forceinline__ void load_units(const E* row, int unit, int M, bool there, float (&x)[kEach]) {
    if (there && unit + kEach <= M) {
        E e[kEach];
        __builtin_memcpy(e, row + unit, sizeof(e));
#pragma unroll
        for (int j = 0; j < kEach; ++j) x[j] = to_f32(e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            x[j] = there && unit + j < M ? to_f32(row[unit + j]) : -__builtin_inff();
    }
}

template <typename E, int G>
__global__ __launch_bounds__(kThreads) void route_tokens(const Args a) {
    constexpr int kTokens = kWave / G;  // a wave takes at a time
    __shared__ double probs[kWaves][G * kEach];
    __shared__ uint32_t counts[kWaves][G * kEach], rows[kWaves];
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id(), sub = lane % G, unit = sub * kEach;
    const E* logits = static_cast<const E*>(a.logits);
    float sum[kEach] = {};
    double whole[kEach] = {};
    uint32_t count[kEach] = {}, live_tokens = 0;
    const int step = a.groups * kWaves * kTokens;
    int turn = 0;
    for (int64_t t = (int64_t(blockIdx.x) * kWaves + wave) * kTokens; t < a.n; t += step) {
        const int64_t i = t + lane / G;
        const bool there = i < a.n;
        float x[kEach];
        load_units(logits + i * a.row, unit, a.M, there, x);
        const bool wanted = there && (!a.valid || a.valid[i]);
        uint32_t key[kEach];
        int rank[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            key[j] = score_key(x[j]);
            key[j] = wanted && key[j] > kKeyNegInf ? key[j] : 0;  // 0: not to be chosen
            rank[j] = -1;
        }
        float m = 0.0f, chosen = 0.0f;
        int found = 0;
        for (int r = 0; r < a.k; ++r) {
            const uint32_t mine = umax(umax(key[0], key[1]), umax(key[2], key[3]));
            const uint32_t most = group_max<G>(mine);
            const float value =
                __uint_as_float(most ^ (static_cast<int32_t>(most) < 0 ? 0x80000000u : 0xffffffffu));
            if (r == 0) m = value;
            if (most) {
                chosen += exp_of(value - m);
                found = r + 1;
            }
            const uint64_t lanes = of_group<G>(ballot(mine == most));
            if (most && sub == __builtin_ctzll(lanes)) {
                bool open = true;
#pragma unroll
                for (int j = 0; j < kEach; ++j) {
                    const bool it = open && key[j] == most;
                    open = open && !it;
                    rank[j] = it ? r : rank[j];
                    key[j] = it ? 0 : key[j];
                }
            }
        }
        const bool live = found > 0;
        float e[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) e[j] = live ? exp_of(x[j] - m) : 0.0f;
        const float total = group_sum<G>((e[0] + e[1]) + (e[2] + e[3]));
        const float part = live ? 1.0f / total : 0.0f, share = live ? 1.0f / chosen : 0.0f;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            sum[j] += e[j] * part;
            if (rank[j] >= 0) {
                ++count[j];
                a.units[i * a.k + rank[j]] = unit + j;
                a.shares[i * a.k + rank[j]] = e[j] * share;
            }
        }
        if (there && sub == 0) {
            live_tokens += live;
            for (int r = found; r < a.k; ++r) {
                a.units[i * a.k + r] = -1;
                a.shares[i * a.k + r] = 0.0f;
            }
        }
        if (++turn % kFlush == 0) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) whole[j] += sum[j], sum[j] = 0.0f;
        }
    }
    // lanes that hold the same units, then waves
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        whole[j] += sum[j];
#pragma unroll
        for (int mask = G; mask < kWave; mask *= 2) {
            whole[j] += __shfl_xor(whole[j], mask, kWave);
            count[j] += __shfl_xor(count[j], mask, kWave);
        }
    }
#pragma unroll
    for (int mask = G; mask < kWave; mask *= 2) live_tokens += __shfl_xor(live_tokens, mask, kWave);
    if (lane < G) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            probs[wave][unit + j] = whole[j];
            counts[wave][unit + j] = count[j];
        }
        if (lane == 0) rows[wave] = live_tokens;
    }
    __syncthreads();
    for (int u = threadIdx.x; u <= a.M; u += kThreads) {
        double p = 0.0;
        uint32_t c = 0;
        for (int w = 0; w < kWaves; ++w) {
            if (u < a.M) p += probs[w][u];
            c += u < a.M ? counts[w][u] : rows[w];
        }
        if (u < a.M) a.part_probs[int64_t(blockIdx.x) * a.M + u] = p;
        a.part_counts[int64_t(blockIdx.x) * (a.M + 1) + u] = c;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.arrived = 0;  // for the launch after this one
}

// The workgroups' sums added, 16 units a workgroup; the last one that arrives makes the balance.
__global__ __launch_bounds__(kFinish) void route_finish(const Args a) {
    __shared__ double probs[kFinishSlices][kFinishUnits];
    __shared__ int64_t counts[kFinishSlices][kFinishUnits], rows[kFinishSlices];
    const int u = blockIdx.x * kFinishUnits + threadIdx.x % kFinishUnits, slice = threadIdx.x / kFinishUnits;
    double p = 0.0;
    int64_t c = 0, r = 0;
    for (int g = slice; g < a.groups; g += kFinishSlices) {
        if (u < a.M) {
            p += a.part_probs[int64_t(g) * a.M + u];
            c += a.part_counts[int64_t(g) * (a.M + 1) + u];
        }
        r += a.part_counts[int64_t(g) * (a.M + 1) + a.M];
    }
    probs[slice][threadIdx.x % kFinishUnits] = p;
    counts[slice][threadIdx.x % kFinishUnits] = c;
    if (threadIdx.x % kFinishUnits == 0) rows[slice] = r;
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    const int lane = threadIdx.x;
    r = rows[lane];  // 64 slices: a lane each
#pragma unroll
    for (int mask = 32; mask; mask >>= 1) r += __shfl_xor(r, mask, kWave);
    // four lanes a unit, a quarter of the slices each
    p = 0.0, c = 0;
    for (int s = lane / kFinishUnits; s < kFinishSlices; s += kWave / kFinishUnits) {
        p += probs[s][lane % kFinishUnits];
        c += counts[s][lane % kFinishUnits];
    }
#pragma unroll
    for (int mask = kFinishUnits; mask < kWave; mask *= 2) {
        p += __shfl_xor(p, mask, kWave);
        c += __shfl_xor(c, mask, kWave);
    }
    p /= static_cast<double>(r > 0 ? r : 1);
    const bool mine = lane < kFinishUnits && u < a.M;
    if (mine) {
        a.tally[u] = c;
        a.probs[u] = static_cast<float>(p);
    }
    double dot = mine ? static_cast<double>(c) * p : 0.0;
    int64_t chosen = mine ? c : 0;
#pragma unroll
    for (int mask = 32; mask; mask >>= 1) {
        dot += __shfl_xor(dot, mask, kWave);
        chosen += __shfl_xor(chosen, mask, kWave);
    }
    if (lane) return;
    if (blockIdx.x == 0) a.tally[a.M] = r;
    if (gridDim.x > 1) {
        a.part_dot[blockIdx.x] = dot;
        a.part_chosen[blockIdx.x] = chosen;
        __threadfence();  // this lane's own stores, before it counts itself
        if (atomicAdd(a.arrived, 1u) + 1 < gridDim.x) return;
        __threadfence();
        dot = 0.0, chosen = 0;
        for (uint32_t g = 0; g < gridDim.x; ++g) {
            dot += __hip_atomic_load(a.part_dot + g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            chosen += __hip_atomic_load(a.part_chosen + g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    *a.balance = static_cast<float>(a.M * dot / static_cast<double>(chosen > 0 ? chosen : 1));
}

constexpr int kBackWaves = 4, kBackThreads = kBackWaves * kWave;

template <typename E, int G>
__global__ __launch_bounds__(kBackThreads) void route_backward(const Args a) {
    constexpr int kTokens = kWave / G;
    __shared__ float2 slots[kBackWaves][kTokens][G * kEach];  // whether a unit is chosen, its cotangent
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id(), sub = lane % G, unit = sub * kEach;
    float2* const mine = slots[wave][lane / G] + unit;
    const E* logits = static_cast<const E*>(a.logits);
    E* to = static_cast<E*>(a.d_logits);
    float load[kEach];
    double all = 0.0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const double c = unit + j < a.M ? static_cast<double>(a.tally[unit + j]) : 0.0;
        load[j] = static_cast<float>(c);
        all += c;
    }
#pragma unroll
    for (int mask = 1; mask < G; mask *= 2) all += __shfl_xor(all, mask, kWave);
#pragma unroll
    for (int j = 0; j < kEach; ++j) load[j] = all > 0.0 ? static_cast<float>(load[j] / all) : 0.0f;
    const int64_t rows = a.tally[a.M];
    const float pull = a.d_balance && rows > 0
                           ? static_cast<float>(static_cast<double>(*a.d_balance) * a.M / static_cast<double>(rows))
                           : 0.0f;
    const int step = gridDim.x * kBackWaves * kTokens;
    for (int64_t t = (int64_t(blockIdx.x) * kBackWaves + wave) * kTokens; t < a.n; t += step) {
        const int64_t i = t + lane / G;
        const bool there = i < a.n;
        float x[kEach];
        load_units(logits + i * a.row, unit, a.M, there, x);
        const bool wanted = there && (!a.valid || a.valid[i]);
        if (a.g) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) mine[j] = make_float2(0.0f, 0.0f);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
            const int64_t left = a.n - t;
            const int n_slots = static_cast<int>(left < kTokens ? left : kTokens) * a.k;
            for (int s = lane; s < n_slots; s += kWave) {
                const int token = s / a.k;
                const int64_t u = a.units[t * a.k + s];
                if (u >= 0 && u < a.M)
                    slots[wave][token][u] = make_float2(1.0f, a.g[(t + token) * a.g_row + (s - token * a.k)]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
        }
        const float m = group_largest<G>(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        const bool strange = x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3];
        const bool live = wanted && (m > -__builtin_inff() || of_group<G>(ballot(strange)) != 0);
        float p[kEach], d[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) p[j] = exp_of(x[j] - m);
        const float part = 1.0f / group_sum<G>((p[0] + p[1]) + (p[2] + p[3]));
        float toward = 0.0f;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            p[j] *= part;
            toward = __builtin_fmaf(p[j], load[j], toward);
        }
        toward = group_sum<G>(toward);
#pragma unroll
        for (int j = 0; j < kEach; ++j) d[j] = pull * p[j] * (load[j] - toward);
        if (a.g) {
            float mass = 0.0f, mean = 0.0f;
            float2 v[kEach];
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                v[j] = mine[j];
                const float q = v[j].x != 0.0f ? p[j] : 0.0f;
                mass += q;
                mean = __builtin_fmaf(q, v[j].y, mean);
            }
            mass = group_sum<G>(mass);
            mean = group_sum<G>(mean);
            const float share = mass != 0.0f ? 1.0f / mass : 0.0f;  // (no unit chosen: 0)
            mean *= share;
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (v[j].x != 0.0f) d[j] = __builtin_fmaf(p[j] * share, v[j].y - mean, d[j]);
        }
        if (!there) continue;
        E out[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) out[j] = from_f32<E>(live ? d[j] : 0.0f);
        E* at = to + i * a.M + unit;
        if (unit + kEach <= a.M) {
            __builtin_memcpy(at, out, sizeof(out));
        } else {
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (unit + j < a.M) at[j] = out[j];
        }
    }
}

// ------------------------------------------------------------------------------------------
// Launches.
// ------------------------------------------------------------------------------------------

int size_of(int dtype) { return dtype == HSN_DTYPE_F32 ? 4 : 2; }

int lanes_of(int M) {  // G
    int g = 1;
    while (g * kEach < M) g *= 2;
    return g;
}

int groups_of(int n, int M) {
    const int64_t tokens = int64_t(kWaves) * (kWave / lanes_of(M));
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMostGroups, (n + tokens - 1) / tokens)));
}

int finishing(int M) { return (M + kFinishUnits - 1) / kFinishUnits; }

int64_t layout(Args& a, char* at) {
    char* const begin = at;
    const auto take = [&](int64_t bytes) {
        char* p = at;
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    a.part_probs = reinterpret_cast<double*>(take(8 * int64_t(a.groups) * a.M));
    a.part_counts = reinterpret_cast<uint32_t*>(take(4 * int64_t(a.groups) * (a.M + 1)));
    a.part_dot = reinterpret_cast<double*>(take(8 * finishing(a.M)));
    a.part_chosen = reinterpret_cast<int64_t*>(take(8 * finishing(a.M)));
    a.arrived = reinterpret_cast<uint32_t*>(take(4));
    return at - begin;
}

template <typename F>
void with_lanes(int M, F&& f) {
    using std::integral_constant;
    switch (lanes_of(M)) {
        case 1: return f(integral_constant<int, 1>());
        case 2: return f(integral_constant<int, 2>());
        case 4: return f(integral_constant<int, 4>());
        case 8: return f(integral_constant<int, 8>());
        case 16: return f(integral_constant<int, 16>());
        case 32: return f(integral_constant<int, 32>());
        default: return f(integral_constant<int, 64>());
    }
}
template <typename F>
void with_type(int dtype, F&& f) {
    if (dtype == HSN_DTYPE_F32)
        f(float{});
    else if (dtype == HSN_DTYPE_F16)
        f(_Float16{});
    else
        f(bf16_t{});
}

void check(int n, int M, int k, int dtype) {
    HSN_REQUIRE(dtype == HSN_DTYPE_F32 || dtype == HSN_DTYPE_F16 || dtype == HSN_DTYPE_BF16,
                HSN_ERR_UNSUPPORTED_DTYPE, "logits must be F32, F16 or BF16");
    HSN_REQUIRE(n >= 0 && M >= 1, HSN_ERR_INVALID_ARGUMENT, "n >= 0 and M >= 1");
    HSN_REQUIRE(M <= HSN_ROUTER_MAX_UNITS && n < 1 << 30, HSN_ERR_SIZE_OVERFLOW,
                "at most 256 units and fewer than 2^30 tokens");
    HSN_REQUIRE(k >= 1 && k <= std::min(M, HSN_ROUTER_MAX_CHOSEN), HSN_ERR_INVALID_ARGUMENT,
                "k in [1, min(M, 16)]");
}

}  // namespace
}  // namespace router
}  // namespace hsn

using namespace hsn;
using namespace hsn::router;

extern "C" int hsn_unit_router_workspace(int n, int M, int dtype, int64_t* bytes) {
    HSN_ABI_BEGIN
    check(n, M, 1, dtype);
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    Args a{};
    a.M = M, a.groups = groups_of(n, M);
    *bytes = layout(a, nullptr);
    HSN_ABI_END
}

extern "C" int hsn_unit_router_forward(const void* logits, int64_t row, int dtype, const uint8_t* valid,
                                       int64_t* units, float* shares, int64_t* tally, float* probs,
                                       float* balance, int n, int M, int k, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    check(n, M, k, dtype);
    HSN_REQUIRE((n == 0 || (logits && units && shares)) && tally && probs && balance && workspace,
                HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size_of(dtype) == 0, HSN_ERR_INVALID_ARGUMENT,
                "logits must be aligned to their type");
    Args a{};
    a.logits = logits, a.row = row, a.valid = valid, a.units = units, a.shares = shares, a.tally = tally;
    a.probs = probs, a.balance = balance, a.n = n, a.M = M, a.k = k, a.groups = groups_of(n, M);
    HSN_REQUIRE(workspace_bytes >= layout(a, static_cast<char*>(workspace)), HSN_ERR_INVALID_ARGUMENT,
                "the workspace is too small");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                "the workspace must be aligned to 16 bytes");
    hipStream_t st = as_stream(stream);
    with_type(dtype, [&](auto e) {
        with_lanes(M, [&](auto g) {
            route_tokens<decltype(e), decltype(g)::value><<<a.groups, kThreads, 0, st>>>(a);
        });
    });
    HSN_HIP(hipGetLastError());
    route_finish<<<finishing(M), kFinish, 0, st>>>(a);
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}

extern "C" int hsn_unit_router_backward(const void* logits, int64_t row, int dtype, const uint8_t* valid,
                                        const int64_t* units, const int64_t* tally, const float* d_shares,
                                        int64_t g_row, const float* d_balance, void* d_logits, int n, int M,
                                        int k, void* stream) {
    HSN_ABI_BEGIN
    check(n, M, k, dtype);
    if (n == 0) return HSN_OK;
    HSN_REQUIRE(logits && units && tally && d_logits, HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size_of(dtype) == 0 &&
                    reinterpret_cast<uintptr_t>(d_logits) % size_of(dtype) == 0,
                HSN_ERR_INVALID_ARGUMENT, "logits and d_logits must be aligned to their type");
    Args a{};
    a.logits = logits, a.row = row, a.valid = valid, a.units = const_cast<int64_t*>(units);
    a.tally = const_cast<int64_t*>(tally), a.n = n, a.M = M, a.k = k;
    a.g = d_shares, a.g_row = g_row, a.d_balance = d_balance, a.d_logits = d_logits;
    hipStream_t st = as_stream(stream);
    with_type(dtype, [&](auto e) {
        with_lanes(M, [&](auto g) {
            constexpr int kG = decltype(g)::value;
            const int64_t tokens = int64_t(kBackWaves) * (kWave / kG);
            const int grid = static_cast<int>(std::min<int64_t>(kMostBackward, (n + tokens - 1) / tokens));
            route_backward<decltype(e), kG><<<grid, kBackThreads, 0, st>>>(a);
        });
    });
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
