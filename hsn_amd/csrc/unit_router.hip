// The choice of units in training, their load with its balance loss, and the gradient
// (include/hsn_unit_router.h).
//
// A token is a group of G lanes with four units each (G the power of two that holds M), so a wave takes
// 64 / G tokens at a time, and maxima and sums over a token are lane steps. A unit's key is its logit's order
// above its number, so keys differ; a lane sorts its four, and the group's largest first key is the next
// unit chosen, k times, without a branch. Each lane adds the probabilities of its own units over all tokens
// that it meets; lanes, waves and at last workgroups are added in a fixed order, so the sums repeat, and a
// second launch makes the balance of them. Counts are whole numbers, added in LDS in any order.
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

constexpr int kMostGroups = 256;  // workgroups of the forward: one a compute unit, its sums are few to add
constexpr int kMostBackward = 2048;  // (65536 x 64 bf16 by 512 / 1024 / 2048 / 4096: 28.1 / 26.9 / 26.3 / 27.7 us)
constexpr int kFlush = 128;       // tokens that a lane adds in fp32
constexpr int kFinish = 1024;
constexpr float kLog2 = 1.4426950408889634f;

struct Args {
    const void* logits;
    int64_t row;
    const uint8_t* valid;
    int64_t* units;
    float* shares;
    int64_t* tally;
    float *probs, *balance;
    int n, M, k;
    // workspace: of each forward workgroup
    double* part_probs;     // [groups, M]
    uint32_t* part_counts;  // [groups, M]
    uint32_t* part_rows;    // [groups]: live tokens
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

// A lane's units are EACH from `begin` on, of which those from `own` on are its own: the last ones of M end
// with M, so that a token's logits are read by whole packs. (Where some lanes read their elements one by
// one, all of them unpack what they read at once and wait for it, and no load stays in flight.) Fewer
// than four units have a lane each.
template <typename E, int EACH>
struct Units {
    E e[EACH];
};
template <int EACH>
struct Place {
    int begin, own;
    __device__ Place(int sub, int M) {
        begin = max(0, min(sub * EACH, M - EACH));
        own = min(sub * EACH - begin, EACH);  // EACH: none
    }
    __device__ __forceinline__ bool mine(int j) const { return j >= own; }
};
template <typename E, int EACH>
__device__ __forceinline__ Units<E, EACH> load_units(const E* p) {
    Units<E, EACH> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}

// A unit's key: the larger the logit, and among equal ones the lower the unit, the larger; NaN above all. Below
// kLeast is -inf, which is never chosen (or nothing: 0).
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
    const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return x == x ? k : 0xffffffffu;
}
__device__ __forceinline__ float of_order(uint32_t k) {
    return __uint_as_float(k ^ (static_cast<int32_t>(k) < 0 ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kLowest = 0x00800000u;  // that is larger than -inf's

template <typename E>
struct Order {  // a 16-bit logit in fp32 leaves at least 13 low bits free: 8 for the unit
    static_assert(HSN_ROUTER_MAX_UNITS <= 256, "8 bits hold a unit");
    using Key = uint32_t;
    static constexpr Key kLeast = kLowest;
    static __device__ __forceinline__ Key key(float x, int unit) {
        return (order_of(x) & 0xffffff00u) | (255u - unit);
    }
    static __device__ __forceinline__ float value(Key k) {
        return __uint_as_float(static_cast<int32_t>(k) < 0 ? (k & 0xffffff00u) ^ 0x80000000u : ~(k | 0xffu));
    }
    static __device__ __forceinline__ int unit(Key k) { return 255 - static_cast<int>(k & 255); }
    template <int G>
    static __device__ __forceinline__ Key largest(Key k) {
        return group_max<G>(k);
    }
};
template <>
struct Order<float> {
    using Key = uint64_t;
    static constexpr Key kLeast = uint64_t(kLowest) << 32;
    static __device__ __forceinline__ Key key(float x, int unit) {
        return uint64_t(order_of(x)) << 32 | (0xffffffffu - unit);
    }
    static __device__ __forceinline__ float value(Key key) { return of_order(static_cast<uint32_t>(key >> 32)); }
    static __device__ __forceinline__ int unit(Key k) {
        return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
    }
    template <int G>
    static __device__ __forceinline__ Key largest(Key k) {
        const uint32_t hi = static_cast<uint32_t>(k >> 32), most = group_max<G>(hi);
        return uint64_t(most) << 32 | group_max<G>(hi == most ? static_cast<uint32_t>(k) : 0u);
    }
};

template <typename K>
__device__ __forceinline__ void order(K& a, K& b) {
    const K hi = a > b ? a : b;
    b = a > b ? b : a;
    a = hi;
}

template <typename E, int G, int EACH, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void route_tokens(const Args a) {
    constexpr int kTokens = kWave / G;  // a wave takes at a time
    constexpr int kThreads = WAVES * kWave;
    // slots that a lane of a group writes: k is at most 16 and at most the units
    constexpr int kMostK = G * EACH < HSN_ROUTER_MAX_CHOSEN ? G * EACH : HSN_ROUTER_MAX_CHOSEN;
    constexpr int kSlots = (kMostK + G - 1) / G;
    using O = Order<E>;
    using Key = typename O::Key;
    __shared__ double probs[WAVES][G * EACH];
    __shared__ uint32_t counts[G * EACH], rows;
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id(), sub = lane % G;
    const Place<EACH> place(sub, a.M);
    for (int u = threadIdx.x; u < G * EACH; u += kThreads) counts[u] = 0;
    if (threadIdx.x == 0) rows = 0;
    const E* logits = static_cast<const E*>(a.logits) + place.begin;
    float sum[EACH] = {};
    double whole[EACH] = {};
    uint32_t live_tokens = 0;
    // (n is below 2^30 and a step at most 2^19; addresses are stepped, not multiplied, from turn to turn)
    const int step = a.groups * WAVES * kTokens;
    int t = (static_cast<int>(blockIdx.x) * WAVES + wave) * kTokens;
    // the next tokens' logits are in flight while these are worked on (a token behind the last one: the last)
    Units<E, EACH> next;
    uint8_t next_valid = 1;
    const E* from = logits + (t + lane / G) * a.row;
    const E* const last = logits + int64_t(a.n - 1) * a.row;
    const int64_t row_step = step * a.row;
    int64_t slot = int64_t(t + lane / G) * a.k + sub;
    const int64_t slot_step = int64_t(step) * a.k;
    const auto load = [&](int first) {
        const int i = first + lane / G;
        next = load_units<E, EACH>(i < a.n ? from : last);
        from += row_step;
        if (a.valid) next_valid = a.valid[i < a.n ? i : a.n - 1];
    };
    if (t < a.n) load(t);
    __syncthreads();
    int turn = 0;
    for (; t < a.n; t += step, slot += slot_step) {
        const bool there = t + lane / G < a.n;
        float x[EACH];
        Key key[EACH];
        const bool wanted = there && next_valid;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            x[j] = place.mine(j) ? to_f32(next.e[j]) : -__builtin_inff();
            key[j] = O::key(x[j], place.begin + j);
        }
        if (t + step < a.n) load(t + step);
        if constexpr (EACH == 4) {
            order(key[0], key[1]), order(key[2], key[3]), order(key[0], key[2]), order(key[1], key[3]);
            order(key[1], key[2]);
        }
        Key kept[kSlots], first = 0;
#pragma unroll
        for (int q = 0; q < kSlots; ++q) {
            kept[q] = 0;
            const int some = min(G, a.k - q * G);
            for (int s = 0; s < some; ++s) {
                const Key most = O::template largest<G>(key[0]);
                if (q == 0 && s == 0) first = most;
                const bool mine = key[0] == most;
#pragma unroll
                for (int j = 0; j < EACH; ++j) {  // (values: a choice between two places is made by number)
                    const Key own = key[j], behind = j + 1 < EACH ? Key(key[j + 1 < EACH ? j + 1 : j]) : Key(0);
                    key[j] = mine ? Key(behind) : Key(own);
                }
                kept[q] = sub == s ? most : kept[q];
            }
        }
        const bool live = wanted && first >= O::kLeast;
        const float m = O::value(first);
        float e[EACH], total = 0.0f;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            e[j] = exp_of(x[j] - m);
            total += e[j];
        }
        const float part = __builtin_amdgcn_rcpf(group_sum<G>(total));  // (1 ulp)
#pragma unroll
        for (int j = 0; j < EACH; ++j) sum[j] += live ? e[j] * part : 0.0f;
        float w[kSlots], chosen = 0.0f;
        bool is_one[kSlots];
#pragma unroll
        for (int q = 0; q < kSlots; ++q) {
            is_one[q] = wanted && kept[q] >= O::kLeast;
            w[q] = is_one[q] ? exp_of(O::value(kept[q]) - m) : 0.0f;
            chosen += w[q];
        }
        const float share = __builtin_amdgcn_rcpf(group_sum<G>(chosen));
#pragma unroll
        for (int q = 0; q < kSlots; ++q) {
            const int r = q * G + sub;
            if (r >= a.k || !there) continue;
            const int u = O::unit(kept[q]);
            a.units[slot + q * G] = is_one[q] ? u : -1;
            a.shares[slot + q * G] = is_one[q] ? w[q] * share : 0.0f;
            if (is_one[q]) atomicAdd(&counts[u], 1u);
        }
        live_tokens += live && sub == 0;
        if (++turn % kFlush == 0) {
#pragma unroll
            for (int j = 0; j < EACH; ++j) whole[j] += sum[j], sum[j] = 0.0f;
        }
    }
    // lanes that hold the same units, then waves
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const double v = wave_sum<G>(whole[j] + sum[j]);
        if (lane < G && place.mine(j)) probs[wave][place.begin + j] = v;
    }
    if (live_tokens) atomicAdd(&rows, live_tokens);
    __syncthreads();
    for (int u = threadIdx.x; u < a.M; u += kThreads) {
        double p = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) p += probs[w][u];
        a.part_probs[int64_t(blockIdx.x) * a.M + u] = p;
        a.part_counts[int64_t(blockIdx.x) * a.M + u] = counts[u];
    }
    if (threadIdx.x == 0) a.part_rows[blockIdx.x] = rows;
}

// The workgroups' sums added and the balance, by one workgroup: a thread a unit and a slice of them.
__global__ __launch_bounds__(kFinish) void route_finish(const Args a, int units) {  // units: a power of two >= M
    constexpr int kFlight = 8;
    __shared__ double probs[kFinish], s[3][kFinish / kWave];
    __shared__ uint64_t counts[kFinish];
    const int u = threadIdx.x % units, slice = threadIdx.x / units, slices = kFinish / units;
    const int at = min(u, a.M - 1);
    double p = 0.0, r = 0.0;
    uint64_t c = 0;
    for (int g0 = slice; g0 < a.groups; g0 += slices * kFlight) {
        double q[kFlight];
        uint32_t d[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            const int64_t g = min(g0 + f * slices, a.groups - 1);
            q[f] = a.part_probs[g * a.M + at];
            d[f] = a.part_counts[g * a.M + at];
        }
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            const bool there = g0 + f * slices < a.groups;
            p += there ? q[f] : 0.0;
            c += there ? d[f] : 0;
        }
    }
    if (static_cast<int>(threadIdx.x) < a.groups) r = a.part_rows[threadIdx.x];
    // the lanes of a wave that hold the same unit, then the threads that still do
    for (int mask = units; mask < kWave; mask *= 2) {
        p += __shfl_xor(p, mask, kWave);
        c += __shfl_xor(c, mask, kWave);
    }
    probs[threadIdx.x] = p;
    counts[threadIdx.x] = c;
    const int wave = threadIdx.x / kWave;
    r = wave_sum(r);
    if (threadIdx.x % kWave == 0) s[0][wave] = r;
    __syncthreads();
    if (threadIdx.x >= HSN_ROUTER_MAX_UNITS) return;  // (whole waves, that pass no further barrier)
    r = 0.0;
    for (int w = 0; w < kMostGroups / kWave; ++w) r += s[0][w];
    p = 0.0, c = 0;
    if (static_cast<int>(threadIdx.x) < a.M) {
        for (int i = threadIdx.x; i < kFinish; i += max(units, kWave)) {
            p += probs[i];
            c += counts[i];
        }
        p /= r > 0.0 ? r : 1.0;
        a.tally[threadIdx.x] = static_cast<int64_t>(c);
        a.probs[threadIdx.x] = static_cast<float>(p);
    }
    const double chosen = wave_sum(static_cast<double>(c)), dot = wave_sum(static_cast<double>(c) * p);
    if (threadIdx.x % kWave == 0) s[1][wave] = chosen, s[2][wave] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0, balance = 0.0;
        for (int w = 0; w < HSN_ROUTER_MAX_UNITS / kWave; ++w) all += s[1][w], balance += s[2][w];
        a.tally[a.M] = static_cast<int64_t>(r);
        *a.balance = static_cast<float>(a.M * balance / (all > 0.0 ? all : 1.0));
    }
}
static_assert(kMostGroups <= kFinish, "a thread a workgroup's live tokens");

constexpr int kBackWaves = 4, kBackThreads = kBackWaves * kWave;

template <typename E, int G, int EACH>
__global__ __launch_bounds__(kBackThreads) void route_backward(const Args a) {
    constexpr int kTokens = kWave / G;
    // slots of a wave's tokens that a lane brings: k is at most 16 and at most the units
    constexpr int kMostK = G * EACH < HSN_ROUTER_MAX_CHOSEN ? G * EACH : HSN_ROUTER_MAX_CHOSEN;
    constexpr int kSlots = (kTokens * kMostK + kWave - 1) / kWave;
    __shared__ float2 slots[kBackWaves][kTokens][G * EACH];  // whether a unit is chosen, its cotangent
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id(), sub = lane % G;
    const Place<EACH> place(sub, a.M);
    float2* const mine = slots[wave][lane / G];
    const E* logits = static_cast<const E*>(a.logits) + place.begin;
    E* to = static_cast<E*>(a.d_logits);
    // (n is below 2^30 and a step at most 2^19; addresses are stepped, not multiplied, from turn to turn)
    const int step = static_cast<int>(gridDim.x) * kBackWaves * kTokens;
    int t = (static_cast<int>(blockIdx.x) * kBackWaves + wave) * kTokens;
    const int behind = a.n - 1;  // a token behind the last one reads the last
    int token_of[kSlots];        // of the slots that the lane brings
    int64_t slot[kSlots], last_slot[kSlots], cot[kSlots], last_cot[kSlots];
#pragma unroll
    for (int q = 0; q < kSlots; ++q) {
        const int s = q * kWave + lane, rank = s % a.k;
        token_of[q] = s / a.k;
        slot[q] = int64_t(t + token_of[q]) * a.k + rank;
        last_slot[q] = int64_t(behind) * a.k + rank;
        cot[q] = (t + token_of[q]) * a.g_row + rank;
        last_cot[q] = behind * a.g_row + rank;
    }
    const E *from = logits + (t + lane / G) * a.row, *const last = logits + behind * a.row;
    int64_t at = int64_t(t + lane / G) * a.M + place.begin;
    const int64_t row_step = step * a.row, slot_step = int64_t(step) * a.k, cot_step = step * a.g_row;
    Units<E, EACH> next;
    uint8_t next_valid = 1;
    int64_t next_unit[kSlots];
    float next_g[kSlots];
    const auto bring = [&](int first) {
        const int i = first + lane / G;
        next = load_units<E, EACH>(i < a.n ? from : last);
        from += row_step;
        if (a.valid) next_valid = a.valid[min(i, behind)];
        if (a.g) {
#pragma unroll
            for (int q = 0; q < kSlots; ++q) {
                const bool there = first + token_of[q] < a.n;
                next_unit[q] = a.units[there ? slot[q] : last_slot[q]];
                next_g[q] = a.g[there ? cot[q] : last_cot[q]];
                slot[q] += slot_step;
                cot[q] += cot_step;
            }
        }
    };
    if (t < a.n) bring(t);
    double count[EACH], all = 0.0;
    float load[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) count[j] = static_cast<double>(a.tally[place.begin + j]);
#pragma unroll
    for (int j = 0; j < EACH; ++j) all += place.mine(j) ? count[j] : 0.0;
#pragma unroll
    for (int mask = 1; mask < G; mask *= 2) all += __shfl_xor(all, mask, kWave);
    const double one = all > 0.0 ? 1.0 / all : 0.0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) load[j] = place.mine(j) ? static_cast<float>(count[j] * one) : 0.0f;
    const int64_t rows = a.tally[a.M];
    const float pull = a.d_balance && rows > 0
                           ? static_cast<float>(static_cast<double>(*a.d_balance) * a.M / static_cast<double>(rows))
                           : 0.0f;
    const int64_t at_step = int64_t(step) * a.M;
    for (; t < a.n; t += step, at += at_step) {
        const bool there = t + lane / G < a.n, wanted = there && next_valid;
        float x[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) x[j] = place.mine(j) ? to_f32(next.e[j]) : -__builtin_inff();
        if (a.g) {
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (place.mine(j)) mine[place.begin + j] = make_float2(0.0f, 0.0f);
            wave_order();
#pragma unroll
            for (int q = 0; q < kSlots; ++q)
                if (token_of[q] < kTokens && t + token_of[q] < a.n && next_unit[q] >= 0 && next_unit[q] < a.M)
                    slots[wave][token_of[q]][next_unit[q]] = make_float2(1.0f, next_g[q]);
            wave_order();
        }
        if (t + step < a.n) bring(t + step);
        float m = x[0];
        bool strange = false;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            m = fmaxf(m, x[j]);
            strange = strange || x[j] != x[j];
        }
        m = group_largest<G>(m);
        const bool live = wanted && (m > -__builtin_inff() || of_group<G>(ballot(strange)) != 0);
        float p[EACH], d[EACH], total = 0.0f;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            p[j] = exp_of(x[j] - m);
            total += p[j];
        }
        const float part = __builtin_amdgcn_rcpf(group_sum<G>(total));  // (1 ulp)
        float toward = 0.0f;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            p[j] *= part;
            toward = __builtin_fmaf(p[j], load[j], toward);
        }
        toward = group_sum<G>(toward);
#pragma unroll
        for (int j = 0; j < EACH; ++j) d[j] = pull * p[j] * (load[j] - toward);
        if (a.g) {
            float mass = 0.0f, mean = 0.0f;
            float2 v[EACH];
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                v[j] = mine[place.begin + j];
                const float q = v[j].x != 0.0f && place.mine(j) ? p[j] : 0.0f;
                mass += q;
                mean = __builtin_fmaf(q, v[j].y, mean);
            }
            mass = group_sum<G>(mass);
            mean = group_sum<G>(mean);
            const float share = mass != 0.0f ? __builtin_amdgcn_rcpf(mass) : 0.0f;  // (no unit chosen: 0)
            mean *= share;
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (v[j].x != 0.0f) d[j] = __builtin_fmaf(p[j] * share, v[j].y - mean, d[j]);
        }
        if (!there) continue;
        E out[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) out[j] = from_f32<E>(live ? d[j] : 0.0f);
        if (place.own == 0) {
            __builtin_memcpy(to + at, out, sizeof(out));
        } else {
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (place.mine(j)) to[at + j] = out[j];
        }
    }
}

// ------------------------------------------------------------------------------------------
// Launches.
// ------------------------------------------------------------------------------------------

int size_of(int dtype) { return dtype == HSN_DTYPE_F32 ? 4 : 2; }

// A token's lanes (G) and a lane's units.
int lanes_of(int M) {
    if (M < 4) return 4;
    int g = 1;
    while (g * 4 < M) g *= 2;
    return g;
}

// Waves of a forward workgroup: 16 where the tokens keep a workgroup of them on each compute unit busy, else 4,
// which leaves a SIMD to a wave (8192 tokens of 8 units: the launch 4.9 us, by workgroups of 16 waves 7.4).
int waves_of(int n, int M) { return n > int64_t(kMostGroups) * 4 * (kWave / lanes_of(M)) ? 16 : 4; }

int groups_of(int n, int M) {
    const int64_t tokens = int64_t(waves_of(n, M)) * (kWave / lanes_of(M));
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMostGroups, (n + tokens - 1) / tokens)));
}

int64_t layout(Args& a, char* at) {
    char* const begin = at;
    const auto take = [&](int64_t bytes) {
        char* p = at;
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    a.part_probs = reinterpret_cast<double*>(take(8 * int64_t(a.groups) * a.M));
    a.part_counts = reinterpret_cast<uint32_t*>(take(4 * int64_t(a.groups) * a.M));
    a.part_rows = reinterpret_cast<uint32_t*>(take(4 * int64_t(a.groups)));
    return at - begin;
}

template <typename F>
void with_lanes(int M, F&& f) {
    using std::integral_constant;
    constexpr integral_constant<int, 4> four;
    if (M < 4) return f(four, integral_constant<int, 1>());
    switch (lanes_of(M)) {
        case 1: return f(integral_constant<int, 1>(), four);
        case 2: return f(integral_constant<int, 2>(), four);
        case 4: return f(four, four);
        case 8: return f(integral_constant<int, 8>(), four);
        case 16: return f(integral_constant<int, 16>(), four);
        case 32: return f(integral_constant<int, 32>(), four);
        default: return f(integral_constant<int, 64>(), four);
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
        with_lanes(M, [&](auto g, auto each) {
            using E = decltype(e);
            constexpr int kG = decltype(g)::value, kEach = decltype(each)::value;
            const int waves = waves_of(n, M);
            (waves == 4 ? route_tokens<E, kG, kEach, 4>
                        : route_tokens<E, kG, kEach, 16>)<<<a.groups, waves * kWave, 0, st>>>(a);
        });
    });
    HSN_HIP(hipGetLastError());
    int units = 1;
    while (units < M) units *= 2;
    route_finish<<<1, kFinish, 0, st>>>(a, units);
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
        with_lanes(M, [&](auto g, auto each) {
            constexpr int kG = decltype(g)::value, kEach = decltype(each)::value;
            const int64_t tokens = int64_t(kBackWaves) * (kWave / kG);
            const int grid = static_cast<int>(std::min<int64_t>(kMostBackward, (n + tokens - 1) / tokens));
            route_backward<decltype(e), kG, kEach><<<grid, kBackThreads, 0, st>>>(a);
        });
    });
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
