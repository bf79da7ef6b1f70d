// Log probabilities of given tokens with the entropy, the most probable alternatives and the gradient
// (include/hsn_score.h).
//
// Forward: one pass over the logits. A thread keeps S = sum e^(l - m) and W = sum e^(l - m) (l - m) of what it
// has seen, from a reference m that it raises to a batch's largest logit once that is well above; lanes, waves
// and a row's parts are joined in a fixed order, from the largest logit. A batch's 16 or 32 numbers are added
// in fp32, by pairs or fours, and a thread's batches in float64: they are up to 2^12 of a row, and sums in
// one fp32 number round the same way where logits are alike (a background at -2.3 of 1048576: 3e-5 of S). The joins
// are few steps, in fp32: in float64 too, 8192 x 32000 bf16 took 102 us instead of 93 and 1 x 32000 8.5 instead of 8.0.
// Where alternatives are wanted, each thread also notes the largest logit of each batch in LDS. After the pass
// the 64 columns' largest logits give a bound that k logits reach and few more do; the batches with such a
// one, some k of them, are read once more, and what reaches the bound goes to a list, where each finds its
// rank among the others. (Taken as the pass goes, by a bound that rises, candidates cost 1000 x 131071 bf16 11 us
// for 5 alternatives and 27 for 20; so, 8 and 15.) A list that is full, of equal logits, is cut to its k largest.
// The parts' sorted lists are merged by one wave, a list a lane.
//
// Backward: d = g ([j = t] - p) - h p (log p + H), a pack at a time from the logits and four numbers a row.
//
// Both are bound by memory where rows are many: the forward reads n V logits, the backward reads and
// writes as many.
#include <algorithm>

#include "../../include/hsn_score.h"
#include "abi_util.h"
#include "packs.cuh"

namespace hsn {
namespace score {
namespace {

constexpr int kBatch = 4;      // packs a thread has in flight
constexpr int kMostParts = 64;  // of a row: a lane each when they are joined
constexpr int kList = 256;      // candidates of a wave
constexpr float kLowest = -3.402823466e38f;
constexpr float kAbove = 4.0f;  // a reference is raised by more than this, so a sum is scaled (and rounded) few times
constexpr float kLog2 = 1.4426950408889634f;
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // score_key(-inf)
constexpr uint64_t kNone = uint64_t(kKeyNegInf) << 32 | 0xffffffffu;  // no candidate is this small

struct Args {
    const void* logits;
    int64_t row;
    const void* tokens;
    int64_t token_stride;
    bool wide;  // 64-bit tokens
    float *logprob, *entropy, *top_logprobs;
    int64_t* top_tokens;
    float4* stats;
    int V, top, parts, part_packs;
    float4* part_sums;     // [n, parts] m, S, W
    uint64_t* part_lists;  // [n, parts, top]
    // backward
    const float *g, *h;
    int64_t g_stride, h_stride;
    void* d_logits;
    __device__ __forceinline__ int64_t token(int i) const {
        return wide ? static_cast<const int64_t*>(tokens)[i * token_stride]
                    : static_cast<const int32_t*>(tokens)[i * token_stride];
    }
};

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2); }

// S and W of some logits from the reference m. Of none: 0, 0 and the lowest number.
template <typename F>
struct Sums {
    F S = 0, W = 0;
    float m = kLowest;
    // The same sums from another reference. What is not finite in m and to enters S by the logits alone.
    __device__ __forceinline__ void raise(float to) {
        const float d = fmaxf(m - to, -1e30f);  // the difference may leave fp32's range
        const F f = exp_of(d);
        W = f * (d * S + W);
        S = f * S;
        m = to;
    }
};

template <int G>
__device__ __forceinline__ float group_largest(float v) {
    v = fmaxf(v, dpp_f32<dpp::kXor1>(v));
    v = fmaxf(v, dpp_f32<dpp::kXor2>(v));
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

// The sums of G lanes added, from the largest of `most`: each lane's largest logit, or below its m.
template <int G>
__device__ __forceinline__ void join_lanes(Sums<float>& s, float most) {
    s.raise(group_largest<G>(fmaxf(s.m, most)));
    s.S = group_sum<G>(s.S);
    s.W = group_sum<G>(s.W);
}

// ------------------------------------------------------------------------------------------
// Candidates: 64-bit numbers, the logit's order above the token's (the lower token the larger).
// ------------------------------------------------------------------------------------------

__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ (static_cast<int32_t>(k) < 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t candidate(float l, int token) {
    return uint64_t(score_key(l)) << 32 | (0xffffffffu - static_cast<uint32_t>(token));
}

// The largest of a wave's numbers, that are different or 0.
__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
    const uint32_t hi = static_cast<uint32_t>(v >> 32), lo = static_cast<uint32_t>(v);
    const uint32_t most = group_max<kWave>(hi);
    const uint64_t lanes = ballot(hi == most);
    if (__popcll(lanes) == 1) return uint64_t(most) << 32 | readlane(lo, __builtin_ctzll(lanes));
    return uint64_t(most) << 32 | group_max<kWave>(hi == most ? lo : 0u);
}

struct Candidates {
    uint64_t* list;  // kList of this wave's, in LDS
    int k, count = 0;
    uint64_t above = kNone;  // candidates are larger than this
    float from = -__builtin_inff();  // and their logits at least this
    float lane_most = -__builtin_inff();  // the largest logit that the lane has seen
    __device__ Candidates(uint64_t* l, int top) : list(l), k(top) {}

    // Leaves the k largest, sorted.
    __device__ void cut() {
        wave_order();
        const int lane = lane_id();
        constexpr int kEach = kList / kWave;
        uint64_t mine[kEach], kept = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine[i] = i * kWave + lane < count ? list[i * kWave + lane] : 0;
        const int n = min(count, k);
        for (int r = 0; r < n; ++r) {
            uint64_t most = mine[0];
#pragma unroll
            for (int i = 1; i < kEach; ++i) most = mine[i] > most ? mine[i] : most;
            most = wave_largest(most);
#pragma unroll
            for (int i = 0; i < kEach; ++i) mine[i] = mine[i] == most ? 0 : mine[i];
            if (lane == r) kept = most;
            if (r == k - 1) above = most;
        }
        wave_order();
        if (lane < n) list[lane] = kept;
        count = n;
        from = fmaxf(from, key_value(static_cast<uint32_t>(above >> 32)));
    }

    // Raises the bound to the k-th largest of the lanes' numbers (to 16 bits of its key, from below).
    __device__ __forceinline__ void bound(float most) {
        const uint32_t key = score_key(most);
        uint32_t least = 0;
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t test = least | 1u << bit;
            if (__popcll(ballot(key >= test)) >= k) least = test;
        }
        if (least > kKeyNegInf) from = fmaxf(from, key_value(least));
    }

    template <typename E, int N>
    __device__ __forceinline__ void take(const Pack<E> (&v)[N], const float (&most)[N], const int (&first)[N]) {
#pragma unroll
        for (int b = 0; b < N; ++b) {
            if (!ballot(most[b] >= from)) continue;
#pragma unroll
            for (int j = 0; j < Pack<E>::kN; ++j) {
                const float l = v[b][j];
                if (ballot(l >= from)) put(l, candidate(l, first[b] + j));
            }
        }
    }
    __device__ __forceinline__ void put(float l, uint64_t c) {
        uint64_t lanes = ballot(l >= from && c > above);
        if (count + __popcll(lanes) > kList) {
            cut();
            lanes = ballot(l >= from && c > above);
        }
        if (lanes >> lane_id() & 1) list[count + lanes_below(lanes)] = c;
        count += __popcll(lanes);
    }
    // The list's numbers from the bound on, at most 64, to `to`, where `*filled` counts them.
    __device__ __forceinline__ void leave(uint64_t* to, uint32_t* filled) {
        wave_order();
        const int lane = lane_id();
        constexpr int kEach = kList / kWave;
        uint64_t c[kEach], lanes[kEach];
        int n = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            c[i] = i * kWave + lane < count ? list[i * kWave + lane] : 0;
            lanes[i] = ballot(c[i] && key_value(static_cast<uint32_t>(c[i] >> 32)) >= from);
            n += __popcll(lanes[i]);
        }
        if (n > kWave) {  // (equal logits, or a row whose every next logit is a new largest one)
            cut();
            wave_order();
            c[0] = lane < count ? list[lane] : 0;
            lanes[0] = ballot(c[0] != 0);
            n = count;
#pragma unroll
            for (int i = 1; i < kEach; ++i) lanes[i] = 0;
        }
        int at = 0;
        if (lane == 0) at = static_cast<int>(atomicAdd(filled, static_cast<uint32_t>(n)));
        at = uniform(at);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (lanes[i] >> lane & 1) to[at + lanes_below(lanes[i])] = c[i];
            at += __popcll(lanes[i]);
        }
    }
};

// The k largest of `lists` sorted lists (a lane each, `each` numbers apart, 0 behind the last), lane r the
// r-th.
__device__ __forceinline__ uint64_t merge(const uint64_t* all, int lists, int each, int k) {
    const int lane = lane_id();
    const uint64_t* mine = all + lane * each;
    int at = 0;
    uint64_t head = lane < lists ? mine[0] : 0, kept = 0;
    for (int r = 0; r < k; ++r) {
        const uint64_t most = wave_largest(head);
        if (lane == r) kept = most;
        if (head == most && most) head = ++at < k ? mine[at] : 0;
    }
    return kept;
}

// A row's values from its sums: one wave, lane 0 and the lanes of the alternatives.
template <typename E>
__device__ __forceinline__ void write_row(const Args& a, int i, const Sums<float>& s, uint64_t best) {
    const int lane = lane_id();
    const bool none = s.S == 0.0f;
    const float rest = none ? 0.0f : logf(s.S);
    if (lane == 0) {
        const int64_t t = a.token(i);
        float logprob = 0.0f;
        if (t >= 0 && t < a.V) {
            const float l = to_f32(static_cast<const E*>(a.logits)[i * a.row + t]);
            logprob = none ? -__builtin_inff() : (l - s.m) - rest;
            if (s.S != s.S) logprob = s.S;
        }
        const float entropy = none ? 0.0f : rest - s.W / s.S;
        a.logprob[i] = logprob;
        a.entropy[i] = entropy;
        if (a.stats) a.stats[i] = make_float4(s.m, none ? 0.0f : 1.0f / s.S, rest, entropy);
    }
    if (lane < a.top) {
        const bool there = best != 0;
        const float l = key_value(static_cast<uint32_t>(best >> 32));
        a.top_tokens[int64_t(i) * a.top + lane] =
            there ? int64_t(0xffffffffu - static_cast<uint32_t>(best)) : int64_t(-1);
        a.top_logprobs[int64_t(i) * a.top + lane] = there ? (l - s.m) - rest : -__builtin_inff();
    }
}

// A row's packs begin on a 16-byte boundary (a vocabulary that is odd leaves most rows off one, and packs from
// the row's start would lie across two cache lines: 1000 x 131071 bf16 59 us instead of 49 without
// alternatives). The elements before the first pack and after the last one are the row's rest.
template <typename E>
struct RowPacks {
    static constexpr int kN = Pack<E>::kN;
    int skip, V, packs;
    __device__ RowPacks(const E* row, int v) : V(v) {
        skip = min(static_cast<int>(-reinterpret_cast<uintptr_t>(row) % 16 / sizeof(E)), V);
        packs = (V - skip) / kN;
    }
    __device__ __forceinline__ int first(int pack) const { return skip + pack * kN; }
    // the i-th element of the rest, V: none
    __device__ __forceinline__ int rest(int i) const { return i < skip ? i : min(packs * kN + i, V); }
    __device__ __forceinline__ bool has_rest() const { return packs * kN < V; }
};

template <typename E>
__device__ __forceinline__ Pack<E> no_pack() {
    Pack<E> v;
#pragma unroll
    for (int j = 0; j < Pack<E>::kN; ++j) v.e[j] = from_f32<E>(-__builtin_inff());
    return v;
}

// The k-th largest of the workgroup's 64 columns' largest logits is a bound for its candidates: k different
// logits are as large. A column is a lane of every wave; about k logits are above its bound (64 ln(64 / (64 -
// k)) where they lie anywhere), 24 for k = 20.
template <int WAVES>
__device__ __forceinline__ void share_bound(Candidates& c, float (*columns)[kWave]) {
    float most = c.lane_most;
    if constexpr (WAVES > 1) {
        const int wave = threadIdx.x / kWave, lane = lane_id();
        columns[wave][lane] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) most = fmaxf(most, columns[w][lane]);
    }
    c.bound(most);
}

// A workgroup a part of a row.
template <typename E, int WAVES, bool TOP>
__global__ __launch_bounds__(WAVES * kWave) void score_rows(const Args a) {
    constexpr int kThreads = WAVES * kWave, kN = Pack<E>::kN;
    // a thread's largest logit of each span of its batches (its order's upper half), to find the candidates again
    constexpr int kSpans = WAVES == 16 ? 8 : 32;
    __shared__ float wave_sums[WAVES][3];
    __shared__ uint64_t lists[TOP ? WAVES : 1][TOP ? kList : 1], left[TOP ? kThreads : 1], sorted[kWave];
    __shared__ float columns[TOP ? WAVES : 1][kWave];
    __shared__ uint16_t spans[TOP ? kSpans : 1][TOP ? kThreads : 1];
    __shared__ uint32_t filled;
    const int i = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id();
    const E* row = static_cast<const E*>(a.logits) + i * a.row;
    const RowPacks<E> in(row, a.V);
    const int begin = part * a.part_packs;
    const int end = part + 1 == a.parts ? in.packs : min(in.packs, begin + a.part_packs);
    const bool last = part + 1 == a.parts;
    constexpr int kPacks = kBatch * kThreads;  // of a batch
    const int batches = (end - begin + kPacks - 1) / kPacks, span = (batches + kSpans - 1) / kSpans;
    Sums<double> sums;
    Candidates c(lists[TOP ? wave : 0], a.top);
    if constexpr (TOP) {
        if (threadIdx.x == 0) filled = 0;
        if (wave == 0) sorted[lane] = 0;
    }
    const auto largest = [](const auto& v, auto& most) {
        constexpr int N = sizeof(v) / sizeof(v[0]);
#pragma unroll
        for (int b = 0; b < N; ++b) {
            most[b] = v[b][0];
#pragma unroll
            for (int j = 1; j < kN; ++j) most[b] = fmaxf(most[b], v[b][j]);
        }
        float all = most[0];
#pragma unroll
        for (int b = 1; b < N; ++b) all = fmaxf(all, most[b]);
        return all;
    };
    const auto add = [&](const auto& v, float all) {
        constexpr int N = sizeof(v) / sizeof(v[0]);
        c.lane_most = fmaxf(c.lane_most, all);
        if (all > sums.m + kAbove) sums.raise(all);
        float S[N], W[N];
#pragma unroll
        for (int b = 0; b < N; ++b) {
            float e[kN], w[kN / 4];
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                float x = v[b][j] - sums.m;
                e[j] = exp_of(x);
                x = fmaxf(x, -200.0f);  // e is 0 there, and x may be -inf
                w[j / 4] = j % 4 ? __builtin_fmaf(e[j], x, w[j / 4]) : e[j] * x;
            }
#pragma unroll
            for (int j = 0; j < kN; j += 4) e[j] = (e[j] + e[j + 1]) + (e[j + 2] + e[j + 3]);
            S[b] = kN == 8 ? e[0] + e[4] : e[0];
            W[b] = kN == 8 ? w[0] + w[kN / 8] : w[0];
        }
        sums.S += N == kBatch ? (S[0] + S[1 % N]) + (S[N / 2] + S[N - 1]) : S[0];
        sums.W += N == kBatch ? (W[0] + W[1 % N]) + (W[N / 2] + W[N - 1]) : W[0];
    };
    Pack<E> next[kBatch];
    const auto load = [&](int p0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            next[b] = load_pack(row + in.first(min(p0 + b * kThreads + int(threadIdx.x), end - 1)));
    };
    const auto taken = [&](int p0, Pack<E> (&v)[kBatch], int (&first)[kBatch]) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int p = p0 + b * kThreads + int(threadIdx.x);
            v[b] = next[b];
            if (p >= end) v[b] = no_pack<E>();
            first[b] = in.first(p);
        }
    };
    if (begin < end) load(begin);
    float span_most = -__builtin_inff();
    for (int batch = 0, p0 = begin; batch < batches; ++batch, p0 += kPacks) {
        Pack<E> v[kBatch];
        int first[kBatch];
        float most[kBatch];
        taken(p0, v, first);
        if (p0 + kPacks < end) load(p0 + kPacks);
        const float all = largest(v, most);
        add(v, all);
        if constexpr (TOP) {
            if (batches == 1) {  // the logits are here still
                share_bound<WAVES>(c, columns);
                c.take(v, most, first);
            } else {
                span_most = batch % span ? fmaxf(span_most, all) : all;
                spans[batch / span][threadIdx.x] = static_cast<uint16_t>(score_key(span_most) >> 16);
            }
        }
    }
    Pack<E> rest[1] = {no_pack<E>()};  // (fewer than 2 kN elements: the first threads')
    const int rest_at[1] = {in.rest(threadIdx.x)};
    float rest_most[1] = {-__builtin_inff()};
    if (last && in.has_rest()) {
        if (rest_at[0] < a.V) rest[0].e[0] = row[rest_at[0]];
        largest(rest, rest_most);
        add(rest, rest_most[0]);
    }
    if constexpr (TOP) {
        if (batches != 1) {
            share_bound<WAVES>(c, columns);
            // the spans with a logit that may be among the largest, once more
            const uint32_t from = score_key(c.from) >> 16;
            for (int t = 0; t * span < batches; ++t) {
                const uint32_t key = spans[t][threadIdx.x];
                const bool mine = key >= from && key > kKeyNegInf >> 16;
                if (!ballot(mine)) continue;
                for (int batch = t * span; batch < min(batches, (t + 1) * span); ++batch) {
                    Pack<E> v[kBatch];
                    int first[kBatch];
                    float most[kBatch];
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) next[b] = no_pack<E>();
                    if (mine) load(begin + batch * kPacks);
                    taken(begin + batch * kPacks, v, first);
                    largest(v, most);
                    c.take(v, most, first);
                }
            }
        }
        if (last && in.has_rest()) c.take(rest, rest_most, rest_at);
    }
    Sums<float> s{static_cast<float>(sums.S), static_cast<float>(sums.W), sums.m};
    join_lanes<kWave>(s, c.lane_most);
    if (lane == 0) wave_sums[wave][0] = s.m, wave_sums[wave][1] = s.S, wave_sums[wave][2] = s.W;
    uint64_t best = 0;
    if constexpr (TOP) {
        c.leave(left, &filled);
        if constexpr (WAVES > 1)
            __syncthreads();
        else
            wave_order();
        const int n = static_cast<int>(filled);
        if (static_cast<int>(threadIdx.x) < n) {
            const uint64_t mine = left[threadIdx.x];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += left[j] > mine;
            if (rank < a.top) sorted[rank] = mine;
        }
        if constexpr (WAVES > 1)
            __syncthreads();
        else
            wave_order();
        if (wave) return;
        best = lane < a.top ? sorted[lane] : 0;
    }
    if constexpr (WAVES > 1) {
        if constexpr (!TOP) __syncthreads();
        if (wave) return;
        const float* const mine = wave_sums[lane % WAVES];
        s = {mine[1], mine[2], mine[0]};
        join_lanes<WAVES>(s, s.m);
    }
    if (a.parts == 1) {
        write_row<E>(a, i, s, best);
    } else {
        if (lane == 0) a.part_sums[blockIdx.x] = make_float4(s.m, s.S, s.W, 0.0f);
        if (TOP && lane < a.top) a.part_lists[int64_t(blockIdx.x) * a.top + lane] = best;
    }
}

// The parts of a row joined, a wave a row.
template <typename E, bool TOP>
__global__ __launch_bounds__(kWave) void score_join(const Args a) {
    __shared__ uint64_t lists[TOP ? kMostParts * HSN_SCORE_MAX_TOP : 1];
    const int i = blockIdx.x, lane = lane_id();
    Sums<float> s;
    if (lane < a.parts) {
        const float4 v = a.part_sums[int64_t(i) * a.parts + lane];
        s = {v.y, v.z, v.x};
    }
    if constexpr (TOP) {
        const uint64_t* from = a.part_lists + int64_t(i) * a.parts * a.top;
        for (int j = lane; j < a.parts * a.top; j += kWave) lists[j] = from[j];
        wave_order();
    }
    join_lanes<kWave>(s, s.m);
    uint64_t best = 0;
    if constexpr (TOP) best = merge(lists, a.parts, a.top, a.top);
    write_row<E>(a, i, s, best);
}

// A workgroup a part of a row, the last rows first: what the forward read last is in the cache still (with
// stores past it, 8192 x 32000 bf16 both ways takes 271 us; 311 with ordinary stores).
template <typename E, int WAVES, bool STREAM>
__global__ __launch_bounds__(WAVES * kWave) void score_grad(const Args a) {
    constexpr int kThreads = WAVES * kWave, kN = Pack<E>::kN;
    const int block = gridDim.x - 1 - blockIdx.x, i = block / a.parts, part = block % a.parts;
    const E* row = static_cast<const E*>(a.logits) + i * a.row;
    E* to = static_cast<E*>(a.d_logits) + int64_t(i) * a.V;
    const float4 stats = a.stats[i];
    const float m = stats.x, r = stats.y, rest = stats.z, entropy = stats.w;
    const int64_t given = a.token(i);
    const bool skipped = given < 0 || given >= a.V || r == 0.0f;
    const int t = skipped ? -1 : static_cast<int>(given);
    const float g = a.g && !skipped ? a.g[i * a.g_stride] : 0.0f;
    const float h = a.h ? a.h[i * a.h_stride] : 0.0f;
    const float lift = entropy - rest;  // log p + H = x + lift
    const auto grad = [&](float l) {
        const float x = l - m;
        const float p = exp_of(x) * r;
        return -p * __builtin_fmaf(h, fmaxf(x, -200.0f) + lift, g);
    };
    const RowPacks<E> in(row, a.V);
    const int begin = part * a.part_packs;
    const int end = part + 1 == a.parts ? in.packs : min(in.packs, begin + a.part_packs);
    for (int p = begin + int(threadIdx.x); p < end; p += kBatch * kThreads) {
        Pack<E> v[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) v[b] = load_pack(row + in.first(min(p + b * kThreads, end - 1)));
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (p + b * kThreads >= end) break;
            const int first = in.first(p + b * kThreads);
            float d[kN];
#pragma unroll
            for (int j = 0; j < kN; ++j) d[j] = grad(v[b][j]);
            if (static_cast<uint32_t>(t - first) < kN) {
#pragma unroll
                for (int j = 0; j < kN; ++j) d[j] += first + j == t ? g : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kN; ++j) v[b].e[j] = from_f32<E>(d[j]);
            store_pack<STREAM>(to + first, v[b]);
        }
    }
    if (part + 1 == a.parts) {
        const int j = in.rest(threadIdx.x);
        if (j < a.V) to[j] = from_f32<E>(grad(to_f32(row[j])) + (j == t ? g : 0.0f));
    }
}

// ------------------------------------------------------------------------------------------
// Launches.
// ------------------------------------------------------------------------------------------

int size_of(int dtype) { return dtype == HSN_DTYPE_F32 ? 4 : 2; }

// Waves of a workgroup and parts of a row.
struct Plan {
    int waves, parts, part_packs;
};

Plan split(int waves, int64_t packs, int64_t parts) {
    Plan p;
    p.waves = waves;
    parts = std::max<int64_t>(1, std::min<int64_t>(parts, kMostParts));
    p.part_packs = static_cast<int>((packs + parts - 1) / parts);
    p.parts = static_cast<int>((packs + p.part_packs - 1) / p.part_packs);
    return p;
}

// The forward's, with packs a row, from sweeps over n rows of V bf16 logits with five alternatives (us):
// - a batch of a wave or two: a wave a row.
// - a batch of four waves: those, whatever n is (64 x 8192: 7.7, by 16 waves 8.3).
// - a batch of 16 waves, of no more than 256 rows: those, without the second launch (1 x 32000 with 20
//   alternatives: 8.0, by parts 12.5); and so all rows where n is above 128, as their waves fill the GPU (200 x
//   262144: 31, four waves in four parts 35).
// - up to 128 longer rows: parts of one batch of four waves, as far as 1024 workgroups go (1 x 131071: 11.0
//   in 16 parts, 15.8 by 16 waves; 64 x 131071: 13.5 in 16 parts, 15 in 4, 16.7 by 16 waves).
// - more rows: four waves each, in parts of at least eight batches while there are fewer than 1024 rows (300 x
//   262144: 45 in 3 parts, 53 in one; but 301 x 50021 in fp32 18 in one and 21 in three).
Plan plan_forward(int n, int V, int dtype) {
    const int64_t packs = std::max<int64_t>(1, V / (16 / size_of(dtype)));
    const int64_t batch = kBatch * 4 * kWave, fill = 1024 / std::max(n, 1);
    if (packs <= batch / 2) return split(1, packs, 1);
    if (packs <= batch) return split(4, packs, 1);
    if (n > 256) return split(4, packs, std::min<int64_t>(fill, packs / (8 * batch)));
    if (packs <= 4 * batch || n > 128) return split(16, packs, 1);
    return split(4, packs, std::min<int64_t>(fill, (packs + batch - 1) / batch));
}

// The backward's, whose parts need no second launch: some 2048 workgroups, a batch at least (1 x 262144 bf16: 4.5 us,
// by one workgroup 32; 301 x 50021: 11, one workgroup a row 15), of four waves, or one where a row is short (16384 x
// 1000: 12 us, by four 18).
Plan plan_backward(int n, int V, int dtype) {
    const int64_t packs = std::max<int64_t>(1, V / (16 / size_of(dtype)));
    const int waves = packs <= 2 * kBatch * kWave ? 1 : 4;
    return split(waves, packs, std::min<int64_t>((2047 + n) / std::max(n, 1), packs / (kBatch * waves * kWave)));
}

int64_t layout(Args& a, char* at, int n, int top) {
    if (a.parts == 1) return 0;
    a.part_sums = reinterpret_cast<float4*>(at);
    const int64_t sums = 16 * int64_t(n) * a.parts;
    a.part_lists = reinterpret_cast<uint64_t*>(at + sums);
    return sums + 8 * int64_t(n) * a.parts * top;
}

template <typename E, bool TOP>
void launch_forward(const Args& a, const Plan& p, int n, hipStream_t st) {
    (p.waves == 1   ? score_rows<E, 1, TOP>
     : p.waves == 4 ? score_rows<E, 4, TOP>
                    : score_rows<E, 16, TOP>)<<<n * p.parts, p.waves * kWave, 0, st>>>(a);
    HSN_HIP(hipGetLastError());
    if (p.parts > 1) score_join<E, TOP><<<n, kWave, 0, st>>>(a);
}

template <typename E>
void launch_backward(const Args& a, const Plan& p, int n, hipStream_t st) {
    const bool stream = int64_t(n) * a.V * sizeof(E) > kStream;
    (p.waves == 1 ? (stream ? score_grad<E, 1, true> : score_grad<E, 1, false>)
                  : (stream ? score_grad<E, 4, true> : score_grad<E, 4, false>))<<<n * p.parts, p.waves * kWave, 0,
                                                                                    st>>>(a);
}

void check(int n, int V, int dtype, int top) {
    HSN_REQUIRE(dtype == HSN_DTYPE_F32 || dtype == HSN_DTYPE_F16 || dtype == HSN_DTYPE_BF16,
                HSN_ERR_UNSUPPORTED_DTYPE, "logits must be F32, F16 or BF16");
    HSN_REQUIRE(n >= 0 && V >= 1, HSN_ERR_INVALID_ARGUMENT, "n >= 0 and V >= 1");
    HSN_REQUIRE(top >= 0 && top <= HSN_SCORE_MAX_TOP, HSN_ERR_INVALID_ARGUMENT, "top in [0, 32]");
    HSN_REQUIRE(V <= HSN_SCORE_MAX_TOKENS, HSN_ERR_SIZE_OVERFLOW, "at most 2^24 tokens");
    // a grid's dimension holds fewer than 2^32 threads, four waves a row
    HSN_REQUIRE(n < 1 << 24, HSN_ERR_SIZE_OVERFLOW, "fewer than 2^24 rows");
    HSN_REQUIRE(int64_t(n) * V < int64_t(1) << 40, HSN_ERR_SIZE_OVERFLOW, "fewer than 2^40 logits");
}

void check_rows(const void* logits, int dtype, const void* tokens, int token_bytes) {
    HSN_REQUIRE(logits && tokens, HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size_of(dtype) == 0, HSN_ERR_INVALID_ARGUMENT,
                "logits must be aligned to their type");
    HSN_REQUIRE(token_bytes == 8 || token_bytes == 4, HSN_ERR_INVALID_ARGUMENT, "token_bytes is 8 or 4");
}

}  // namespace
}  // namespace score
}  // namespace hsn

using namespace hsn;
using namespace hsn::score;

extern "C" int hsn_score_workspace(int n, int V, int dtype, int top, int64_t* bytes) {
    HSN_ABI_BEGIN
    check(n, V, dtype, top);
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    Args a{};
    a.parts = plan_forward(n, V, dtype).parts;
    *bytes = layout(a, nullptr, n, top);
    HSN_ABI_END
}

extern "C" int hsn_score_forward(const void* logits, int64_t row, int dtype, const void* tokens,
                                 int64_t token_stride, int token_bytes, float* logprob, float* entropy,
                                 int64_t* top_tokens, float* top_logprobs, float* stats, int n, int V,
                                 int top, void* workspace, int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    check(n, V, dtype, top);
    if (n == 0) return HSN_OK;
    check_rows(logits, dtype, tokens, token_bytes);
    HSN_REQUIRE(logprob && entropy && (top == 0 || (top_tokens && top_logprobs)), HSN_ERR_INVALID_ARGUMENT,
                "a required pointer is NULL");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                "stats must be aligned to 16 bytes");
    const Plan p = plan_forward(n, V, dtype);
    Args a{};
    a.logits = logits, a.row = row, a.tokens = tokens, a.token_stride = token_stride;
    a.wide = token_bytes == 8;
    a.logprob = logprob, a.entropy = entropy, a.top_tokens = top_tokens, a.top_logprobs = top_logprobs;
    a.stats = reinterpret_cast<float4*>(stats);
    a.V = V, a.top = top, a.parts = p.parts, a.part_packs = p.part_packs;
    const int64_t bytes = layout(a, static_cast<char*>(workspace), n, top);
    HSN_REQUIRE(!bytes || (workspace && workspace_bytes >= bytes), HSN_ERR_INVALID_ARGUMENT,
                "the workspace is too small");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                "the workspace must be aligned to 16 bytes");
    hipStream_t st = as_stream(stream);
    const auto with = [&](auto e) {
        using E = decltype(e);
        if (top)
            launch_forward<E, true>(a, p, n, st);
        else
            launch_forward<E, false>(a, p, n, st);
    };
    if (dtype == HSN_DTYPE_F32)
        with(float{});
    else if (dtype == HSN_DTYPE_F16)
        with(_Float16{});
    else
        with(bf16_t{});
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}

extern "C" int hsn_score_backward(const void* logits, int64_t row, int dtype, const void* tokens,
                                  int64_t token_stride, int token_bytes, const float* stats,
                                  const float* d_logprob, int64_t g_stride, const float* d_entropy,
                                  int64_t h_stride, void* d_logits, int n, int V, void* stream) {
    HSN_ABI_BEGIN
    check(n, V, dtype, 0);
    if (n == 0) return HSN_OK;
    check_rows(logits, dtype, tokens, token_bytes);
    HSN_REQUIRE(stats && d_logits, HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                "stats must be aligned to 16 bytes");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(d_logits) % size_of(dtype) == 0, HSN_ERR_INVALID_ARGUMENT,
                "d_logits must be aligned to their type");
    const Plan p = plan_backward(n, V, dtype);
    Args a{};
    a.logits = logits, a.row = row, a.tokens = tokens, a.token_stride = token_stride;
    a.wide = token_bytes == 8;
    a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
    a.V = V, a.parts = p.parts, a.part_packs = p.part_packs;
    a.g = d_logprob, a.g_stride = g_stride, a.h = d_entropy, a.h_stride = h_stride;
    a.d_logits = d_logits;
    hipStream_t st = as_stream(stream);
    if (dtype == HSN_DTYPE_F32)
        launch_backward<float>(a, p, n, st);
    else if (dtype == HSN_DTYPE_F16)
        launch_backward<_Float16>(a, p, n, st);
    else
        launch_backward<bf16_t>(a, p, n, st);
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
