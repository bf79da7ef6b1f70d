// The gated linear recurrence's kernels over tiles of positions (include/hsn_scan.h).
//
// A position is a map of the state, h -> a h + x with a = sigmoid(-g), x = sigmoid(g) c; maps join
// (first (A1, H1), then (A2, H2)) to (A1 A2, A2 H1 + H2), so a span of positions is one pair, and
// the time axis splits anywhere. A reset makes the map constant; it is marked by a negative A, so
// that joins select the later value instead of multiplying the earlier one by zero (0 * inf). A NaN A
// counts as constant too: a NaN gate makes the span's value NaN whatever comes in, unless, going backward,
// a reset between the gate and the span's start drops it.
//
// Tile: a workgroup of 512 threads takes 64 channels of one row (128 bytes of 16-bit storage) and
// kTile positions. A thread has V neighbouring channels (2 where the layout allows, else 1) and a
// segment of S positions, kept in registers from the one load to the one store: it folds its segment,
// the segments of a wave join by lane shuffles, the waves by LDS, and the thread walks its segment
// again from the state before it. Wider packs halve the loads but double the segments of a wave and
// with them the joins, and the kernel is bound by the instructions it issues before it is bound by
// HBM: with V = 4 a walk over 8 x 4096 x 2048 in bf16 takes 130 us forward and 255 us backward, with
// V = 2 98 and 187 us.
//
// Time axis: a workgroup walks its 64 channels' tiles one after the other, the next tile's loads in
// flight, where rows and channels alone fill the GPU and the tiles are few. Else every tile is a
// workgroup of its own (kSplit): it publishes its pair and takes the pairs before it from device
// memory. Tiles are numbered by a ticket, so that whatever a workgroup waits for belongs to one that
// already runs and publishes without waiting for a later one: every wait ends. Pairs are folded in
// groups of 32 tiles in a fixed order, so the bits do not depend on who arrives first. Split, the
// same 8 x 4096 x 2048 take 104 and 184 us (3.9 and 3.6 TB/s of the 3 and 5 elements that have to
// move; a copy reaches 5.3), and one row of 32769 x 1024 64 us, which one walk a strip takes 1.0 ms
// for; at 32 x 256 x 512 in fp32 the walk's 13.5 and 19.5 us are less than the split's and the clearing of its
// words. What is left between that and a copy is a workgroup's own latencies: its ticket, its loads and
// its wait follow one another, and the registers allow two workgroups a compute unit to overlap them.
#pragma once

#include <type_traits>

#include "../../include/hsn_scan.h"
#include "common.cuh"
#include "dpp.cuh"

namespace hsn {
namespace scan {

constexpr int kSpan = HSN_SCAN_SPAN;
constexpr int kThreads = 512, kWaves = kThreads / kWave;
constexpr int kChannels = 64;  // of a tile
constexpr int kGroup = 32;     // tiles whose pairs are folded one by one

struct Args {
    const void *y, *gate, *d_h;
    int64_t y_row, y_pos, gate_row, gate_pos, d_row, d_pos;
    const uint8_t* reset;
    const float *h0, *d_h_T;
    float *h_T, *marks, *d_h0;
    void *h, *d_y, *d_gate;
    int T, D, candidate;
    int strips_a_row, strips, tiles;
    bool reset_words;  // every fourth flag of a row is aligned to four bytes
    uint64_t* box;  // kSplit: the ticket's 64 words, [tiles][strips][64] pairs, [groups][strips][64]
};

// a = sigmoid(-g) (the share of the old state kept) and b = sigmoid(g) (the share written): 1/(1+e) and
// e/(1+e) with e = exp(-g), neither a difference from 1 (1 - b would leave nothing of a small a). The
// exponent's rounding and that of log2(e) leave e right to 1.25 |g| 2^-24 of itself, so a small share is
// right to that and a few ulps (7.5e-7 at |g| = 10, 4.5e-6 at 60); the product in two parts takes 3% more
// time (8 x 4096 x 2048 in bf16, forward and backward: 288 us, not 280). e stops at 2^126, so that a is 1 and b 2^-126 for every g below
// -87 and not inf * 0; the minimum keeps a NaN.
__device__ __forceinline__ void gates(float g, float& a, float& b) {
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(-kLog2e * g, 126.0f));
    b = __builtin_amdgcn_rcpf(1.0f + e);
    a = e * b;
}

// tanh(y) = 1 - 2 / (1 + exp(2y)), right to 2.7e-7 of 1, and for small |y|, where that is a
// difference of equals, the series y - y^3/3 + 2 y^5/15 (fp32 storage: below 1/8 the next term,
// 17 y^7 / 315, is at most 2.1e-7 of y) or y alone (16-bit storage: below 1/128 it is off by at most
// 1.6e-7 of 1, as the other form is, and 2e-5 of itself, a 24th of fp16's rounding of y and a 190th of
// bf16's). The fp32 states of 16-bit inputs take the latter too; the series takes 4% more time there
// (8 x 4096 x 2048 in bf16, forward and backward: 292 us, not 280).
template <typename E>
__device__ __forceinline__ float tanh_of(float y) {
    const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * y);
    const float t = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
    if constexpr (sizeof(E) == 2) return __builtin_fabsf(y) < 0.0078125f ? y : t;
    const float y2 = y * y;
    const float s = __builtin_fmaf(y2 * y, __builtin_fmaf(y2, 2.0f / 15.0f, -1.0f / 3.0f), y);
    return __builtin_fabsf(y) < 0.125f ? s : t;
}

// The share of a linear candidate: 0 where gates() stops at 2^-126, which times the largest values is not
// small (a mask that puts the type's lowest value into gate and candidate); a NaN stays. A tanh is at most
// 1 and takes the share as it is.
__device__ __forceinline__ float linear_share(float b) { return b <= 0x1.1p-126f ? 0.0f : b; }

struct Pair {
    float A, H;
};

// A sign, or a NaN of either.
__device__ __forceinline__ bool constant(float A) { return __float_as_uint(A) > 0x7f800000u; }
__device__ __forceinline__ float apply(Pair m, float h) {
    return constant(m.A) ? m.H : __builtin_fmaf(m.A, h, m.H);
}
// `first`, then `then`.
__device__ __forceinline__ Pair join(Pair first, Pair then) {
    return constant(then.A) ? then
                            : Pair{first.A * then.A, __builtin_fmaf(then.A, first.H, then.H)};
}

template <typename E, int V>
struct alignas(sizeof(E) * V) Pack {
    E e[V];
};

template <typename E, int V>
__device__ __forceinline__ Pack<E, V> filled(float v) {
    Pack<E, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.e[i] = from_f32<E>(v);
    return p;
}

// The segment's values of one tensor: S positions from t0 on, `fill` after the last.
template <typename E, int V, int S>
__device__ __forceinline__ void load_segment(Pack<E, V> (&to)[S], const E* row, int64_t pos, int t0,
                                             int T, bool whole, float fill) {
    using P = Pack<E, V>;
    const E* at = row + t0 * pos;
    if (whole) {
#pragma unroll
        for (int i = 0; i < S; ++i, at += pos) to[i] = *reinterpret_cast<const P*>(at);
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i, at += pos) {
            to[i] = filled<E, V>(fill);
            if (t0 + i < T) to[i] = *reinterpret_cast<const P*>(at);
        }
    }
}

template <typename E, int V, int S>
__device__ __forceinline__ void store_segment(const Pack<E, V> (&from)[S], E* row, int64_t pos,
                                              int t0, int T) {
    using P = Pack<E, V>;
    E* at = row + t0 * pos;
    if (t0 + S <= T) {
#pragma unroll
        for (int i = 0; i < S; ++i, at += pos) *reinterpret_cast<P*>(at) = from[i];
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i, at += pos)
            if (t0 + i < T) *reinterpret_cast<P*>(at) = from[i];
    }
}

// Bit i: a reset before position t0 + i.
template <int S>
__device__ __forceinline__ uint32_t load_resets(const uint8_t* row, int t0, int T, bool words) {
    uint32_t bits = 0;
    if (!row) return 0;
    if (words) {  // four flags a load: byte k (0 or 1) goes to bit 24 + k
#pragma unroll
        for (int i = 0; i < S; i += 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(row + t0 + i);
            bits |= ((w & 0x01010101u) * 0x01020408u >> 24 & 15u) << i;
        }
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (t0 + i < T) bits |= uint32_t(row[t0 + i] != 0) << i;
    }
    return bits;
}

// --------------------------------------------------------------------------------------------
// The exchange of pairs between a row's tiles.
// --------------------------------------------------------------------------------------------

// A pair as one word that is never 0 (A's bits are at most 0x7f800000 or negative, plus one; a NaN A as -0,
// which says the same).
__device__ __forceinline__ uint64_t pair_word(Pair m) {
    const uint32_t a = m.A != m.A ? 0x80000000u : __float_as_uint(m.A);
    return uint64_t(a + 1) << 32 | __float_as_uint(m.H);
}
__device__ __forceinline__ Pair word_pair(uint64_t w) {
    return {__uint_as_float(uint32_t(w >> 32) - 1), __uint_as_float(uint32_t(w))};
}

// One relaxed agent-scope word: it is complete by itself, so the reader needs no fence.
__device__ __forceinline__ void publish(uint64_t* at, uint64_t w) {
    __hip_atomic_store(at, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Waits for N times a wave's 64 words, N loads in flight. Each belongs to a workgroup with a lower
// ticket; the bound (seconds) is there so that no fault elsewhere can hang the grid, and what it
// gives up on becomes NaN. An absent item (NULL) is the identity.
template <int N>
__device__ __forceinline__ void await(const uint64_t* const (&at)[N], Pair (&pair)[N]) {
    for (int spin = 0; spin < (1 << 21); ++spin) {
        uint64_t w[N];
        bool missing = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
            w[i] = at[i] ? __hip_atomic_load(at[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                         : pair_word({1.0f, 0.0f});
#pragma unroll
        for (int i = 0; i < N; ++i) {
            missing |= w[i] == 0;
            pair[i] = word_pair(w[i]);
        }
        if (ballot(missing) == 0) return;
        __builtin_amdgcn_s_sleep(1);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) pair[i] = {-1.0f, __int_as_float(0x7fc00000)};
}

struct ExchangeLds {
    Pair item[kGroup][kChannels];
};

// The state before tile k of the strip (k counts in the order of processing), for each channel of
// the first wave's lanes, from this tile's pair and `start`, the state before tile 0.
__device__ __forceinline__ float exchange(const Args& p, ExchangeLds& lds, int k, int strip,
                                          Pair total, float start) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint64_t* pairs = p.box + 64 + int64_t(strip) * kChannels + lane;
    const int64_t line = int64_t(p.strips) * kChannels;
    uint64_t* prefix = pairs + p.tiles * line;
    if (wave == 0) publish(pairs + k * line, pair_word(total));
    // item 0: the state before the group; item i: the pair of the group's tile i - 1
    const int group = k / kGroup, before = k % kGroup;
    constexpr int kItems = kGroup / kWaves;
    const uint64_t* at[kItems];
    Pair item[kItems];
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
        const int i = wave + j * kWaves;
        at[j] = nullptr;
        if (i == 0 && group) at[j] = prefix + (group - 1) * line;
        if (i > 0 && i <= before) at[j] = pairs + (group * kGroup + i - 1) * line;
    }
    await<kItems>(at, item);
#pragma unroll
    for (int j = 0; j < kItems; ++j) lds.item[wave + j * kWaves][lane] = item[j];
    __syncthreads();
    float h = start;
    if (wave == 0) {
        if (group) h = lds.item[0][lane].H;
        for (int i = 1; i <= before; ++i) h = apply(lds.item[i][lane], h);
        if (before == kGroup - 1 && k + 1 < p.tiles)
            publish(prefix + group * line, pair_word({-1.0f, apply(total, h)}));
    }
    return h;
}
static_assert(kGroup % kWaves == 0, "a group's items, its prefix and the pairs before, by waves");

// --------------------------------------------------------------------------------------------
// Forward.
// --------------------------------------------------------------------------------------------

template <typename E, int V, int S>
struct Tile {
    static constexpr int kLanes = kChannels / V;           // threads side by side
    static constexpr int kSegs = kThreads / kLanes;        // segments of S positions
    static constexpr int kTile = kSegs * S;
    static_assert(kSpan % S == 0 && kTile % kSpan == 0, "marks lie between segments");
};

// The thread's inclusive join over the wave's segments up to its own, from the first on (UP) or
// from the last on. RESETS: whether a segment of the wave may be constant.
template <int LANES, bool UP, bool RESETS, int V>
__device__ __forceinline__ void wave_join(float (&A)[V], float (&H)[V]) {
    const int lane = lane_id();
#pragma unroll
    for (int d = LANES; d < kWave; d *= 2) {
        const bool has = UP ? lane >= d : lane < kWave - d;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Pair o = UP ? Pair{__shfl_up(A[v], d, kWave), __shfl_up(H[v], d, kWave)}
                              : Pair{__shfl_down(A[v], d, kWave), __shfl_down(H[v], d, kWave)};
            const Pair m = RESETS ? join(o, {A[v], H[v]})
                                  : Pair{o.A * A[v], __builtin_fmaf(A[v], o.H, H[v])};
            A[v] = has ? m.A : A[v];
            H[v] = has ? m.H : H[v];
        }
    }
}

template <typename E, int V, int S, bool kSplit, bool kTanh>
__global__ __launch_bounds__(kThreads) void forward_tiles(Args p) {
    using G = Tile<E, V, S>;
    using P = Pack<E, V>;
    __shared__ Pair wave_pair[2][kWaves][kChannels];
    __shared__ float carry[2][kChannels];
    __shared__ ExchangeLds lds;
    __shared__ uint32_t ticket;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int cl = tid % G::kLanes, seg = tid / G::kLanes;
    int strip = blockIdx.x, tile = 0, end = p.tiles;
    if constexpr (kSplit) {
        if (tid == 0) ticket = atomicAdd(reinterpret_cast<uint32_t*>(p.box), 1u);
        __syncthreads();
        strip = ticket % p.strips, tile = ticket / p.strips, end = tile + 1;
    }
    const int64_t r = strip / p.strips_a_row;
    const int ch0 = (strip % p.strips_a_row) * kChannels, ch = ch0 + cl * V;
    const bool on = ch < p.D;
    // lanes past the last channel load the last ones and store nothing
    const int from = on ? ch : p.D - V;
    const E* y = static_cast<const E*>(p.y) + r * p.y_row + from;
    const E* g = static_cast<const E*>(p.gate) + r * p.gate_row + from;
    const uint8_t* reset = p.reset ? p.reset + r * p.T : nullptr;
    E* out = static_cast<E*>(p.h) + r * p.T * p.D + ch;
    const int64_t spans = (p.T + kSpan - 1) / kSpan;
    float start = 0.0f;
    if (tid < kChannels && ch0 + tid < p.D && p.h0) start = p.h0[r * p.D + ch0 + tid];
    if (tid < kChannels) carry[0][tid] = start;

    P ry[S], rg[S];
    uint32_t resets;
    // after the last position: a gate of -inf, which keeps the state
    auto load = [&](int at) {
        const int t0 = at * G::kTile + seg * S;
        const bool whole = (at + 1) * G::kTile <= p.T;
        load_segment<E, V, S>(ry, y, p.y_pos, t0, p.T, whole, 0.0f);
        load_segment<E, V, S>(rg, g, p.gate_pos, t0, p.T, whole, -__builtin_inff());
        resets = load_resets<S>(reset, t0, p.T, whole && p.reset_words);
    };
    load(tile);
    for (int buf = 0; tile < end; ++tile, buf ^= 1) {
        const int t0 = tile * G::kTile + seg * S;
        float a[S][V], x[S][V], A[V], H[V];
        const uint32_t drop = resets;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gates(to_f32(rg[i].e[v]), a[i][v], x[i][v]);
            }
        // the candidates' instructions stay behind the gates' (1 x 32769 x 1024 in bf16: 64 us, mixed 66)
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kTanh) {
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) x[i][v] *= tanh_of<E>(to_f32(ry[i].e[v]));
        } else {
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) x[i][v] = linear_share(x[i][v]) * to_f32(ry[i].e[v]);
        }
        // most waves have no reset in their segments: they skip what resets cost at every position
        const bool any = ballot(drop != 0) != 0;
        auto fold = [&](auto resets_too) {
            constexpr bool R = decltype(resets_too)::value;
#pragma unroll
            for (int v = 0; v < V; ++v) A[v] = 1.0f, H[v] = 0.0f;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                if (R && (drop >> i & 1))
#pragma unroll
                    for (int v = 0; v < V; ++v) A[v] = -1.0f, H[v] = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    A[v] *= a[i][v];
                    H[v] = __builtin_fmaf(a[i][v], H[v], x[i][v]);
                }
            }
            wave_join<G::kLanes, true, R, V>(A, H);
        };
        if (any)
            fold(std::true_type{});
        else
            fold(std::false_type{});
        if (!kSplit && tile + 1 < end) load(tile + 1);
        if (lane >= kWave - G::kLanes)
#pragma unroll
            for (int v = 0; v < V; ++v) wave_pair[buf][wave][cl * V + v] = {A[v], H[v]};
        __syncthreads();
        Pair total{1.0f, 0.0f};
        if (tid < kChannels)
            for (int w = 0; w < kWaves; ++w) total = join(total, wave_pair[buf][w][tid]);
        float before = 0.0f;
        if constexpr (kSplit) before = exchange(p, lds, tile, strip, total, start);
        if (tid < kChannels) {
            if constexpr (kSplit)
                carry[0][tid] = before;
            else
                before = carry[buf][tid];
            const float after = apply(total, before);
            carry[buf ^ 1][tid] = after;
            if (tile == p.tiles - 1 && ch0 + tid < p.D) p.h_T[r * p.D + ch0 + tid] = after;
        }
        if constexpr (kSplit) __syncthreads();
        // the state before the thread's segment: the waves before, then the lanes before
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = carry[buf][cl * V + v];
            for (int w = 0; w < wave; ++w) h[v] = apply(wave_pair[buf][w][cl * V + v], h[v]);
            if constexpr (G::kLanes < kWave) {
                const Pair m{__shfl_up(A[v], G::kLanes, kWave), __shfl_up(H[v], G::kLanes, kWave)};
                h[v] = lane >= G::kLanes ? apply(m, h[v]) : h[v];
            }
        }
        if (p.marks && on && t0 < p.T && t0 % kSpan == 0)
#pragma unroll
            for (int v = 0; v < V; ++v) p.marks[(r * spans + t0 / kSpan) * p.D + ch + v] = h[v];
        P o[S];
        auto walk = [&](auto resets_too) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                if (decltype(resets_too)::value && (drop >> i & 1))
#pragma unroll
                    for (int v = 0; v < V; ++v) h[v] = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[v] = __builtin_fmaf(a[i][v], h[v], x[i][v]);
                    o[i].e[v] = from_f32<E>(h[v]);
                }
            }
        };
        if (any)
            walk(std::true_type{});
        else
            walk(std::false_type{});
        store_segment<E, V, S>(o, out, p.D, t0, on ? p.T : 0);
    }
}

// --------------------------------------------------------------------------------------------
// Backward: from the last tile to the first. mu, the cotangent that a position hands to the one
// before it, is a (d_h + mu of the one after): the same pairs from the other end, with x = a d_h.
// A tile makes its states again from the mark before it; d_gate is l q with q = a b (c - m h[t-1]).
// --------------------------------------------------------------------------------------------

template <typename E, int V, int S, bool kSplit, bool kTanh>
__global__ __launch_bounds__(kThreads) void backward_tiles(Args p) {
    using G = Tile<E, V, S>;
    using P = Pack<E, V>;
    __shared__ Pair wave_pair[2][kWaves][kChannels];
    __shared__ float wave_mu[2][kWaves][kChannels];
    __shared__ float carry[2][kChannels], mark[2][kChannels];
    __shared__ ExchangeLds lds;
    __shared__ uint32_t ticket;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int cl = tid % G::kLanes, seg = tid / G::kLanes;
    int strip = blockIdx.x, turn = 0, end = p.tiles;  // turn 0 is the last tile
    if constexpr (kSplit) {
        if (tid == 0) ticket = atomicAdd(reinterpret_cast<uint32_t*>(p.box), 1u);
        __syncthreads();
        strip = ticket % p.strips, turn = ticket / p.strips, end = turn + 1;
    }
    const int64_t r = strip / p.strips_a_row;
    const int ch0 = (strip % p.strips_a_row) * kChannels, ch = ch0 + cl * V;
    const bool on = ch < p.D, owner = tid < kChannels && ch0 + tid < p.D;
    const int from = on ? ch : p.D - V;
    const E* y = static_cast<const E*>(p.y) + r * p.y_row + from;
    const E* g = static_cast<const E*>(p.gate) + r * p.gate_row + from;
    const E* d = static_cast<const E*>(p.d_h) + r * p.d_row + from;
    const uint8_t* reset = p.reset ? p.reset + r * p.T : nullptr;
    E* dy = static_cast<E*>(p.d_y) + r * p.T * p.D + ch;
    E* dg = static_cast<E*>(p.d_gate) + r * p.T * p.D + ch;
    const int64_t spans = (p.T + kSpan - 1) / kSpan;
    float start = 0.0f;
    if (owner && p.d_h_T) start = p.d_h_T[r * p.D + ch0 + tid];
    if (tid < kChannels) carry[0][tid] = start;

    P ry[S], rg[S], rd[S];
    uint32_t resets;
    float next_mark = 0.0f;
    if (!p.d_h)
#pragma unroll
        for (int i = 0; i < S; ++i) rd[i] = P{};
    auto load = [&](int at) {
        const int t0 = at * G::kTile + seg * S;
        const bool whole = (at + 1) * G::kTile <= p.T;
        load_segment<E, V, S>(ry, y, p.y_pos, t0, p.T, whole, 0.0f);
        load_segment<E, V, S>(rg, g, p.gate_pos, t0, p.T, whole, -__builtin_inff());
        if (p.d_h) load_segment<E, V, S>(rd, d, p.d_pos, t0, p.T, whole, 0.0f);
        resets = load_resets<S>(reset, t0, p.T, whole && p.reset_words);
        if (owner) next_mark = p.marks[(r * spans + at * (G::kTile / kSpan)) * p.D + ch0 + tid];
    };
    load(p.tiles - 1 - turn);
    for (int buf = 0; turn < end; ++turn, buf ^= 1) {
        const int tile = p.tiles - 1 - turn, t0 = tile * G::kTile + seg * S;
        float a[S][V], b[S][V], c[S][V], A[V], H[V], B[V], M[V];
        P rl[S];
        const uint32_t drop = resets;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            rl[i] = rd[i];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gates(to_f32(rg[i].e[v]), a[i][v], b[i][v]);
                c[i][v] = to_f32(ry[i].e[v]);
                if constexpr (kTanh)
                    c[i][v] = tanh_of<E>(c[i][v]);
                else
                    b[i][v] = linear_share(b[i][v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.0f, H[v] = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (drop >> i & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) A[v] = -1.0f, H[v] = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A[v] *= a[i][v];
                H[v] = __builtin_fmaf(a[i][v], H[v], b[i][v] * c[i][v]);
            }
        }
        if (tid < kChannels) mark[buf][tid] = next_mark;
#pragma unroll
        for (int v = 0; v < V; ++v) B[v] = A[v], M[v] = 0.0f;
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
#pragma unroll
            for (int v = 0; v < V; ++v) M[v] = a[i][v] * (to_f32(rl[i].e[v]) + M[v]);
            if (drop >> i & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) M[v] = 0.0f;
        }
        if (!kSplit && turn + 1 < end) load(tile - 1);
        if (ballot(drop != 0)) {
            wave_join<G::kLanes, true, true, V>(A, H);
            wave_join<G::kLanes, false, true, V>(B, M);
        } else {
            wave_join<G::kLanes, true, false, V>(A, H);
            wave_join<G::kLanes, false, false, V>(B, M);
        }
        if (lane >= kWave - G::kLanes)
#pragma unroll
            for (int v = 0; v < V; ++v) wave_pair[buf][wave][cl * V + v] = {A[v], H[v]};
        if (lane < G::kLanes)
#pragma unroll
            for (int v = 0; v < V; ++v) wave_mu[buf][wave][cl * V + v] = M[v];
        __syncthreads();
        Pair total{1.0f, 0.0f};
        if (tid < kChannels)
            for (int w = kWaves - 1; w >= 0; --w)
                total = join(total, {wave_pair[buf][w][tid].A, wave_mu[buf][w][tid]});
        float after = 0.0f;  // in time
        if constexpr (kSplit) after = exchange(p, lds, turn, strip, total, start);
        if (tid < kChannels) {
            if constexpr (kSplit)
                carry[0][tid] = after;
            else
                after = carry[buf][tid];
            const float before = apply(total, after);
            carry[buf ^ 1][tid] = before;
            if (tile == 0 && owner) p.d_h0[r * p.D + ch0 + tid] = before;
        }
        if constexpr (kSplit) __syncthreads();
        // q over c, and b c'(y) over b, on the way through the states
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = mark[buf][cl * V + v];
            for (int w = 0; w < wave; ++w) h[v] = apply(wave_pair[buf][w][cl * V + v], h[v]);
            if constexpr (G::kLanes < kWave) {
                const Pair m{__shfl_up(A[v], G::kLanes, kWave), __shfl_up(H[v], G::kLanes, kWave)};
                h[v] = lane >= G::kLanes ? apply(m, h[v]) : h[v];
            }
        }
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (drop >> i & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float cand = c[i][v], share = b[i][v];
                c[i][v] = a[i][v] * share * (cand - h[v]);
                h[v] = __builtin_fmaf(a[i][v], h[v], share * cand);
                if constexpr (kTanh) b[i][v] = share * __builtin_fmaf(-cand, cand, 1.0f);  // c' = 1 - c^2
            }
        }
        float mu[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            mu[v] = carry[buf][cl * V + v];
            for (int w = kWaves - 1; w > wave; --w)
                mu[v] = apply({wave_pair[buf][w][cl * V + v].A, wave_mu[buf][w][cl * V + v]}, mu[v]);
            if constexpr (G::kLanes < kWave) {
                const Pair m{__shfl_down(B[v], G::kLanes, kWave),
                             __shfl_down(M[v], G::kLanes, kWave)};
                mu[v] = lane < kWave - G::kLanes ? apply(m, mu[v]) : mu[v];
            }
        }
        P oy[S], og[S];
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float l = to_f32(rl[i].e[v]) + mu[v];
                oy[i].e[v] = from_f32<E>(b[i][v] * l);
                og[i].e[v] = from_f32<E>(c[i][v] * l);
                mu[v] = a[i][v] * l;
            }
            if (drop >> i & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) mu[v] = 0.0f;
        }
        store_segment<E, V, S>(oy, dy, p.D, t0, on ? p.T : 0);
        store_segment<E, V, S>(og, dg, p.D, t0, on ? p.T : 0);
    }
}

// vec: the elements of a load, a divisor of the row length, the strides and the addresses.
template <typename E>
void launch_forward(const Args& p, int vec, bool split, hipStream_t st);
template <typename E>
void launch_backward(const Args& p, int vec, bool split, hipStream_t st);

// Elements of a thread's segments. Forward in fp32, 16: more workgroups fit a compute unit and the
// loads overlap better (8 x 8192 x 1024 split: 165 us, with 32 184). In 16 bits the halves' joins
// cost more than that gives (8 x 4096 x 2048 split: 100 us with 32, 119 with 16). The backward has
// three values an element to keep and no room for 32.
template <typename E>
constexpr int kForwardPer = sizeof(E) == 4 ? 16 : 32;
constexpr int kBackwardPer = 16;

// Positions of a tile.
inline int forward_tile(int element_size) {
    return kThreads / kChannels * (element_size == 4 ? kForwardPer<float> : kForwardPer<bf16_t>);
}
inline int backward_tile() { return kThreads / kChannels * kBackwardPer; }

#ifdef HSN_SCAN_INSTANTIATE
template <typename E, int V, bool kTanh>
void launch_forward_as(const Args& p, bool split, hipStream_t st) {
    if (split)
        forward_tiles<E, V, kForwardPer<E> / V, true, kTanh><<<p.strips * p.tiles, kThreads, 0, st>>>(p);
    else
        forward_tiles<E, V, kForwardPer<E> / V, false, kTanh><<<p.strips, kThreads, 0, st>>>(p);
}
template <typename E, int V, bool kTanh>
void launch_backward_as(const Args& p, bool split, hipStream_t st) {
    if (split)
        backward_tiles<E, V, kBackwardPer / V, true, kTanh><<<p.strips * p.tiles, kThreads, 0, st>>>(p);
    else
        backward_tiles<E, V, kBackwardPer / V, false, kTanh><<<p.strips, kThreads, 0, st>>>(p);
}
// A kernel a candidate: with both in one, the registers of the split passes in 16 bits pass 128 and a compute
// unit holds one workgroup instead of two (8 x 4096 x 2048 forward and backward: 403 us instead of 280).
template <typename E, int V>
void launch_forward_as(const Args& p, bool split, hipStream_t st) {
    p.candidate == HSN_SCAN_TANH ? launch_forward_as<E, V, true>(p, split, st)
                                 : launch_forward_as<E, V, false>(p, split, st);
}
template <typename E, int V>
void launch_backward_as(const Args& p, bool split, hipStream_t st) {
    p.candidate == HSN_SCAN_TANH ? launch_backward_as<E, V, true>(p, split, st)
                                 : launch_backward_as<E, V, false>(p, split, st);
}
template <typename E>
void launch_forward(const Args& p, int vec, bool split, hipStream_t st) {
    vec == 2 ? launch_forward_as<E, 2>(p, split, st) : launch_forward_as<E, 1>(p, split, st);
}
template <typename E>
void launch_backward(const Args& p, int vec, bool split, hipStream_t st) {
    vec == 2 ? launch_backward_as<E, 2>(p, split, st) : launch_backward_as<E, 1>(p, split, st);
}
#endif

}  // namespace scan
}  // namespace hsn
