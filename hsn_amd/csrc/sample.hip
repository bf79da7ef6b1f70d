// The choice of a token from logits (include/hsn_sample.h): one workgroup a row, or, where rows are few
// and long, a workgroup a slice of one for the passes over the logits and then one a row.
//
// A token's weight is a whole number, so masses can be added in any order: by atomics into
// histogram bins, by lanes, by waves. The order of tokens is the order of score_key(logit), then
// of the token. A row takes these passes over its logits:
//   1. the largest logit and its first token (all that a greedy row needs).
//   2. with top_k up to 512, or without a top_k and with a top_p: a list. The k-th largest of the 1024
//      threads' own largest keys is no larger than the k-th largest key of the row, so every token
//      that top_k keeps is among those from it on, some k (1 + k / 2048) of them where the large
//      ones lie anywhere. They (or those from a little below it on, found by one histogram of the 1024
//      keys) are gathered into LDS and sorted there, the other filters and the choice follow on the
//      list, and no other token's exponential is ever taken. top_p alone takes some 680 tokens and
//      the row's whole mass, and is done where they hold its share.
//      Else: counts and masses in 2048 bins, linear in x over the range where a weight is not 0 (x >
//      -27.73). They say in which bin a filter cuts, and the bin's tokens, gathered and sorted, at which
//      token; where a bin has more than 1024 (equal logits), the cut is found on the keys' digits (11, 11
//      and 10 bits), a pass over the row for each.
//   3. without a list: the kept weights' sums in the order of tokens, 64 packs of 16 bytes at a time,
//      then one wave's walk through the 64 packs that hold the answer.
// What bounds a row is one workgroup's steps in turn, and in the passes that take exponentials its
// instructions (an exact one and its fixed point are some 30). One row of 32000 in bf16 with top_k and
// top_p takes 12 us. 64 rows of 131072 in bf16 take 33 us,
// 12.6 of them the slices' launch; 256 rows of 200003 in fp32 96 us, 59 of them the slices', which read the
// logits once from HBM and where there are lists once more from the last-level cache (38.5 us at a
// copy's 5.3 TB/s), and 25 the exponentials of the rows that top_k does not cut.
#include <algorithm>
#include <type_traits>

#include "../../include/hsn_sample.h"
#include "abi_util.h"
#include "common.cuh"
#include "dpp.cuh"

namespace hsn {
namespace sample {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
// Packs a thread has in flight where it only compares keys; where it takes exponentials the other
// waves' instructions hide a load.
constexpr int kBatch = 4;
constexpr int kBins = 2048, kList = 1024;
constexpr int kListTop = kList / 2;  // the largest top_k that a list is tried for
constexpr int kMostSlices = 16;
constexpr int kSumThreads = 256;  // of sample_sums
constexpr int kAhead = 4;          // sums of 64 packs that a wave makes in one go
constexpr float kBinScale = kBins / 27.75f;  // 2^-40 = exp(-27.726)
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // score_key(-inf)
constexpr int kChunks = 2 * kThreads;        // sums of 64 packs: 2^18 / (64 * 4) + 1 at most

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct Args {
    const void* logits;
    int64_t row;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    hsn_sample_settings settings;
    int64_t* tokens;
    int V;
    // a row in slices of slice_packs packs (0: whole rows), with [n, slices] each, and lists of kList
    int slices, slice_packs;
    uint32_t* best;    // the slice's largest key
    int* first;        // its first token
    uint32_t* listed;  // how many tokens the slice's list has; above kList: no list
    uint64_t* lists;
    uint64_t* sums;    // [n, kChunks] sums of 64 packs' weights
    uint32_t* arrived; // [n] how many parts of the sums are there
    int parts;         // workgroups a row in sample_parts; 0: sample_sums has made the sums
};

// A row's settings; NaN and 0 temperatures are greedy.
struct Settings {
    float t, top_p, min_p, u;
    int top_k;
    bool cuts_k, cuts_p;
    __device__ Settings(const Args& a, int i) {
        t = a.temperature ? a.temperature[i] : a.settings.temperature;
        top_k = a.top_k ? a.top_k[i] : a.settings.top_k;
        top_p = a.top_p ? a.top_p[i] : a.settings.top_p;
        min_p = a.min_p ? a.min_p[i] : a.settings.min_p;
        u = a.u[i];
        cuts_k = top_k > 0 && top_k < a.V;
        cuts_p = !(top_p >= 1.0f);
    }
    __device__ bool greedy() const { return !(t > 0); }
    // whether a list of the largest tokens is tried, and from the how-many-th largest of the threads'
    // maxima over `packs` packs on: top_k's, or as many as a list holds (a twelfth of the tokens
    // where the packs are few)
    __device__ bool lists() const { return cuts_k ? top_k <= kListTop : cuts_p; }
    __device__ int list_top(int packs) const { return cuts_k ? top_k : min(kListTop, max(1, packs / 2)); }
};

struct Shared {
    uint64_t mass[kBins];   // bins; then the sums of 64 packs
    uint32_t count[kBins];
    uint64_t list[kList];
    uint64_t wave64[kWaves];
    uint32_t wave32[kWaves];
    uint32_t n_list, found, found_below;
    uint64_t found_mass;
};
static_assert(kBins == 2 * kThreads && kChunks <= kBins, "two bins a thread");

__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ (static_cast<int32_t>(k) < 0 ? 0x80000000u : 0xffffffffu));
}

// A row's logits as packs of 16 bytes from the last 16-byte boundary at or before its start. Packs
// [whole, whole_end) lie inside the row.
template <typename E>
struct Row {
    static constexpr int kVec = 16 / sizeof(E);
    const E* at;  // of pack 0's first element
    int skip, V, packs, whole, whole_end;
    __device__ Row(const E* row, int v) : V(v) {
        skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) / sizeof(E)) % kVec);
        at = row - skip;
        packs = (V + skip + kVec - 1) / kVec;
        whole = skip ? 1 : 0;
        whole_end = (V + skip) / kVec;
    }
    __device__ __forceinline__ int first(int p) const { return p * kVec - skip; }
    // Packs p, p + stride, ..: N loads in flight. A pack that is not whole is read element by element
    // afterwards; outside the row there is -inf.
    template <int N>
    __device__ __forceinline__ void load(int p, int stride, v4u (&pack)[N]) const {
        if (whole < whole_end)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int q = min(max(p + n * stride, whole), whole_end - 1);
                pack[n] = *reinterpret_cast<const v4u*>(at + int64_t(q) * kVec);
            }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int q = p + n * stride;
            if (q >= whole && q < whole_end) continue;
            E e[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const int t = first(q) + j;
                e[j] = t >= 0 && t < V ? at[int64_t(q) * kVec + j] : from_f32<E>(-__builtin_inff());
            }
            __builtin_memcpy(&pack[n], e, 16);
        }
    }
    // A pack's logits, and their keys; NaN counts as -inf.
    static __device__ __forceinline__ void values(const v4u& pack, float (&l)[kVec]) {
        E e[kVec];
        __builtin_memcpy(e, &pack, 16);
#pragma unroll
        for (int j = 0; j < kVec; ++j) l[j] = to_f32(e[j]);
    }
    static __device__ __forceinline__ uint32_t key(float l) { return l != l ? kKeyNegInf : score_key(l); }
    static __device__ __forceinline__ void keys(const v4u& pack, uint32_t (&k)[kVec]) {
        float l[kVec];
        values(pack, l);
#pragma unroll
        for (int j = 0; j < kVec; ++j) k[j] = key(l[j]);
    }
    // f(first token, pack) for packs [from, to), the workgroup's threads side by side, N loads in flight.
    template <int N, typename F>
    __device__ __forceinline__ void each(int from, int to, F&& f) const {
        for (int p = from + int(threadIdx.x); p < to; p += N * kThreads) {
            v4u pack[N];
            load(p, kThreads, pack);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (p + n * kThreads >= to) break;
                f(first(p + n * kThreads), pack[n]);
            }
        }
    }
};

// The largest of a pack's logits, NaN aside.
template <int N>
__device__ __forceinline__ float largest(const float (&l)[N]) {
    float m = l[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = __builtin_fmaxf(m, l[j]);
    return m;
}

// The weight of a logit by its key: e, and w as the fixed point of e.
//
// x = d / t, d = l - best, is the correctly rounded quotient. With r the rounded 1 / t, d r is within 2
// ulps of it; q + (d - q t) r brings that within 1 ulp, and once more to the correctly rounded quotient
// (Markstein, IBM J. Res. Dev. 34, 1990: the last step of a division by iteration), as long as nothing
// leaves the normal range: t within 2^+-60 (`quick`), and a d so small that it does gives e = 1 either
// way. A d of -inf gives a NaN, and no weight.
struct Weigh {
    uint32_t best_key;
    float best, t, r;
    bool quick;
    __device__ Weigh(uint32_t key, float temperature) : best_key(key), best(key_value(key)), t(temperature) {
        r = 1.0f / t;
        quick = t > 0x1p-60f && t < 0x1p60f && best < __builtin_inff();
    }
    __device__ __forceinline__ float x(uint32_t k) const {
        if (k == best_key) return 0.0f;
        const float d = key_value(k) - best;
        if (!quick) return d / t;
        const float near = d * r;
        const float q = __builtin_fmaf(__builtin_fmaf(-near, t, d), r, near);
        return __builtin_fmaf(__builtin_fmaf(-q, t, d), r, q);
    }
    static __device__ __forceinline__ float e_of(float x) {
        return x > -30.0f ? expf(x) : 0.0f;  // 2^40 e is below 1 from x = -27.73 on; NaN: none
    }
    __device__ __forceinline__ float e(uint32_t k) const {
        return k == kKeyNegInf ? 0.0f : e_of(x(k));
    }
    // floor(2^40 e) for 0 <= e <= 1: the 24 bits of e, shifted
    static __device__ __forceinline__ uint64_t fixed(float e) {
        const uint32_t bits = __float_as_uint(e);
        const uint64_t m = uint64_t((bits & 0x7fffffu) | 0x800000u) << 17;  // 2^40 at exponent 0
        const int down = 127 - static_cast<int>(bits >> 23);
        return down < 64 ? m >> down : 0;
    }
    __device__ __forceinline__ uint64_t w(uint32_t k) const { return fixed(e(k)); }
};

// The value CTRL lanes below by DPP (0 where there is none), for the sums below.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_below(uint32_t v) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_below(uint64_t v) {
    return uint64_t(dpp_below<CTRL, ROWS>(static_cast<uint32_t>(v >> 32))) << 32 |
           dpp_below<CTRL, ROWS>(static_cast<uint32_t>(v));
}

// Inclusive sum over 16 lanes, or over the wave, in lane order.
template <typename T>
__device__ __forceinline__ T row_scan(T v) {
    v += dpp_below<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp_below<0x112, 0xf>(v);
    v += dpp_below<0x114, 0xf>(v);
    v += dpp_below<0x118, 0xf>(v);
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v = row_scan(v);
    v += dpp_below<0x142, 0xa>(v);  // row_bcast:15 into the odd rows
    v += dpp_below<0x143, 0xc>(v);  // row_bcast:31 into the upper half
    return v;
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
    return uint64_t(readlane(static_cast<uint32_t>(v >> 32), lane)) << 32 |
           readlane(static_cast<uint32_t>(v), lane);
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return readlane(v, lane); }

__device__ __forceinline__ int bin_of(float x) {
    return min(kBins - 1, static_cast<int>(-x * kBinScale));
}

// Inclusive sum over the workgroup in thread order; `total` the whole. Ends with a barrier passed.
template <typename T>
__device__ __forceinline__ T block_scan(T v, Shared& s, T& total) {
    const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
    T* waves = reinterpret_cast<T*>(s.wave64);
    v = wave_scan(v);
    __syncthreads();
    if (lane == kWave - 1) waves[wave] = v;
    __syncthreads();
    const T run = row_scan(waves[lane % kWaves]);  // the waves' sums, in every row of lanes
    total = lane_value(run, kWaves - 1);
    return v + (wave ? lane_value(run, wave - 1) : T(0));
}
static_assert(kWaves == 16, "a row of lanes holds the waves' sums");

__device__ __forceinline__ uint32_t block_max(uint32_t v, Shared& s) {
    v = group_max<kWave>(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) s.wave32[threadIdx.x / kWave] = v;
    __syncthreads();
    return group_max<16>(s.wave32[threadIdx.x % kWaves]);
}

// The number of threads with `flag`, in every thread.
__device__ __forceinline__ int block_count(bool flag, Shared& s) {
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    const uint64_t lanes = ballot(flag);
    if (lanes && threadIdx.x % kWave == 0) atomicAdd(&s.n_list, uint32_t(__popcll(lanes)));
    __syncthreads();
    const int n = static_cast<int>(s.n_list);
    __syncthreads();
    return n;
}

__device__ __forceinline__ void clear_bins(Shared& s) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
}

// Where a filter cuts: it keeps the keys above `key` and the first `equal` tokens of `key`.
struct Cut {
    uint32_t key;
    uint64_t equal;
};

// The bin where the running count reaches `k` (by_count) or the running mass reaches `target`, in
// bin order; the counts and masses before it. `all` where none does.
struct Place {
    bool found;
    int bin;
    uint32_t count_before, count;
    uint64_t mass_before, mass;
};

__device__ __forceinline__ Place find_bin(Shared& s, bool by_count, uint64_t k, double target, uint64_t base) {
    const int b = 2 * threadIdx.x;
    const uint64_t m0 = s.mass[b], m1 = s.mass[b + 1];
    const uint32_t c0 = s.count[b], c1 = s.count[b + 1];
    uint64_t mt, ct;
    const uint64_t mi = block_scan(m0 + m1, s, mt), ci = block_scan(uint64_t(c0) + c1, s, ct);
    if (threadIdx.x == 0) s.found = kBins;
    __syncthreads();
    const uint64_t m_at[3] = {mi - m1 - m0, mi - m1, mi};
    const uint64_t c_at[3] = {ci - c1 - c0, ci - c1, ci};
    for (int i = 0; i < 2; ++i) {
        const bool before = by_count ? c_at[i] < k : static_cast<double>(base + m_at[i]) < target;
        const bool after = by_count ? c_at[i + 1] < k
                                    : static_cast<double>(base + m_at[i + 1]) < target;
        if (before && !after) {
            s.found = b + i;
            s.found_below = static_cast<uint32_t>(c_at[i]);
            s.found_mass = m_at[i];
        }
    }
    __syncthreads();
    Place p;
    p.found = s.found < kBins;
    p.bin = static_cast<int>(s.found);
    p.count_before = p.found ? s.found_below : static_cast<uint32_t>(ct);
    p.mass_before = p.found ? s.found_mass : mt;
    p.count = p.found ? s.count[p.bin] : 0;
    p.mass = p.found ? s.mass[p.bin] : 0;
    __syncthreads();
    return p;
}

// How many of `n` equal weights w a mass filter keeps, `base` of mass before them: the j-th is kept
// where the mass before it is under the target.
__device__ __forceinline__ uint64_t equal_under(uint64_t base, uint64_t w, uint64_t n, double target) {
    const double guess = (target - static_cast<double>(base)) / static_cast<double>(w);
    uint64_t c = guess > 0 ? (guess < double(n) ? static_cast<uint64_t>(guess) : n) : 0;
    while (c < n && static_cast<double>(base + c * w) < target) ++c;
    while (c > 0 && !(static_cast<double>(base + (c - 1) * w) < target)) --c;
    return c;
}

// The cut of one filter, found digit by digit; mass_at: the mass of what it keeps.
template <typename E>
__device__ __forceinline__ Cut descend(const Row<E>& row, const Weigh& weigh, Shared& s, bool by_count, uint64_t k,
                       double target, uint64_t& mass_at) {
    uint32_t prefix = 0;
    uint64_t base_mass = 0, base_count = 0;
    const int shifts[4] = {32, 21, 10, 0};
    for (int level = 1; level <= 3; ++level) {
        const int up = shifts[level - 1], shift = shifts[level], bits = up - shift;
        clear_bins(s);
        row.template each<1>(0, row.packs, [&](int, const v4u& pack) {
            uint32_t key[Row<E>::kVec];
            Row<E>::keys(pack, key);
            for (int i = 0; i < Row<E>::kVec; ++i) {
                if (level > 1 && key[i] >> up != prefix) continue;
                const uint64_t w = weigh.w(key[i]);
                if (!w) continue;
                const uint32_t digit = (key[i] >> shift) & ((1u << bits) - 1);
                const uint32_t bin = (1u << bits) - 1 - digit;  // the largest keys first
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[bin]), (unsigned long long)w);
                atomicAdd(&s.count[bin], 1u);
            }
        });
        __syncthreads();
        const Place at = find_bin(s, by_count, by_count ? k - base_count : 0, target, base_mass);
        if (!at.found) {  // the filter keeps everything
            mass_at = base_mass + at.mass_before;
            return Cut{0, 0};
        }
        base_mass += at.mass_before;
        base_count += at.count_before;
        prefix = prefix << bits | ((1u << bits) - 1 - at.bin);
        if (level == 3) {
            const uint64_t w = at.mass / at.count;
            const uint64_t n = by_count ? k - base_count
                                        : equal_under(base_mass, w, at.count, target);
            mass_at = base_mass + n * w;
            return {prefix, n};
        }
    }
    return {0, 0};
}

template <typename E, typename F>
__device__ __forceinline__ uint64_t pack_sum(const Row<E>& row, int p, const v4u& pack, F&& f,
                                             uint64_t (&w)[Row<E>::kVec]) {
    uint64_t sum = 0;
    uint32_t key[Row<E>::kVec];
    Row<E>::keys(pack, key);
#pragma unroll
    for (int i = 0; i < Row<E>::kVec; ++i) {
        w[i] = p < row.packs ? f(key[i], row.first(p) + i) : 0;
        sum += w[i];
    }
    return sum;
}

// The sums of f(key, token) over 64 packs each, from chunk `from` up to `to` (`sums`: the first one's
// place), a wave a sum, the loads of N in flight.
template <int N, typename E, typename F>
__device__ __forceinline__ void chunk_sums(const Row<E>& row, int from, int to, uint64_t* sums, F&& f) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    for (int c = from + wave; c < to; c += N * waves) {
        v4u pack[N];
        row.load(c * kWave + lane, waves * kWave, pack);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = c + k * waves;
            if (at >= to) break;
            uint64_t w[Row<E>::kVec];
            const uint64_t sum = wave_scan(pack_sum(row, at * kWave + lane, pack[k], f, w));
            if (lane == kWave - 1) sums[at - from] = sum;
        }
    }
}

// The first token, in order, at which the running sum of f(key, token) exceeds `limit(total)`;
// V where none does. `sums`: the sums of 64 packs where they are made already, else NULL.
template <typename E, typename F, typename L>
__device__ __forceinline__ int walk(const Row<E>& row, Shared& s, const uint64_t* sums, F&& f, L&& limit) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int chunks = (row.packs + kWave - 1) / kWave;
    __syncthreads();
    if (threadIdx.x == 0) s.found = kChunks;
    if (!sums) chunk_sums<1>(row, 0, chunks, s.mass, f);
    __syncthreads();
    if (!sums) sums = s.mass;
    const int c0 = 2 * threadIdx.x, c1 = c0 + 1;
    const uint64_t s0 = c0 < chunks ? sums[c0] : 0, s1 = c1 < chunks ? sums[c1] : 0;
    uint64_t total;
    const uint64_t end = block_scan(s0 + s1, s, total);
    const uint64_t r = limit(total);
    const uint64_t at[3] = {end - s1 - s0, end - s1, end};
    for (int i = 0; i < 2; ++i)
        if (at[i] <= r && at[i + 1] > r) {
            s.found = 2 * threadIdx.x + i;
            s.found_mass = at[i];
            s.found_below = row.V;
        }
    __syncthreads();
    const uint32_t c = s.found;
    if (c >= kChunks) return row.V;
    if (wave == 0) {
        const int p = c * kWave + lane;
        v4u pack[1];
        row.load(p, 0, pack);
        uint64_t w[Row<E>::kVec];
        const uint64_t sum = pack_sum(row, p, pack[0], f, w);
        uint64_t run = wave_scan(sum) + s.found_mass - sum;  // before this pack
        if (run <= r && run + sum > r) {
            int below = 0;  // tokens of the pack before the answer
#pragma unroll
            for (int i = 0; i < Row<E>::kVec; ++i) {
                run += w[i];
                below += run <= r;
            }
            s.found_below = row.first(p) + below;
        }
    }
    __syncthreads();
    return static_cast<int>(s.found_below);
}

// The value of lane ^ J, without LDS: within 16 lanes by DPP, across rows by the permlane swaps.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (J == 1) return dpp_u32<dpp::kXor1>(v);
    if constexpr (J == 2) return dpp_u32<dpp::kXor2>(v);
    if constexpr (J == 4) return dpp_u32<0x1B>(dpp_u32<dpp::kHalfMirror>(v));  // ^7, then ^3
    if constexpr (J == 8) return dpp_u32<dpp::kRor8>(v);
    if constexpr (J == 16) {
        const RowPair r = pair16(v);
        return lane_id() & 16 ? r.lo : r.hi;
    }
    if constexpr (J == 32) {
        const RowPair r = pair32(v);
        return lane_id() & 32 ? r.lo : r.hi;
    }
}
template <int J>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
    return uint64_t(lane_xor<J>(static_cast<uint32_t>(v >> 32))) << 32 |
           lane_xor<J>(static_cast<uint32_t>(v));
}

// The steps J, J / 2, .. 1 of a bitonic merge within a wave.
template <int J>
__device__ __forceinline__ void wave_merge(uint64_t& v, bool down) {
    const uint64_t o = lane_xor<J>(v);
    v = down == ((lane_id() & J) == 0) ? max(v, o) : min(v, o);
    if constexpr (J > 1) wave_merge<J / 2>(v, down);
}
template <int K>
__device__ __forceinline__ void wave_sort(uint64_t& v) {
    if constexpr (K > 2) wave_sort<K / 2>(v);
    wave_merge<K / 2>(v, (threadIdx.x & K) == 0);
}

// Sorts the first `n` threads' values (n <= kList), the largest first; the other threads up to the
// next power of two hold 0. Waves beyond it only pass the barriers.
__device__ __forceinline__ uint64_t sort_down(uint64_t v, int n, Shared& s) {
    const int i = threadIdx.x;
    int size = kWave;
    while (size < n) size *= 2;
    const bool in = i < size;
    if (in) wave_sort<kWave>(v);
    for (int k = 2 * kWave; k <= size; k *= 2) {
        for (int j = k / 2; j >= kWave; j /= 2) {
            __syncthreads();
            s.list[i] = v;
            __syncthreads();
            const uint64_t o = s.list[i ^ j];
            if (in) v = ((i & k) == 0) == ((i & j) == 0) ? max(v, o) : min(v, o);
        }
        if (in) wave_merge<kWave / 2>(v, (i & k) == 0);
    }
    __syncthreads();
    return v;
}

__device__ __forceinline__ uint64_t at_share(float u, uint64_t total) {
    const double r = floor(static_cast<double>(u) * static_cast<double>(total));
    const uint64_t i = r > 0 ? static_cast<uint64_t>(r) : 0;
    return i < total ? i : total - 1;
}

// The mass that top_p asks for; a positive one, so that the first token is under it.
__device__ __forceinline__ double mass_target(float top_p, uint64_t total) {
    const double target = static_cast<double>(top_p) * static_cast<double>(total);
    return target > 0 ? target : 1.0;
}

// The rest of a row on its list of `n` tokens (in LDS, any order), whose `sure` largest are the row's
// largest. by_count: these are what top_k keeps; else top_p cuts, `total` is the row's whole mass,
// and where the sure tokens do not hold what top_p keeps the answer is false and nothing is written.
__device__ __forceinline__ bool finish_list(Shared& s, const Weigh& weigh, int n, bool by_count, int sure,
                                            float top_p, float min_p, float u, uint64_t total,
                                            int64_t* token) {
    const int tid = threadIdx.x;
    uint64_t v = tid < n ? s.list[tid] : 0;
    v = sort_down(v, n, s);
    uint32_t key = static_cast<uint32_t>(v >> 32);
    const float e = tid < n ? weigh.e(key) : 0.0f;
    uint64_t w = tid < min(n, sure) ? Weigh::fixed(e) : 0;
    uint64_t sum;
    const uint64_t run = block_scan(w, s, sum);
    const double target = mass_target(top_p, by_count ? sum : total);
    if (!by_count && static_cast<double>(sum) < target) return false;
    bool kept = w && (top_p >= 1.0f || static_cast<double>(run - w) < target) && e >= min_p;
    kept |= tid == 0;
    // the kept tokens, the list's first ones, in their order: the least token is the largest complement
    const int left = block_count(kept, s);
    v = kept ? (v << 32 | v >> 32) : 0;
    v = sort_down(v, left, s);
    key = static_cast<uint32_t>(v);
    w = v && tid < left ? weigh.w(key) : 0;
    const uint64_t end = block_scan(w, s, sum);
    const uint64_t r = at_share(u, sum);
    if (w && end > r && end - w <= r) *token = int64_t(uint32_t(~(v >> 32)));
    return true;
}

// Every token of packs [from, to) with a key from `least` on that `wanted(key)` takes, into the list; how
// many there are (the list holds kList).
template <typename E, typename F>
__device__ __forceinline__ int gather(const Row<E>& row, int from, int to, Shared& s, uint32_t least, F&& wanted) {
    __syncthreads();
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    const float edge = key_value(least);  // keys from `least` on are the logits from here on
    row.template each<kBatch>(from, to, [&](int first, const v4u& pack) {
        float l[Row<E>::kVec];
        Row<E>::values(pack, l);
        if (!(largest(l) >= edge)) return;
#pragma unroll
        for (int j = 0; j < Row<E>::kVec; ++j) {
            if (!(l[j] >= edge)) continue;
            const uint32_t key = Row<E>::key(l[j]);
            if (!wanted(key)) continue;
            const uint32_t place = atomicAdd(&s.n_list, 1u);
            if (place < kList) s.list[place] = uint64_t(key) << 32 | uint32_t(~(first + j));
        }
    });
    __syncthreads();
    const int n = static_cast<int>(s.n_list);
    __syncthreads();
    return n;
}

// A filter's cut inside one bin, whose `n` tokens are the list: by_count, the first k tokens stay, else
// those with a mass before them, `before` and the bin's, under the target. mass_at: what stays, with
// `before`.
__device__ __forceinline__ Cut cut_list(Shared& s, const Weigh& weigh, int n, bool by_count, int k,
                                        double target, uint64_t before, uint64_t& mass_at) {
    const int tid = threadIdx.x;
    const uint64_t v = sort_down(tid < n ? s.list[tid] : 0, n, s);
    const uint32_t key = static_cast<uint32_t>(v >> 32);
    const uint64_t w = tid < n ? weigh.w(key) : 0;
    uint64_t sum;
    const uint64_t run = before + block_scan(w, s, sum);
    const bool kept = tid < n && (by_count ? tid < k : static_cast<double>(run - w) < target);
    const int stay = block_count(kept, s);  // the first ones
    if (tid == stay - 1) s.found = key, s.found_mass = run;
    __syncthreads();
    const uint32_t last = s.found;
    mass_at = s.found_mass;
    return Cut{last, uint64_t(stay - block_count(tid < n && key > last, s))};
}

// A token's weight where top_k and top_p do not cut (min_p 0: where they have not cut yet); the row's
// first token always has one.
struct Plain {
    Weigh weigh;
    float min_p;
    int first;
    __device__ __forceinline__ uint64_t operator()(uint32_t k, int token) const {
        const float e = weigh.e(k);
        return e >= min_p || token == first ? Weigh::fixed(e) : 0;
    }
};

// The largest key of packs [from, to) and its first token; `mine`: the thread's largest.
template <typename E>
__device__ __forceinline__ void find_best(const Row<E>& row, int from, int to, Shared& s, uint32_t& mine,
                                          uint32_t& best, int& first) {
    float top = -__builtin_inff();
    first = row.V;
    row.template each<kBatch>(from, to, [&](int at, const v4u& pack) {
        float l[Row<E>::kVec];
        Row<E>::values(pack, l);
        if (!(largest(l) > top)) return;
#pragma unroll
        for (int j = 0; j < Row<E>::kVec; ++j)
            if (l[j] > top) top = l[j], first = at + j;
    });
    mine = score_key(top);
    best = block_max(mine, s);
    // the least first token: the largest of its complement
    first = ~block_max(mine == best ? ~static_cast<uint32_t>(first) : 0, s);
}

// A key no larger than the k-th largest of the threads' keys `mine`, and above -inf: the end of the bin
// that the k-th lies in, of 1024 bins from `best` down to the least of them or to three octaves below.
__device__ __forceinline__ uint32_t list_from(uint32_t mine, uint32_t best, int k, Shared& s) {
    constexpr uint32_t kFurthest = 3u << 23;
    const int tid = threadIdx.x;
    mine = max(mine, kKeyNegInf);
    const uint32_t lowest = ~block_max(~mine, s);
    const uint32_t range = min(best - lowest, kFurthest);
    const int shift = max(0, 32 - __clz(int(range)) - 10);  // range >> shift < 1024
    s.count[tid] = 0;
    if (tid == 0) s.found = kThreads;
    __syncthreads();
    if (mine > kKeyNegInf) atomicAdd(&s.count[min(best - mine, range) >> shift], 1u);
    __syncthreads();
    uint32_t all;
    const uint32_t here = s.count[tid], run = block_scan(here, s, all);
    if (run >= uint32_t(k) && run - here < uint32_t(k)) s.found = tid;
    __syncthreads();
    const uint32_t bin = s.found;
    if (bin == kThreads) return kKeyNegInf + 1;  // fewer than k threads have a key
    const uint32_t end = (bin + 1) << shift;
    if (end <= range) return best - end + 1;
    return range < kFurthest ? max(lowest, kKeyNegInf + 1) : kKeyNegInf + 1;  // the last bin
}

// One slice of a row: its largest key, and its list where top_k is tried by lists.
template <typename E>
__global__ __launch_bounds__(kThreads) void sample_slices(Args a) {
    __shared__ Shared s;
    const int i = blockIdx.y, at = i * a.slices + blockIdx.x, tid = threadIdx.x;
    const Row<E> row(static_cast<const E*>(a.logits) + i * a.row, a.V);
    const Settings set(a, i);
    const int from = blockIdx.x * a.slice_packs, to = min(row.packs, from + a.slice_packs);
    uint32_t mine, best;
    int first;
    find_best(row, from, to, s, mine, best, first);
    if (tid == 0) a.best[at] = best, a.first[at] = first;
    if (tid == 0 && blockIdx.x == 0) a.arrived[i] = 0;
    if (set.greedy() || !set.lists()) return;
    const int n = best > kKeyNegInf ? gather(row, from, to, s, list_from(mine, best, set.list_top(row.packs), s),
                                              [](uint32_t) { return true; }) : 0;
    if (tid == 0) a.listed[at] = n;
    if (tid < n) a.lists[int64_t(at) * kList + tid] = s.list[tid];
}

// The largest key and its first token from the slices', a lane a slice.
__device__ __forceinline__ void best_of_slices(const Args& a, int i, uint32_t& best, int& first) {
    const int k = threadIdx.x % kMostSlices, at = i * a.slices + min(k, a.slices - 1);
    const uint32_t key = a.best[at], token = a.first[at];
    best = group_max<kMostSlices>(key);
    first = ~group_max<kMostSlices>(key == best ? ~token : 0);
}
static_assert(kMostSlices == 16, "a row of lanes holds the slices");

// The slices' lists as one: the tokens from the k-th largest of the threads' maxima over them on;
// how many, or more than kList where there is no such list.
__device__ __forceinline__ int merge_lists(const Args& a, int i, int k, uint32_t best, Shared& s) {
    const int tid = threadIdx.x;
    uint64_t v[kMostSlices];
    uint32_t mine = 0;
    bool whole = true;
#pragma unroll
    for (int j = 0; j < kMostSlices; ++j) {
        const int at = i * a.slices + min(j, a.slices - 1);
        const uint32_t n = j < a.slices ? a.listed[at] : 0;
        whole &= n <= kList;
        v[j] = tid < int(n) && n <= kList ? a.lists[int64_t(at) * kList + tid] : 0;
    }
    if (!whole) return kList + 1;
#pragma unroll
    for (int j = 0; j < kMostSlices; ++j) mine = max(mine, static_cast<uint32_t>(v[j] >> 32));
    const uint32_t least = list_from(mine, best, k, s);
    if (tid == 0) s.n_list = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMostSlices; ++j)
        if (static_cast<uint32_t>(v[j] >> 32) >= least) {
            const uint32_t place = atomicAdd(&s.n_list, 1u);
            if (place < kList) s.list[place] = v[j];
        }
    __syncthreads();
    return static_cast<int>(s.n_list);
}

// A row: from its logits, or (kSlices) from what its slices have left.
template <typename E, bool kSlices>
__device__ __forceinline__ void finish_row(const Args& a, Shared& s, int i) {
    const int tid = threadIdx.x;
    const Row<E> row(static_cast<const E*>(a.logits) + i * a.row, a.V);
    constexpr int kVec = Row<E>::kVec;
    const Settings set(a, i);
    const int top_k = set.top_k;
    const float top_p = set.top_p, min_p = set.min_p, u = set.u;
    const bool cuts_k = set.cuts_k, cuts_p = set.cuts_p;

    uint32_t mine = 0, best;
    int first;
    if constexpr (kSlices)
        best_of_slices(a, i, best, first);
    else
        find_best(row, 0, row.packs, s, mine, best, first);
    if (best <= kKeyNegInf || set.greedy()) {
        if (tid == 0) a.tokens[i] = best <= kKeyNegInf ? -1 : first;
        return;
    }
    const Weigh weigh(best, set.t);
    if (set.lists()) {
        int n;
        if constexpr (kSlices)
            n = merge_lists(a, i, set.list_top(row.packs), best, s);
        else
            n = gather(row, 0, row.packs, s, list_from(mine, best, set.list_top(row.packs), s),
                       [](uint32_t) { return true; });
        if (n <= kList) {
            uint64_t total = 0;
            if (!cuts_k) {
                uint64_t here = 0;
                if constexpr (kSlices) {
                    for (int c = tid; c * kWave < row.packs; c += kThreads)
                        here += a.sums[int64_t(i) * kChunks + c];
                } else {
                    row.template each<1>(0, row.packs, [&](int, const v4u& pack) {
                        uint32_t key[kVec];
                        Row<E>::keys(pack, key);
#pragma unroll
                        for (int j = 0; j < kVec; ++j) here += weigh.w(key[j]);
                    });
                }
                block_scan(here, s, total);
            }
            // the slices' lists are whole down to their own ends only, and each has as many as asked for
            const int sure = cuts_k ? top_k : kSlices ? set.list_top(row.packs) : n;
            if (finish_list(s, weigh, n, cuts_k, sure, top_p, min_p, u, total, a.tokens + i)) return;
        }
    }
    Cut cut{0, 0};
    if (cuts_k || cuts_p) {
        clear_bins(s);
        row.template each<1>(0, row.packs, [&](int, const v4u& pack) {
            uint32_t key[kVec];
            Row<E>::keys(pack, key);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                if (key[j] == kKeyNegInf) continue;
                const float x = weigh.x(key[j]);
                const uint64_t w = Weigh::fixed(Weigh::e_of(x));
                if (!w) continue;
                const int bin = bin_of(x);
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[bin]), (unsigned long long)w);
                if (cuts_k) atomicAdd(&s.count[bin], 1u);
            }
        });
        __syncthreads();
        uint64_t total;
        block_scan(s.mass[2 * tid] + s.mass[2 * tid + 1], s, total);
        bool bins = true;
#pragma unroll 1
        for (int filter = 0; filter < 2; ++filter) {  // top_k, then top_p of what it keeps
            const bool by_count = filter == 0;
            if (by_count ? !cuts_k : !cuts_p) continue;
            const double target = mass_target(top_p, total);
            Place at{};
            int n = kList + 1;
            if (bins) {
                at = find_bin(s, by_count, top_k, target, 0);
                if (!at.found) continue;  // it keeps every token with a weight
                n = gather(row, 0, row.packs, s, kKeyNegInf + 1, [&](uint32_t k) {
                    const float x = weigh.x(k);
                    return x > -30.0f && bin_of(x) == at.bin && weigh.w(k);
                });
            }
            Cut c;
            uint64_t mass;
            if (n <= kList) {
                c = cut_list(s, weigh, n, by_count, top_k - int(at.count_before), target, at.mass_before, mass);
            } else {
                c = descend(row, weigh, s, by_count, top_k, target, mass);
                bins = false;
            }
            if (by_count) total = mass;
            if (c.key > cut.key || (c.key == cut.key && c.equal < cut.equal)) cut = c;
        }
    }
    // the last token kept among those equal to the cut's key
    int last_equal = a.V;
    if (cut.key)
        last_equal = walk(row, s, nullptr, [&](uint32_t k, int) { return uint64_t(k == cut.key); },
                          [&](uint64_t) { return cut.equal - 1; });
    const Plain plain{weigh, min_p, first};
    const int token = walk(
        row, s, kSlices && !cuts_k && !cuts_p ? a.sums + int64_t(i) * kChunks : nullptr,
        [&](uint32_t k, int j) {
            return k < cut.key || (k == cut.key && j > last_equal) ? uint64_t(0) : plain(k, j);
        },
        [&](uint64_t whole) { return at_share(u, whole); });
    if (tid == 0) a.tokens[i] = token;
}

template <typename E>
__global__ __launch_bounds__(kThreads) void sample_rows(Args a) {
    __shared__ Shared s;
    finish_row<E, false>(a, s, blockIdx.x);
}

// A row's sums of 64 packs' weights, chunks [from, to) of them, to `sums`.
template <typename E>
__device__ __forceinline__ void part_sums(const Args& a, int i, int from, int to, uint64_t* sums,
                                          const Settings& set, uint32_t best, int first) {
    const Row<E> row(static_cast<const E*>(a.logits) + i * a.row, a.V);
    chunk_sums<kAhead>(row, from, min((row.packs + kWave - 1) / kWave, to), sums,
                       Plain{Weigh(best, set.t), set.cuts_p ? 0.0f : set.min_p, first});
}

// The sums of all rows that need them: those that top_k does not cut.
template <typename E>
__global__ __launch_bounds__(kSumThreads) void sample_sums(Args a) {
    const int i = blockIdx.y;
    const Settings set(a, i);
    if (set.greedy() || set.cuts_k) return;
    uint32_t best;
    int first;
    best_of_slices(a, i, best, first);
    constexpr int kPart = kAhead * kSumThreads / kWave;  // kAhead a wave
    const int from = blockIdx.x * kPart;
    if (best > kKeyNegInf)
        part_sums<E>(a, i, from, from + kPart, a.sums + int64_t(i) * kChunks + from, set, best, first);
}

// The rows whose slices are there. One that needs the sums has them made by `parts` workgroups, and
// whoever comes last finishes it; no workgroup waits. Any other row is one workgroup's, at the same time.
// A workgroup's sums go through LDS to its first wave, which stores them, releases them to the device and
// counts: the reader may sit behind another L2, and a wave's release waits for its own stores only. (Sums
// stored by every wave need a release by every wave: 64 rows of 131072 in bf16 37.6 us.)
template <typename E>
__global__ __launch_bounds__(kThreads) void sample_parts(Args a) {
    __shared__ Shared s;
    const int parts = max(a.parts, 1), i = blockIdx.x / parts, part = blockIdx.x % parts;
    if (a.parts) {
        const Settings set(a, i);
        uint32_t best;
        int first;
        best_of_slices(a, i, best, first);
        if (set.greedy() || set.cuts_k || best <= kKeyNegInf) {
            if (part) return;
        } else {
            constexpr int kPart = kAhead * kThreads / kWave;
            static_assert(kPart == kWave, "a part's sums, a lane each");
            const int from = part * kPart, lane = threadIdx.x;
            part_sums<E>(a, i, from, from + kPart, s.mass, set, best, first);
            __syncthreads();
            if (lane < kWave) {
                const Row<E> row(static_cast<const E*>(a.logits) + i * a.row, a.V);
                if ((from + lane) * kWave < row.packs) a.sums[int64_t(i) * kChunks + from + lane] = s.mass[lane];
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
                if (lane == 0)
                    s.found = __hip_atomic_fetch_add(a.arrived + i, 1u, __ATOMIC_ACQ_REL,
                                                     __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (s.found != uint32_t(parts - 1)) return;
            __syncthreads();
        }
    }
    finish_row<E, true>(a, s, i);
}

}  // namespace
}  // namespace sample
}  // namespace hsn

namespace hsn {
namespace sample {
namespace {

// Rows in slices: some 512 workgroups, each with at least a pack a thread. Whole rows (0) where they
// fill the GPU or are short.
int slices_of(int n, int V, int size) {
    const int packs = (V + 16 / size - 1) / (16 / size) + 1;
    const int slices = std::min(kMostSlices, std::min(packs / (2 * kThreads), 512 / std::max(n, 1)));
    return slices > 1 ? slices : 0;
}

int64_t layout(Args& a, char* base, int n, int size) {
    a.slices = slices_of(n, a.V, size);
    if (!a.slices) return 0;
    const int packs = (a.V + 16 / size - 1) / (16 / size) + 1;  // of a row at any address
    a.slice_packs = ((packs + a.slices - 1) / a.slices + kWave - 1) / kWave * kWave;
    const int64_t parts = int64_t(n) * a.slices;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char* p = base + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    a.lists = reinterpret_cast<uint64_t*>(take(8 * parts * kList));
    a.sums = reinterpret_cast<uint64_t*>(take(8 * int64_t(n) * kChunks));
    a.arrived = reinterpret_cast<uint32_t*>(take(4 * int64_t(n)));
    a.best = reinterpret_cast<uint32_t*>(take(4 * parts));
    a.first = reinterpret_cast<int*>(take(4 * parts));
    a.listed = reinterpret_cast<uint32_t*>(take(4 * parts));
    return at;
}

template <typename E>
void launch(Args a, int n, hipStream_t st) {
    if (!a.slices) {
        sample_rows<E><<<n, kThreads, 0, st>>>(a);
        return;
    }
    sample_slices<E><<<dim3(a.slices, n), kThreads, 0, st>>>(a);
    // Where top_k is the same for all rows, whether they need the sums is known here. A few rows' are made on
    // the way (64 rows of 131072 in bf16, some of them cut: 33.5 us a call, with a launch of their own 38.3).
    // Many rows' workgroups would mostly find nothing to do, and a compute unit holds one of them (256
    // rows of 200003 in fp32: 131 against 96 us).
    const hsn_sample_settings& f = a.settings;
    const bool cut = !a.top_k && f.top_k > 0 && f.top_k < a.V;
    const int chunks = (a.slices * a.slice_packs + kWave - 1) / kWave;
    auto parts = [&](int threads) {
        const int of = kAhead * threads / kWave;
        return (chunks + of - 1) / of;
    };
    a.parts = cut ? 0 : parts(kThreads);
    if (int64_t(n) * a.parts > 512) {
        a.parts = 0;
        sample_sums<E><<<dim3(parts(kSumThreads), n), kSumThreads, 0, st>>>(a);
    }
    sample_parts<E><<<n * std::max(a.parts, 1), kThreads, 0, st>>>(a);
}

void check(int n, int V, int dtype) {
    HSN_REQUIRE(dtype == HSN_DTYPE_F32 || dtype == HSN_DTYPE_F16 || dtype == HSN_DTYPE_BF16,
                HSN_ERR_UNSUPPORTED_DTYPE, "logits must be F32, F16 or BF16");
    HSN_REQUIRE(n >= 0 && V >= 1, HSN_ERR_INVALID_ARGUMENT, "n >= 0 and V >= 1");
    HSN_REQUIRE(V <= HSN_SAMPLE_MAX_TOKENS, HSN_ERR_SIZE_OVERFLOW, "at most 2^18 tokens");
    // a workgroup a row, and a grid's dimension holds fewer than 2^32 threads
    HSN_REQUIRE(n < (int64_t(1) << 32) / kThreads, HSN_ERR_SIZE_OVERFLOW, "fewer than 2^22 rows");
}

}  // namespace
}  // namespace sample
}  // namespace hsn

using namespace hsn;
using namespace hsn::sample;

extern "C" int hsn_sample_workspace(int n, int V, int dtype, int64_t* bytes) {
    HSN_ABI_BEGIN
    check(n, V, dtype);
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    Args a{};
    a.V = V;
    *bytes = layout(a, nullptr, n, dtype == HSN_DTYPE_F32 ? 4 : 2);
    HSN_ABI_END
}

extern "C" int hsn_sample(const void* logits, int64_t row, int dtype, const float* u,
                          const float* temperature, const int32_t* top_k, const float* top_p,
                          const float* min_p, const hsn_sample_settings* settings, int64_t* tokens,
                          int n, int V, void* workspace, int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    check(n, V, dtype);
    if (n == 0) return HSN_OK;
    HSN_REQUIRE(logits && u && tokens, HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    HSN_REQUIRE(settings || (temperature && top_k && top_p && min_p), HSN_ERR_INVALID_ARGUMENT,
                "a setting without an array needs settings");
    Args a{};
    a.logits = logits, a.row = row, a.u = u, a.temperature = temperature, a.top_p = top_p;
    a.min_p = min_p, a.top_k = top_k, a.tokens = tokens, a.V = V;
    if (settings) a.settings = *settings;
    const int64_t bytes = layout(a, static_cast<char*>(workspace), n, dtype == HSN_DTYPE_F32 ? 4 : 2);
    HSN_REQUIRE(!bytes || (workspace && workspace_bytes >= bytes), HSN_ERR_INVALID_ARGUMENT,
                "the workspace is too small");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                "the workspace must be aligned to 16 bytes");
    if (dtype == HSN_DTYPE_F32)
        launch<float>(a, n, as_stream(stream));
    else if (dtype == HSN_DTYPE_F16)
        launch<_Float16>(a, n, as_stream(stream));
    else
        launch<bf16_t>(a, n, as_stream(stream));
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
