// The choice of a token from logits (include/hsn_sample.h): one workgroup a row.
//
// A token's weight is a whole number, so masses can be added in any order: by atomics into
// histogram bins, by lanes, by waves. The order of tokens is the order of score_key(logit), then
// of the token. A row takes these passes over its logits:
//   1. the largest logit and its first token (all that a greedy row needs);
//   2. with top_k or top_p: counts and masses in 2048 bins, linear in x over the range where a
//      weight is not 0 (x > -27.73). They say in which bin each filter cuts. Where the tokens down
//      to that bin are at most 1024 they are gathered into LDS and sorted there, and the row ends
//      without another pass; otherwise the cut is found on the keys' digits (11, 11 and 10 bits),
//      a pass over the row for each;
//   3. the kept weights' sums in the order of tokens, 64 packs of 16 bytes at a time, then one
//      wave's walk through the 64 packs that hold the answer.
#include "../../include/hsn_sample.h"
#include "abi_util.h"
#include "common.cuh"

namespace hsn {
namespace sample {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 2048, kList = 1024;
constexpr float kBinScale = kBins / 27.75f;  // 2^-40 = exp(-27.726)
constexpr float kOne = 1099511627776.0f;     // 2^40
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // score_key(-inf)
constexpr int kChunks = 2 * kThreads;        // sums of 64 packs: 2^18 / (64 * 4) + 1 at most

struct Args {
    const void* logits;
    int64_t row;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    hsn_sample_settings settings;
    int64_t* tokens;
    int V;
};

struct Shared {
    uint64_t mass[kBins];   // bins; then the sums of 64 packs
    uint32_t count[kBins];
    uint64_t list[kList];
    uint64_t wave64[kWaves];
    uint32_t wave32[kWaves];
    uint64_t total64;
    uint32_t total32, n_list, found, found_below;
    uint64_t found_mass;
};
static_assert(kBins == 2 * kThreads && kChunks <= kBins, "two bins a thread");

__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ (static_cast<int32_t>(k) < 0 ? 0x80000000u : 0xffffffffu));
}

// A row's logits as packs of 16 bytes from the last 16-byte boundary at or before its start.
template <typename E>
struct Row {
    static constexpr int kVec = 16 / sizeof(E);
    const E* at;  // of pack 0's first element
    int skip, V, packs;
    __device__ Row(const E* row, int v) : V(v) {
        skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) / sizeof(E)) % kVec);
        at = row - skip;
        packs = (V + skip + kVec - 1) / kVec;
    }
    // The keys of pack p's logits (-inf outside the row; NaN counts as -inf), first token p0.
    __device__ __forceinline__ int keys(int p, uint32_t (&k)[kVec]) const {
        const int first = p * kVec - skip;
        E e[kVec];
        if (first >= 0 && first + kVec <= V) {
            __builtin_memcpy(e, __builtin_assume_aligned(at + int64_t(p) * kVec, 16), 16);
#pragma unroll
            for (int i = 0; i < kVec; ++i) k[i] = key(to_f32(e[i]));
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const bool in = first + i >= 0 && first + i < V;
                k[i] = in ? key(to_f32(at[int64_t(p) * kVec + i])) : kKeyNegInf;
            }
        }
        return first;
    }
    static __device__ __forceinline__ uint32_t key(float l) {
        return l != l ? kKeyNegInf : score_key(l);
    }
};

// The weight of a logit by its key: e, and w as the fixed point of e.
struct Weigh {
    uint32_t best_key;
    float best, t;
    __device__ __forceinline__ float x(uint32_t k) const {
        return k == best_key ? 0.0f : (key_value(k) - best) / t;
    }
    __device__ __forceinline__ float e(uint32_t k) const {
        const float v = k == kKeyNegInf ? 0.0f : expf(x(k));
        return v > 0.0f ? v : 0.0f;  // +inf over an infinite temperature is no share
    }
    static __device__ __forceinline__ uint64_t fixed(float e) {
        return static_cast<uint64_t>(e * kOne);
    }
    __device__ __forceinline__ uint64_t w(uint32_t k) const { return fixed(e(k)); }
};

// Inclusive sum over the workgroup in thread order; `total` the whole. Ends with a barrier passed.
__device__ uint64_t block_scan(uint64_t v, Shared& s, uint64_t& total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    for (int d = 1; d < kWave; d *= 2) {
        const uint64_t o = __shfl_up(static_cast<unsigned long long>(v), d, kWave);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == kWave - 1) s.wave64[wave] = v;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave) before = total;
        total += s.wave64[w];
    }
    return before + v;
}

__device__ uint32_t block_max(uint32_t v, Shared& s) {
    for (int d = 1; d < kWave; d *= 2) v = max(v, wave_shfl_xor(v, d));
    __syncthreads();
    if (threadIdx.x % kWave == 0) s.wave32[threadIdx.x / kWave] = v;
    __syncthreads();
    uint32_t m = 0;
    for (int w = 0; w < kWaves; ++w) m = max(m, s.wave32[w]);
    return m;
}

__device__ void clear_bins(Shared& s) {
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

__device__ Place find_bin(Shared& s, bool by_count, uint64_t k, double target, uint64_t base) {
    const int b = 2 * threadIdx.x;
    const uint64_t m0 = s.mass[b], m1 = s.mass[b + 1];
    const uint32_t c0 = s.count[b], c1 = s.count[b + 1];
    uint64_t mt, ct;
    const uint64_t mi = block_scan(m0 + m1, s, mt), ci = block_scan(c0 + uint64_t(c1), s, ct);
    if (threadIdx.x == 0) s.found = kBins;
    __syncthreads();
    const uint64_t m_at[3] = {mi - m1 - m0, mi - m1, mi};
    const uint64_t c_at[3] = {ci - c1 - c0, ci - c1, ci};
    for (int i = 0; i < 2; ++i) {
        const bool before = by_count ? c_at[i] < k : static_cast<double>(base + m_at[i]) < target;
        const bool after = by_count ? c_at[i + 1] < k
                                    : static_cast<double>(base + m_at[i + 1]) < target;
        if (before && !after && c_at[i + 1] > c_at[i]) {
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
__device__ uint64_t equal_under(uint64_t base, uint64_t w, uint64_t n, double target) {
    const double guess = (target - static_cast<double>(base)) / static_cast<double>(w);
    uint64_t c = guess > 0 ? (guess < double(n) ? static_cast<uint64_t>(guess) : n) : 0;
    while (c < n && static_cast<double>(base + c * w) < target) ++c;
    while (c > 0 && !(static_cast<double>(base + (c - 1) * w) < target)) --c;
    return c;
}

// The cut of one filter, found digit by digit; mass_at: the mass of what it keeps.
template <typename E>
__device__ Cut descend(const Row<E>& row, const Weigh& weigh, Shared& s, bool by_count, uint64_t k,
                       double target, uint64_t& mass_at) {
    uint32_t prefix = 0;
    uint64_t base_mass = 0, base_count = 0;
    const int shifts[4] = {32, 21, 10, 0};
    for (int level = 1; level <= 3; ++level) {
        const int up = shifts[level - 1], shift = shifts[level], bits = up - shift;
        clear_bins(s);
        for (int p = threadIdx.x; p < row.packs; p += kThreads) {
            uint32_t key[Row<E>::kVec];
            row.keys(p, key);
            for (int i = 0; i < Row<E>::kVec; ++i) {
                if (level > 1 && key[i] >> up != prefix) continue;
                const uint64_t w = weigh.w(key[i]);
                if (!w) continue;
                const uint32_t digit = (key[i] >> shift) & ((1u << bits) - 1);
                const uint32_t bin = (1u << bits) - 1 - digit;  // the largest keys first
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[bin]), (unsigned long long)w);
                atomicAdd(&s.count[bin], 1u);
            }
        }
        __syncthreads();
        const Place at = find_bin(s, by_count, by_count ? k - base_count : 0, target, base_mass);
        if (!at.found) {  // the filter keeps everything
            mass_at = base_mass + at.mass_before;
            return {0, 0};
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

// The first token, in order, at which the running sum of f(key, token) exceeds `limit(total)`;
// V where none does.
template <typename E, typename F, typename L>
__device__ int walk(const Row<E>& row, Shared& s, F&& f, L&& limit) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int chunks = (row.packs + kWave - 1) / kWave;
    __syncthreads();
    for (int i = threadIdx.x; i < kChunks; i += kThreads) s.mass[i] = 0;
    if (threadIdx.x == 0) s.found = kChunks;
    __syncthreads();
    auto pack_sum = [&](int p) {
        uint64_t sum = 0;
        if (p < row.packs) {
            uint32_t key[Row<E>::kVec];
            const int first = row.keys(p, key);
            for (int i = 0; i < Row<E>::kVec; ++i) sum += f(key[i], first + i);
        }
        return sum;
    };
    for (int c = wave; c < chunks; c += kWaves) {
        uint64_t sum = pack_sum(c * kWave + lane);
        for (int d = 1; d < kWave; d *= 2)
            sum += __shfl_xor(static_cast<unsigned long long>(sum), d, kWave);
        if (lane == 0) s.mass[c] = sum;
    }
    __syncthreads();
    const uint64_t s0 = s.mass[2 * threadIdx.x], s1 = s.mass[2 * threadIdx.x + 1];
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
        const uint64_t sum = pack_sum(p);
        uint64_t run = sum;
        for (int d = 1; d < kWave; d *= 2) {
            const uint64_t o = __shfl_up(static_cast<unsigned long long>(run), d, kWave);
            if (lane >= d) run += o;
        }
        run += s.found_mass - sum;  // before this pack
        if (run <= r && run + sum > r) {
            uint32_t key[Row<E>::kVec];
            const int first = row.keys(p, key);
            for (int i = 0; i < Row<E>::kVec; ++i) {
                run += f(key[i], first + i);
                if (run > r) {
                    s.found_below = first + i;
                    break;
                }
            }
        }
    }
    __syncthreads();
    return static_cast<int>(s.found_below);
}

// Sorts the first `n` (a power of two up to kList) threads' values, the largest first.
__device__ uint64_t sort_down(uint64_t v, int n, Shared& s) {
    const int i = threadIdx.x;
    for (int k = 2; k <= n; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            uint64_t o;
            if (j < kWave) {
                o = __shfl_xor(static_cast<unsigned long long>(v), j, kWave);
            } else {
                __syncthreads();
                s.list[i] = v;
                __syncthreads();
                o = s.list[i ^ j];
            }
            const bool keep_max = ((i & k) == 0) == ((i & j) == 0);
            if (i < n) v = keep_max ? max(v, o) : min(v, o);
        }
    __syncthreads();
    return v;
}

__device__ __forceinline__ uint64_t at_share(float u, uint64_t total) {
    const double r = floor(static_cast<double>(u) * static_cast<double>(total));
    const uint64_t i = r > 0 ? static_cast<uint64_t>(r) : 0;
    return i < total ? i : total - 1;
}

template <typename E>
__global__ __launch_bounds__(kThreads) void sample_rows(Args a) {
    __shared__ Shared s;
    const int i = blockIdx.x, tid = threadIdx.x;
    const Row<E> row(static_cast<const E*>(a.logits) + i * a.row, a.V);
    constexpr int kVec = Row<E>::kVec;
    const float t = a.temperature ? a.temperature[i] : a.settings.temperature;
    const int top_k = a.top_k ? a.top_k[i] : a.settings.top_k;
    const float top_p = a.top_p ? a.top_p[i] : a.settings.top_p;
    const float min_p = a.min_p ? a.min_p[i] : a.settings.min_p;
    const float u = a.u[i];

    uint32_t best = 0;
    int first = a.V;
    for (int p = tid; p < row.packs; p += kThreads) {
        uint32_t key[kVec];
        const int at = row.keys(p, key);
        for (int j = 0; j < kVec; ++j)
            if (key[j] > best) best = key[j], first = at + j;
    }
    const uint32_t mine = best;
    best = block_max(best, s);
    // the least first token: the largest of its complement
    first = ~block_max(mine == best ? ~static_cast<uint32_t>(first) : 0, s);
    if (best <= kKeyNegInf || !(t > 0)) {
        if (tid == 0) a.tokens[i] = best <= kKeyNegInf ? -1 : first;
        return;
    }
    const Weigh weigh{best, key_value(best), t};

    Cut cut_k{0, 0}, cut_p{0, 0};
    if ((top_k > 0 && top_k < a.V) || !(top_p >= 1.0f)) {
        clear_bins(s);
        for (int p = tid; p < row.packs; p += kThreads) {
            uint32_t key[kVec];
            row.keys(p, key);
            for (int j = 0; j < kVec; ++j) {
                const uint64_t w = weigh.w(key[j]);
                if (!w) continue;
                const int bin = min(kBins - 1, static_cast<int>(-weigh.x(key[j]) * kBinScale));
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[bin]), (unsigned long long)w);
                atomicAdd(&s.count[bin], 1u);
            }
        }
        __syncthreads();
        bool by_count = top_k > 0 && top_k < a.V;
        Place at{};
        if (by_count) {
            at = find_bin(s, true, top_k, 0.0, 0);
            by_count = at.found;  // else fewer tokens than top_k have a weight
        }
        uint64_t total = 0;
        double target = 0.0;
        if (!by_count) {
            block_scan(s.mass[2 * tid] + s.mass[2 * tid + 1], s, total);
            target = static_cast<double>(top_p) * static_cast<double>(total);
            if (!(top_p >= 1.0f)) {
                at = find_bin(s, false, 0, target > 0 ? target : 1.0, 0);
            } else {
                at = Place{};
                at.found = false;
                at.count_before = kList + 1;  // nothing cuts
            }
        }
        const uint32_t n = at.count_before + at.count;
        const bool cuts = by_count || !(top_p >= 1.0f);
        if (cuts && n <= kList) {
            // every token down to the cut's bin, sorted in LDS
            if (tid == 0) s.n_list = 0;
            s.list[tid] = 0;
            __syncthreads();
            const int last = at.found ? at.bin : kBins - 1;
            for (int p = tid; p < row.packs; p += kThreads) {
                uint32_t key[kVec];
                const int at0 = row.keys(p, key);
                for (int j = 0; j < kVec; ++j) {
                    if (key[j] == kKeyNegInf || !weigh.w(key[j])) continue;
                    if (min(kBins - 1, static_cast<int>(-weigh.x(key[j]) * kBinScale)) > last) continue;
                    const uint32_t place = atomicAdd(&s.n_list, 1u);
                    if (place < kList) s.list[place] = uint64_t(key[j]) << 32 | uint32_t(~(at0 + j));
                }
            }
            __syncthreads();
            int size = 1;
            while (size < static_cast<int>(n)) size *= 2;
            uint64_t v = s.list[tid];
            v = sort_down(v, size, s);
            uint32_t key = static_cast<uint32_t>(v >> 32);
            float e = tid < int(n) ? weigh.e(key) : 0.0f;
            uint64_t w = tid < int(n) && (!by_count || tid < top_k) ? Weigh::fixed(e) : 0;
            uint64_t sum;
            const uint64_t run = block_scan(w, s, sum);
            if (by_count) target = static_cast<double>(top_p) * static_cast<double>(sum);
            bool kept = w && (top_p >= 1.0f || static_cast<double>(run - w) < target) && e >= min_p;
            kept |= tid == 0;
            // the kept tokens in their order: the least token is the largest complement
            v = kept ? (v << 32 | v >> 32) : 0;
            v = sort_down(v, size, s);
            key = static_cast<uint32_t>(v);
            w = v && tid < int(n) ? weigh.w(key) : 0;
            const uint64_t end = block_scan(w, s, sum);
            const uint64_t r = at_share(u, sum);
            if (w && end > r && end - w <= r) a.tokens[i] = int64_t(uint32_t(~(v >> 32)));
            return;
        }
        if (by_count) cut_k = descend(row, weigh, s, true, top_k, 0.0, total);
        if (!(top_p >= 1.0f)) {
            uint64_t unused;
            target = static_cast<double>(top_p) * static_cast<double>(total);
            cut_p = descend(row, weigh, s, false, 0, target > 0 ? target : 1.0, unused);
        }
    }
    // the earlier of the two cuts
    Cut cut = cut_k;
    if (cut_p.key > cut.key || (cut_p.key == cut.key && cut_p.equal < cut.equal)) cut = cut_p;
    int last_equal = a.V;
    if (cut.key)
        last_equal = walk(row, s, [&](uint32_t k, int) { return uint64_t(k == cut.key); },
                          [&](uint64_t) { return cut.equal ? cut.equal - 1 : 0; });
    const int token = walk(
        row, s,
        [&](uint32_t k, int j) {
            if (k < cut.key || (k == cut.key && (!cut.equal || j > last_equal))) return uint64_t(0);
            const float e = weigh.e(k);
            return e >= min_p || j == first ? Weigh::fixed(e) : 0;
        },
        [&](uint64_t total) { return at_share(u, total); });
    if (tid == 0) a.tokens[i] = token;
}

}  // namespace
}  // namespace sample
}  // namespace hsn

using namespace hsn;

extern "C" int hsn_sample(const void* logits, int64_t row, int dtype, const float* u,
                          const float* temperature, const int32_t* top_k, const float* top_p,
                          const float* min_p, const hsn_sample_settings* settings, int64_t* tokens,
                          int n, int V, void* stream) {
    HSN_ABI_BEGIN
    HSN_REQUIRE(dtype == HSN_DTYPE_F32 || dtype == HSN_DTYPE_F16 || dtype == HSN_DTYPE_BF16,
                HSN_ERR_UNSUPPORTED_DTYPE, "logits must be F32, F16 or BF16");
    HSN_REQUIRE(n >= 0 && V >= 1, HSN_ERR_INVALID_ARGUMENT, "n >= 0 and V >= 1");
    HSN_REQUIRE(V <= HSN_SAMPLE_MAX_TOKENS, HSN_ERR_SIZE_OVERFLOW, "at most 2^18 tokens");
    if (n == 0) return HSN_OK;
    HSN_REQUIRE(logits && u && tokens, HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    HSN_REQUIRE(settings || (temperature && top_k && top_p && min_p), HSN_ERR_INVALID_ARGUMENT,
                "a setting without an array needs settings");
    sample::Args a{logits, row, u, temperature, top_p, min_p, top_k, {}, tokens, V};
    if (settings) a.settings = *settings;
    hipStream_t st = as_stream(stream);
    if (dtype == HSN_DTYPE_F32)
        sample::sample_rows<float><<<n, sample::kThreads, 0, st>>>(a);
    else if (dtype == HSN_DTYPE_F16)
        sample::sample_rows<_Float16><<<n, sample::kThreads, 0, st>>>(a);
    else
        sample::sample_rows<bf16_t><<<n, sample::kThreads, 0, st>>>(a);
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}
