// The embedding of tokens and its gradient (include/hsn_embed.h).
//
// Forward: a copy of rows. A group of lanes takes a slice of a row, several positions in flight.
//
// Backward: the positions are sorted by token, and then every sum is over neighbours. The sort is by digits
// of up to ten bits from the lowest on, stable, so a token's positions stay in order: a workgroup counts a
// tile's digits, and the next launch ranks the tile's entries (lanes of a wave with the same digit find each
// other by ballots) and adds up where they go from all tiles' counts. Up to 8192 positions need one launch:
// each workgroup counts, for a few entries, what lies before them in the whole list. The sums are taken over
// chunks of the sorted list, one as long as the other, so a token that fills a tenth of the text costs no
// workgroup more than another: a group of lanes walks a chunk with a slice of the columns, writes the rows
// that begin and end inside it, and leaves the sums that cross a border to a last launch, which adds them in
// order. Short lists take one launch, whose workgroups follow their tokens across such borders. Workgroups of
// the sums' launch write the rows that no token names.
//
// What bounds it is memory: the cotangents are read once, the table's gradient is written once.
#include <algorithm>
#include <string>

#include "../../include/hsn_embed.h"
#include "abi_util.h"
#include "packs.cuh"

namespace hsn {
namespace embed {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kDigit = 10, kBins = 1 << kDigit;
constexpr int kSmall = 8192, kSmallThreads = 1024, kSmallWaves = kSmallThreads / kWave;
// Entries that a workgroup of the short sort places (gradients of 8192 x 512 with 8 / 16 / 32: 34.7 / 33.2 / 33.2 us,
// 3063 x 100 17.0 / 16.5 / 17.2; the counts of half the registers, or of all, by vector instructions 34.6 and 35.1).
constexpr int kEntries = 16;
constexpr int kBatch = 8;       // entries of a chunk in flight
constexpr int kCounts = 16;     // tiles' counts in flight
constexpr int kRunThreads = 512, kRunChunk = 128;
constexpr int kZeroRows = 64;   // rows that a workgroup looks through for those without a token

struct Entry {
    uint32_t token;  // V: padding, behind all others
    uint32_t position;
};

struct Args {
    const void* tokens;
    int64_t token_b, token_t;
    bool wide;  // 64-bit tokens
    const void* rows;  // the table, or the cotangents
    int64_t row_b, row_t;
    float scale;
    void* out;
    uint32_t n, T, V;
    int D, slices;  // of 64 packs (or 16) of a row
    // the sort
    const Entry* from;
    Entry* to;
    uint32_t* counts;  // [tiles, kBins]
    int tiles, shift, bits;
    // the sums
    int chunk, chunks, sum_groups;  // sum_groups: workgroups of sums before those that write zeros
    float* parts;  // [chunks, 2, D]: the sum that comes from the chunk before, the one that begins here
};

// Positions' offsets, and their tokens (V: padding). The branches are taken once for all N, so that the loads
// are in flight together: each in a branch of its own, every one waits for the one before.
template <int N>
__device__ __forceinline__ void offsets_of(const Args& a, const uint32_t (&i)[N], int64_t b, int64_t t,
                                           int64_t (&at)[N]) {
    if (a.T == a.n) {
#pragma unroll
        for (int f = 0; f < N; ++f) at[f] = i[f] * t;
    } else {
#pragma unroll
        for (int f = 0; f < N; ++f) {
            const uint32_t r = i[f] / a.T;
            at[f] = r * b + int64_t(i[f] - r * a.T) * t;
        }
    }
}
template <int N>
__device__ __forceinline__ void tokens_of(const Args& a, const uint32_t (&i)[N], uint32_t (&token)[N]) {
    int64_t at[N], raw[N];
    offsets_of(a, i, a.token_b, a.token_t, at);
    if (a.wide) {
#pragma unroll
        for (int f = 0; f < N; ++f) raw[f] = static_cast<const int64_t*>(a.tokens)[at[f]];
    } else {
        int32_t narrow[N];
#pragma unroll
        for (int f = 0; f < N; ++f) narrow[f] = static_cast<const int32_t*>(a.tokens)[at[f]];
#pragma unroll
        for (int f = 0; f < N; ++f) raw[f] = narrow[f];
    }
#pragma unroll
    for (int f = 0; f < N; ++f) token[f] = raw[f] >= 0 && raw[f] < a.V ? static_cast<uint32_t>(raw[f]) : a.V;
}

// A product rounded to fp32, whatever it is rounded to next: left to itself, the compiler takes fp16 products
// by an instruction that rounds once in some places and not in others.
__device__ __forceinline__ float times(float a, float b) {
    float p = a * b;
    asm("" : "+v"(p));
    return p;
}

// F times N elements, and N elements, at any address.
template <typename E, int F, int N>
__device__ __forceinline__ void load_some(const E* p, const int64_t (&at)[F], E (&v)[F][N]) {
#pragma unroll
    for (int f = 0; f < F; ++f) __builtin_memcpy(v[f], p + at[f], sizeof(v[f]));
}
template <typename E, int N>
__device__ __forceinline__ void store_some(E* p, const float (&v)[N]) {
    E e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = from_f32<E>(v[j]);
    __builtin_memcpy(p, e, sizeof(e));
}

// The first of a lane's N columns: a row's last pack ends with the row, and where it overlaps the one before
// both lanes compute and write the same values. (Its elements one by one, each with a branch and a wait of
// its own, took most of a narrow row's time.) Rows of less than a pack have one column a lane.
template <int N>
__device__ __forceinline__ int column_of(int pack, int D) {
    return min(pack * N, D - N);
}

// ------------------------------------------------------------------------------------------
// Forward.
// ------------------------------------------------------------------------------------------

// A group of G lanes a slice of a row (blockIdx.y), several positions in flight.
template <typename E, typename O, int G, int kN>
__global__ __launch_bounds__(kThreads) void gather(const Args a) {
    constexpr int kGroups = kThreads / G, kFlight = 4;
    const int pack = int(blockIdx.y) * G + int(threadIdx.x % G);
    if (pack * kN >= a.D) return;
    const int column = column_of<kN>(pack, a.D);
    const E* table = static_cast<const E*>(a.rows) + column;
    O* out = static_cast<O*>(a.out) + column;
    const uint32_t step = gridDim.x * kGroups;
    for (uint32_t i = blockIdx.x * kGroups + threadIdx.x / G; i < a.n; i += kFlight * step) {
        uint32_t position[kFlight], token[kFlight];
        int64_t at[kFlight];
        E e[kFlight][kN];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) position[f] = min(i + f * step, a.n - 1);
        tokens_of(a, position, token);
#pragma unroll
        for (int f = 0; f < kFlight; ++f) at[f] = min(token[f], a.V - 1) * a.row_t;
        load_some(table, at, e);
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            if (i + f * step >= a.n) break;
            float v[kN];
#pragma unroll
            for (int j = 0; j < kN; ++j) v[j] = token[f] < a.V ? times(to_f32(e[f][j]), a.scale) : 0.0f;
            store_some(out + int64_t(i + f * step) * a.D, v);
        }
    }
}

// ------------------------------------------------------------------------------------------
// The sort.
// ------------------------------------------------------------------------------------------

// Each entry's place among the wave's entries of the same digit, in order; `count` (the wave's, zero
// before) then holds how many of each there are.
template <int N, typename C>
__device__ __forceinline__ void rank_wave(const uint32_t (&digit)[N], int bits, C* count, uint32_t (&rank)[N]) {
#pragma unroll
    for (int r = 0; r < N; ++r) {
        uint64_t same = ~uint64_t(0);
        for (int b = 0; b < bits; ++b) {
            const bool set = digit[r] >> b & 1;
            const uint64_t lanes = ballot(set);
            same &= set ? lanes : ~lanes;
        }
        const uint32_t before = lanes_below(same), base = count[digit[r]];
        rank[r] = base + before;
        wave_order();
        if (before == 0) count[digit[r]] = static_cast<C>(base + __popcll(same));
        wave_order();
    }
}

// Exclusive sum over the workgroup's threads, in their order. `s`: a word a wave.
template <int WAVES>
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t* s) {
    const int lane = lane_id(), wave = threadIdx.x / kWave;
    uint32_t sum = v;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const uint32_t o = __shfl_up(sum, d, kWave);
        sum += lane >= d ? o : 0;
    }
    if (lane == kWave - 1) s[wave] = sum;
    __syncthreads();
    for (int w = 0; w < wave; ++w) sum += s[w];
    return sum - v;
}

// The whole list of up to R 1024 positions in one launch: entry i's place is the number of entries with a
// smaller token and of earlier ones with the same. A wave holds a sixteenth of the list, 64 entries a
// register, and counts for one entry after the other: a comparison of 64 is one vector instruction, its
// ballot's bits are counted by scalar ones. With k' = 2 k + (1 for the entries' own 64 and later ones), k' < 2
// k_i + 1 says k < k_i there and k <= k_i before; what is equal and earlier among the entries' own 64 is
// added by one wave. 8192 entries take 10 us, where two digits by two launches each took 24; the scalar
// counts bound it, and 16384 take longer (26) than by digits.
template <int R>
__global__ __launch_bounds__(kSmallThreads) void sort_small(const Args a) {
    __shared__ int counts[kSmallWaves][kWave];
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id();
    const uint32_t first = blockIdx.x * kEntries, own = first / kWave;
    // the list; then the lane's entry (of the first kEntries lanes) and the lane's of the entries' own 64
    uint32_t at[R + 2], key[R + 2];
    const uint32_t mine = first + lane, beside = own * kWave + lane;
#pragma unroll
    for (int r = 0; r < R; ++r) at[r] = min((wave * R + r) * kWave + lane, a.n - 1);
    at[R] = min(mine, a.n - 1), at[R + 1] = min(beside, a.n - 1);
    tokens_of(a, at, key);
    const uint32_t token = key[R], near = beside < a.n ? key[R + 1] : ~0u;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t block = wave * R + r;
        key[r] = 2 * (block * kWave + lane < a.n ? key[r] : 1u << 30) + (block >= own ? 1 : 0);
    }
    int count = 0;
    for (int i = 0; i < kEntries; ++i) {
        const uint32_t t = readlane(token, i);
        int c = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) c += __popcll(ballot(key[r] < 2 * t + 1));
        if (wave == 0) c += __popcll(ballot(near == t && beside < first + i));
        if (lane == i) count = c;
    }
    counts[wave][lane] = count;
    __syncthreads();
    if (wave || lane >= kEntries || mine >= a.n) return;
    for (int w = 1; w < kSmallWaves; ++w) count += counts[w][lane];
    a.to[count] = {token, mine};
}

// Entries before this pass: the first one reads the tokens.
template <int N>
__device__ __forceinline__ void entries_of(const Args& a, const uint32_t (&i)[N], Entry (&e)[N]) {
    if (a.from) {
#pragma unroll
        for (int r = 0; r < N; ++r) e[r] = a.from[i[r]];
    } else {
        uint32_t token[N];
        tokens_of(a, i, token);
#pragma unroll
        for (int r = 0; r < N; ++r) e[r] = {token[r], i[r]};
    }
}

template <int ITEMS>
__global__ __launch_bounds__(kThreads) void count_digits(const Args a) {
    __shared__ uint32_t count[kBins];
    for (int b = threadIdx.x; b < kBins; b += kThreads) count[b] = 0;
    const uint32_t begin = blockIdx.x * (kThreads * ITEMS), mask = (1u << a.bits) - 1;
    uint32_t i[ITEMS];
    Entry e[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) i[r] = min(begin + r * kThreads + threadIdx.x, a.n - 1);
    entries_of(a, i, e);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (begin + r * kThreads + threadIdx.x < a.n) atomicAdd(&count[e[r].token >> a.shift & mask], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) a.counts[int64_t(blockIdx.x) * kBins + b] = count[b];
}

template <int ITEMS>
__global__ __launch_bounds__(kThreads) void move_entries(const Args a) {
    constexpr int kMine = kBins / kThreads;
    __shared__ uint32_t count[kWaves][kBins];
    __shared__ uint32_t s[kWaves];
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id();
    for (int b = threadIdx.x; b < kWaves * kBins; b += kThreads) (&count[0][0])[b] = 0;
    const uint32_t begin = blockIdx.x * (kThreads * ITEMS) + wave * (kWave * ITEMS) + lane;
    Entry e[ITEMS];
    uint32_t digit[ITEMS], rank[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) rank[r] = min(begin + r * kWave, a.n - 1);
    entries_of(a, rank, e);
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {  // what is behind the end is not moved, and behind all others
        digit[r] = (begin + r * kWave < a.n ? e[r].token : ~0u) >> a.shift & ((1u << a.bits) - 1);
    }
    // where a digit's entries of this tile begin: all entries of lower digits, those of earlier tiles
    uint32_t total[kMine] = {}, earlier[kMine] = {}, all = 0;
    const uint32_t first = threadIdx.x * kMine;
    for (int t0 = 0; t0 < a.tiles; t0 += kCounts) {
        uint4 c[kCounts];
#pragma unroll
        for (int f = 0; f < kCounts; ++f)
            c[f] = *reinterpret_cast<const uint4*>(a.counts + int64_t(min(t0 + f, a.tiles - 1)) * kBins + first);
#pragma unroll
        for (int f = 0; f < kCounts; ++f) {
            const uint32_t v[kMine] = {c[f].x, c[f].y, c[f].z, c[f].w};
#pragma unroll
            for (int b = 0; b < kMine; ++b) {
                total[b] += t0 + f < a.tiles ? v[b] : 0;
                earlier[b] += t0 + f < static_cast<int>(blockIdx.x) ? v[b] : 0;
            }
        }
    }
    __syncthreads();
    rank_wave(digit, a.bits, count[wave], rank);
#pragma unroll
    for (int b = 0; b < kMine; ++b) all += total[b];
    uint32_t before = block_before<kWaves>(all, s);  // (passes a barrier: the waves' counts are there)
#pragma unroll
    for (int b = 0; b < kMine; ++b) {
        uint32_t at = before + earlier[b];
        for (int w = 0; w < kWaves; ++w) {
            const uint32_t c = count[w][first + b];
            count[w][first + b] = at;
            at += c;
        }
        before += total[b];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (begin + r * kWave < a.n) a.to[count[wave][digit[r]] + rank[r]] = e[r];
}

// ------------------------------------------------------------------------------------------
// The sums.
// ------------------------------------------------------------------------------------------

// The first entry of the sorted list whose token is at least `token`, by one wave: 64 probes a step.
__device__ __forceinline__ uint32_t first_of(const Args& a, uint32_t token) {
    uint32_t lo = 0, hi = a.n;  // entries before lo are smaller, from hi on not
    while (lo < hi) {
        const uint64_t span = hi - lo;
        const uint32_t probe = lo + static_cast<uint32_t>(span * lane_id() / kWave);
        const uint64_t smaller = ballot(a.from[probe].token < token);  // the lowest lanes
        const int k = __popcll(smaller);
        const uint32_t new_hi = k < kWave ? lo + static_cast<uint32_t>(span * k / kWave) : hi;
        lo = k ? lo + static_cast<uint32_t>(span * (k - 1) / kWave) + 1 : lo;
        hi = new_hi;
    }
    return lo;
}

// Zeros into the rows [first, first + kZeroRows) that no token names. The entries of these rows are read to see which
// do: where 64 neighbouring rows have most of a long list, by one workgroup (2^20 x 8 bf16 over 131072 rows: tokens
// drawn alike 121 us, the lowest the most frequent by 1 / r 485, a single token 1516).
template <typename T, int G, int kN, int THREADS>
__device__ void write_zeros(const Args& a, uint32_t first) {
    __shared__ uint32_t named[2], range[2];
    const int wave = uniform(threadIdx.x / kWave);
    const uint32_t end = min(first + kZeroRows, a.V);
    if (threadIdx.x < 2) named[threadIdx.x] = 0;
    if (wave < 2) {
        const uint32_t at = first_of(a, wave ? end : first);
        if (lane_id() == 0) range[wave] = at;
    }
    __syncthreads();
    for (uint32_t i = range[0] + threadIdx.x; i < range[1]; i += THREADS) {
        const uint32_t r = a.from[i].token - first;
        atomicOr(&named[r / 32], 1u << r % 32);
    }
    __syncthreads();
    const float zeros[kN] = {};
    T* out = static_cast<T*>(a.out);
    for (uint32_t v = first + threadIdx.x / G; v < end; v += THREADS / G) {
        if (named[(v - first) / 32] >> (v - first) % 32 & 1) continue;
        for (int pack = threadIdx.x % G; pack * kN < a.D; pack += G)
            store_some(out + int64_t(v) * a.D + column_of<kN>(pack, a.D), zeros);
    }
}

// Columns of a lane that writes zeros: 16 bytes, and no more than a lane of sums has.
template <typename T, int N>
constexpr int zeros_of() {
    return N < 16 / int(sizeof(T)) ? N : 16 / int(sizeof(T));
}

// A short list's sums in one launch: a workgroup takes the runs (a token's entries) that begin among its 128
// entries, each to its end, and a slice of 16 packs of the columns. Its 32 groups of 16 lanes share the entries
// evenly; what crosses two groups meets in LDS and is added in order by the group where the run begins. Bf16
// gradients by this launch / by chunks and joins, of tokens drawn alike, by 1 / r, and all the same (us): 64 x 2048
// 9.4 / 12.6, 9.5 / 13.5, 12.8 / 13.8; 8192 x 512 15 / 19, 22 / 24, 52 / 65; but 8192 x 4096 36 / 34, 36 / 34, 62 /
// 47, as one workgroup a slice reads a run, so beyond 2^24 elements the chunks do it.
template <typename E, typename T, int kN>
__global__ __launch_bounds__(kRunThreads) void sum_runs(const Args a) {
    constexpr int G = 16, kGroups = kRunThreads / G;
    __shared__ float parts[kGroups][G * kN];  // the sum that comes from the group before
    __shared__ bool comes_in[kGroups], through[kGroups];  // whether a group has one; whether it is all it has
    __shared__ uint32_t range[2];
    if (static_cast<int>(blockIdx.x) >= a.sum_groups) {
        write_zeros<T, G, zeros_of<T, kN>(), kRunThreads>(a, (blockIdx.x - a.sum_groups) * kZeroRows);
        return;
    }
    const int chunk = blockIdx.x / a.slices, lane = lane_id(), group = threadIdx.x / G, sub = threadIdx.x % G;
    const uint32_t begin = static_cast<uint32_t>(chunk) * kRunChunk, end = min(begin + kRunChunk, a.n);
    if (threadIdx.x < kWave) {
        const uint32_t before = begin ? a.from[begin - 1].token : ~0u;
        const uint32_t last = a.from[end - 1].token, after = a.from[min(end, a.n - 1)].token;
        uint32_t from = begin;  // the first entry that does not continue an earlier run
#pragma unroll
        for (int i = 0; i < kRunChunk; i += kWave) {
            const uint32_t at = min(begin + i + lane, end - 1);
            const uint64_t same = ballot(a.from[at].token == before);
            if (from == begin + i) from += ~same ? __builtin_ctzll(~same) : kWave;
        }
        uint32_t to = end;
        if (from < end && end < a.n && after == last && last < a.V) to = first_of(a, last + 1);
        if (lane == 0) range[0] = from, range[1] = from < end ? to : from;
    }
    __syncthreads();
    const uint32_t from = range[0], to = range[1], each = (to - from + kGroups - 1) / kGroups;
    const uint32_t mine = min(from + group * each, to), mine_end = min(mine + each, to);
    const int pack = (blockIdx.x - chunk * a.slices) * G + sub;
    const bool there = pack * kN < a.D;
    const int column = there ? column_of<kN>(pack, a.D) : 0;
    const E* d_out = static_cast<const E*>(a.rows) + column;
    T* out = static_cast<T*>(a.out) + column;
    float sum[kN] = {};
    uint32_t token = a.V;
    bool comes = false, goes = false, one = true;
    const auto write = [&] {
        float v[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] = times(sum[j], a.scale);
        if (there) store_some(out + int64_t(token) * a.D, v);
    };
    const auto keep = [&] {
#pragma unroll
        for (int j = 0; j < kN; ++j) parts[group][sub * kN + j] = sum[j];
    };
    if (mine < mine_end) {
        token = a.from[mine].token;
        comes = mine > from && a.from[mine - 1].token == token;
        const uint32_t after = mine_end < to ? a.from[mine_end].token : ~0u;
        for (uint32_t i = mine; i < mine_end; i += kBatch) {
            uint32_t tokens[kBatch], position[kBatch];
            int64_t at[kBatch];
            E v[kBatch][kN];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const Entry e = a.from[min(i + b, mine_end - 1)];
                tokens[b] = e.token, position[b] = e.position;
            }
            offsets_of(a, position, a.row_b, a.row_t, at);
            load_some(d_out, at, v);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (i + b >= mine_end) break;
                if (tokens[b] != token) {
                    if (comes && one)
                        keep();
                    else if (token < a.V)
                        write();
                    one = false;
                    token = tokens[b];
#pragma unroll
                    for (int j = 0; j < kN; ++j) sum[j] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < kN; ++j) sum[j] += to_f32(v[b][j]);
            }
        }
        goes = token == after && token < a.V;
        if (comes && one)
            keep();
        else if (!goes && token < a.V)
            write();
    }
    if (sub == 0) comes_in[group] = comes, through[group] = comes && one && goes;
    __syncthreads();
    if (!goes || (comes && one)) return;  // a run that begins here goes on
    for (int g = group + 1; g < kGroups && comes_in[g]; ++g) {
#pragma unroll
        for (int j = 0; j < kN; ++j) sum[j] += parts[g][sub * kN + j];
        if (!through[g]) break;
    }
    write();
}

// A group of G lanes a chunk of the sorted list and a slice of the columns.
template <typename E, typename T, int G, int kN>
__global__ __launch_bounds__(kThreads) void sum_chunks(const Args a) {
    if (static_cast<int>(blockIdx.x) >= a.sum_groups) {
        write_zeros<T, G, zeros_of<T, kN>(), kThreads>(a, (blockIdx.x - a.sum_groups) * kZeroRows);
        return;
    }
    const int unit = blockIdx.x * (kThreads / G) + threadIdx.x / G;
    const int chunk = unit / a.slices;
    const int pack = (unit - chunk * a.slices) * G + int(threadIdx.x % G);
    if (chunk >= a.chunks || pack * kN >= a.D) return;
    const int column = column_of<kN>(pack, a.D);
    const E* d_out = static_cast<const E*>(a.rows) + column;
    T* out = static_cast<T*>(a.out) + column;
    const uint32_t begin = static_cast<uint32_t>(chunk) * a.chunk, end = min(begin + a.chunk, a.n);
    const uint32_t before = begin ? a.from[begin - 1].token : ~0u, after = end < a.n ? a.from[end].token : ~0u;
    float sum[kN] = {};
    uint32_t token = a.from[begin].token;
    bool comes = token == before;  // the sum began in an earlier chunk
    const auto leave = [&](bool goes) {
        if (token >= a.V) return;
        if (comes || goes) {
            store_some(a.parts + (int64_t(chunk) * 2 + (comes ? 0 : 1)) * a.D + column, sum);
            return;
        }
        float v[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] = times(sum[j], a.scale);
        store_some(out + int64_t(token) * a.D, v);
    };
    for (uint32_t i = begin; i < end; i += kBatch) {
        uint32_t tokens[kBatch], position[kBatch];
        int64_t at[kBatch];
        E v[kBatch][kN];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const Entry e = a.from[min(i + b, end - 1)];
            tokens[b] = e.token, position[b] = e.position;
        }
        offsets_of(a, position, a.row_b, a.row_t, at);
        load_some(d_out, at, v);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i + b >= end) break;
            if (tokens[b] != token) {
                leave(false);
                token = tokens[b];
                comes = false;
#pragma unroll
                for (int j = 0; j < kN; ++j) sum[j] = 0.0f;
            }
            if (token >= a.V) return;  // padding from here on
#pragma unroll
            for (int j = 0; j < kN; ++j) sum[j] += to_f32(v[b][j]);
        }
    }
    leave(token == after);
}

// The sum that begins in a chunk and goes on behind it, if there is one: a workgroup a slice of 64 packs,
// a quarter of the parts a wave.
template <typename T, int kN>
__global__ __launch_bounds__(kThreads) void join_chunks(const Args a) {
    constexpr int kFlight = 8;
    __shared__ float sums[kWaves][kN][kWave];
    const int chunk = blockIdx.x / a.slices, slice = blockIdx.x - chunk * a.slices;
    const int wave = uniform(threadIdx.x / kWave), lane = lane_id();
    const uint32_t begin = static_cast<uint32_t>(chunk) * a.chunk, end = begin + a.chunk;
    if (end >= a.n) return;
    const uint32_t token = a.from[end].token, last = a.from[end - 1].token;
    const uint32_t before = a.from[begin ? begin - 1 : 0].token;
    if (token >= a.V || last != token) return;
    if (begin && before == token) return;  // (so is its first: it began earlier)
    int parts = 1;  // this chunk's, and those of the chunks that begin with the token
    for (;;) {
        const int64_t at = (int64_t(chunk) + parts + lane) * a.chunk;
        const uint64_t same = ballot(at < a.n && a.from[at < a.n ? at : 0].token == token);
        const int run = ~same ? __builtin_ctzll(~same) : kWave;
        parts += run;
        if (run < kWave) break;
    }
    const int pack = slice * kWave + lane, column = column_of<kN>(pack, a.D);
    const bool there = pack * kN < a.D;
    const int from = static_cast<int>(int64_t(parts) * wave / kWaves);
    const int to = static_cast<int>(int64_t(parts) * (wave + 1) / kWaves);
    float sum[kN] = {};
    if (there) {
        for (int p = from; p < to; p += kFlight) {
            float v[kFlight][kN];
            int64_t at[kFlight];
#pragma unroll
            for (int f = 0; f < kFlight; ++f) {
                const int q = min(p + f, to - 1);
                at[f] = (int64_t(chunk + q) * 2 + (q ? 0 : 1)) * a.D + column;
            }
            load_some(a.parts, at, v);
#pragma unroll
            for (int f = 0; f < kFlight; ++f)
                if (p + f < to)
#pragma unroll
                    for (int j = 0; j < kN; ++j) sum[j] += v[f][j];
        }
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) sums[wave][j][lane] = sum[j];
    __syncthreads();
    if (wave || !there) return;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        for (int w = 1; w < kWaves; ++w) sum[j] += sums[w][j][lane];
        sum[j] = times(sum[j], a.scale);
    }
    store_some(static_cast<T*>(a.out) + int64_t(token) * a.D + column, sum);
}

// ------------------------------------------------------------------------------------------
// Launches.
// ------------------------------------------------------------------------------------------

int size_of(int dtype) { return dtype == HSN_DTYPE_F32 ? 4 : 2; }
// A lane's columns: 16 bytes of a row's type, or one column of rows that have less.
int columns_of(int D, int dtype) { return D * size_of(dtype) < 16 ? 1 : 16 / size_of(dtype); }
int packs_of(int D, int dtype) { return (D + columns_of(D, dtype) - 1) / columns_of(D, dtype); }
int lanes_of(int D, int dtype) { return packs_of(D, dtype) <= 16 ? 16 : kWave; }

void check(int B, int T, int V, int D, int dtype, int other) {
    for (int t : {dtype, other})
        HSN_REQUIRE(t == HSN_DTYPE_F32 || t == HSN_DTYPE_F16 || t == HSN_DTYPE_BF16, HSN_ERR_UNSUPPORTED_DTYPE,
                    "rows must be F32, F16 or BF16");
    HSN_REQUIRE(B >= 0 && T >= 0 && V >= 1 && D >= 1, HSN_ERR_INVALID_ARGUMENT,
                "B >= 0, T >= 0, V >= 1 and D >= 1");
    HSN_REQUIRE(V <= HSN_EMBED_MAX_TOKENS && D <= HSN_EMBED_MAX_WIDTH, HSN_ERR_SIZE_OVERFLOW,
                "V at most 2^24 and D at most 65536");
    HSN_REQUIRE(int64_t(B) * T < 1 << 26, HSN_ERR_SIZE_OVERFLOW, "fewer than 2^26 tokens");
}

void check_rows(const void* p, int dtype, const char* name) {
    HSN_REQUIRE(p && reinterpret_cast<uintptr_t>(p) % size_of(dtype) == 0, HSN_ERR_INVALID_ARGUMENT,
                std::string(name) + " must be there and aligned to its type");
}

// One row of positions where the strides allow it.
void set_tokens(Args& a, const void* tokens, int64_t b, int64_t t, int bytes, int B, int T) {
    HSN_REQUIRE(tokens, HSN_ERR_INVALID_ARGUMENT, "tokens is NULL");
    HSN_REQUIRE(bytes == 8 || bytes == 4, HSN_ERR_INVALID_ARGUMENT, "token_bytes is 8 or 4");
    a.tokens = tokens, a.token_b = b, a.token_t = t, a.wide = bytes == 8;
    a.n = static_cast<uint32_t>(B) * T, a.T = T;
    if (B == 1 || (b == T * t && a.row_b == T * a.row_t)) {
        a.T = a.n;
    } else if (T == 1) {
        a.token_t = b, a.row_t = a.row_b, a.T = a.n;
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

// Chunks of the sorted list: as long as leaves some 2048 waves to fill the GPU, 8 entries (one
// batch of loads) at least (32768 x 2048 bf16 both ways with 4096 / 2048 / 1024 / 512 waves: 209 / 202 / 210 / 241
// us; shorter lists do not care).
int chunk_of(int64_t n, int D, int dtype) {
    const int lanes = lanes_of(D, dtype);
    const int64_t slices = (packs_of(D, dtype) + lanes - 1) / lanes;
    const int64_t groups = 2048 * (kWave / lanes);
    int chunk = kBatch;
    while (chunk < 1024 && n * slices > groups * chunk) chunk *= 2;
    return chunk;
}

// Entries a tile, of 256 threads: small tiles leave more workgroups for a short list, but the next launch reads
// all tiles' counts in every workgroup (gradients of n x 8 bf16 with 4 / 8 / 32 entries a thread: 20000 28 / 30 / 56
// us, 65536 39 / 39 / 64, 200000 63 / 57 / 75, 400000 108 / 76 / 87, 1000000 343 / 148 / 114). That reading grows with
// the square of the positions: 2^22 take 0.30 ms, 2^24 2.0 and 2^26 - 1, the most, 21 (by tokens drawn alike).
int items_of(int64_t n) { return n <= 1 << 16 ? 4 : n <= 1 << 19 ? 8 : 32; }

// Whether the sums are one launch's.
bool by_runs(int64_t n, int D) { return n <= kSmall && n * D <= 1 << 24; }

struct Workspace {
    Entry *a, *b;
    uint32_t* counts;
    float* parts;
    int64_t bytes;
};

Workspace layout(char* at, int64_t n, int D, int dtype) {
    char* const begin = at;
    const auto take = [&](int64_t bytes) {
        char* p = at;
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    Workspace w;
    const bool small = n <= kSmall;
    const int64_t tile = kThreads * items_of(n), chunk = chunk_of(n, D, dtype);
    w.a = reinterpret_cast<Entry*>(take(8 * n));
    w.b = reinterpret_cast<Entry*>(take(small ? 0 : 8 * n));
    w.counts = reinterpret_cast<uint32_t*>(take(small ? 0 : (n + tile - 1) / tile * kBins * 4));
    w.parts = reinterpret_cast<float*>(take(by_runs(n, D) ? 0 : (n + chunk - 1) / chunk * 2 * D * 4));
    w.bytes = std::max<int64_t>(16, at - begin);
    return w;
}

// The entries in the order of their tokens; returns where they are.
const Entry* sort(Args a, const Workspace& w, hipStream_t st) {
    int bits = 1;
    while (a.V >> bits) ++bits;  // padding is V
    if (a.n <= kSmall) {
        a.to = w.a;
        const int grid = (a.n + kEntries - 1) / kEntries;
        const int held = (a.n + kSmallThreads - 1) / kSmallThreads;
        (held <= 1   ? sort_small<1>
         : held <= 2 ? sort_small<2>
         : held <= 4 ? sort_small<4>
                     : sort_small<8>)<<<grid, kSmallThreads, 0, st>>>(a);
        HSN_HIP(hipGetLastError());
        return w.a;
    }
    const int passes = (bits + kDigit - 1) / kDigit;
    const int items = items_of(a.n);
    a.tiles = static_cast<int>((a.n + kThreads * items - 1) / (kThreads * items));
    a.counts = w.counts;
    a.bits = (bits + passes - 1) / passes;
    for (int p = 0; p < passes; ++p) {
        a.shift = p * a.bits;
        a.to = p % 2 ? w.b : w.a;
        (items == 4   ? count_digits<4>
         : items == 8 ? count_digits<8>
                      : count_digits<32>)<<<a.tiles, kThreads, 0, st>>>(a);
        HSN_HIP(hipGetLastError());
        (items == 4   ? move_entries<4>
         : items == 8 ? move_entries<8>
                      : move_entries<32>)<<<a.tiles, kThreads, 0, st>>>(a);
        HSN_HIP(hipGetLastError());
        a.from = a.to;
    }
    return a.from;
}

// A grid's dimension holds fewer than 2^32 threads.
int grid_of(int64_t groups, int threads) {
    HSN_REQUIRE(groups < (int64_t(1) << 32) / threads, HSN_ERR_SIZE_OVERFLOW,
                "more workgroups than one grid holds");
    return static_cast<int>(groups);
}

}  // namespace
}  // namespace embed
}  // namespace hsn

using namespace hsn;
using namespace hsn::embed;

extern "C" int hsn_embed_forward(const void* tokens, int64_t token_b, int64_t token_t, int token_bytes,
                                 const void* table, int64_t table_row, int table_dtype, float scale, void* out,
                                 int out_dtype, int B, int T, int V, int D, void* stream) {
    HSN_ABI_BEGIN
    check(B, T, V, D, table_dtype, out_dtype);
    if (B == 0 || T == 0) return HSN_OK;
    check_rows(table, table_dtype, "table");
    check_rows(out, out_dtype, "out");
    Args a{};
    a.rows = table, a.scale = scale, a.out = out, a.V = V, a.D = D;
    set_tokens(a, tokens, token_b, token_t, token_bytes, B, T);
    a.row_t = table_row;
    hipStream_t st = as_stream(stream);
    with_type(table_dtype, [&](auto e) {
        with_type(out_dtype, [&](auto o) {
            using E = decltype(e);
            using O = decltype(o);
            const int packs = packs_of(D, table_dtype);
            const int lanes = packs <= 16 ? 16 : packs <= kWave ? kWave : kThreads, groups = kThreads / lanes;
            a.slices = (packs + lanes - 1) / lanes;
            // some 4096 workgroups: 16 a compute unit
            const int most = std::max(1, 4096 / a.slices);
            const dim3 grid(std::min<int>((a.n + groups - 1) / groups, most), a.slices);
            constexpr int kN = 16 / sizeof(E);
            (columns_of(D, table_dtype) == 1 ? gather<E, O, 16, 1>
             : lanes == 16                   ? gather<E, O, 16, kN>
             : lanes == kWave                ? gather<E, O, kWave, kN>
                                             : gather<E, O, kThreads, kN>)<<<grid, kThreads, 0, st>>>(a);
        });
    });
    HSN_HIP(hipGetLastError());
    HSN_ABI_END
}

extern "C" int hsn_embed_workspace(int B, int T, int V, int D, int d_out_dtype, int64_t* bytes) {
    HSN_ABI_BEGIN
    check(B, T, V, D, d_out_dtype, d_out_dtype);
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    *bytes = layout(nullptr, int64_t(B) * T, D, d_out_dtype).bytes;
    HSN_ABI_END
}

extern "C" int hsn_embed_backward(const void* tokens, int64_t token_b, int64_t token_t, int token_bytes,
                                  const void* d_out, int64_t d_out_b, int64_t d_out_t, int d_out_dtype,
                                  float scale, void* d_table, int table_dtype, int B, int T, int V, int D,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
    HSN_ABI_BEGIN
    check(B, T, V, D, d_out_dtype, table_dtype);
    check_rows(d_table, table_dtype, "d_table");
    HSN_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                "the workspace must be there and aligned to 16 bytes");
    Args a{};
    a.scale = scale, a.out = d_table, a.V = V, a.D = D;
    const int64_t n = int64_t(B) * T;
    if (n) {
        check_rows(d_out, d_out_dtype, "d_out");
        a.rows = d_out, a.row_b = d_out_b, a.row_t = d_out_t;
        set_tokens(a, tokens, token_b, token_t, token_bytes, B, T);
    }
    const Workspace w = layout(static_cast<char*>(workspace), n, D, d_out_dtype);
    HSN_REQUIRE(workspace_bytes >= w.bytes, HSN_ERR_INVALID_ARGUMENT, "the workspace is too small");
    const bool small = by_runs(n, D), narrow = columns_of(D, d_out_dtype) == 1;
    const int packs = packs_of(D, d_out_dtype), lanes = small ? 16 : lanes_of(D, d_out_dtype);
    a.slices = (packs + lanes - 1) / lanes;
    a.chunk = small ? kRunChunk : chunk_of(n, D, d_out_dtype);
    a.chunks = static_cast<int>((n + a.chunk - 1) / a.chunk);
    const int groups = small ? 1 : kThreads / lanes;  // of a workgroup, a chunk's slice each
    const int64_t units = int64_t(a.chunks) * a.slices, zeros = (V + kZeroRows - 1) / kZeroRows;
    const int grid = grid_of((units + groups - 1) / groups + zeros, small ? kRunThreads : kThreads);
    const int joins = small || a.chunks < 2 ? 0 : grid_of(int64_t(a.chunks) * ((packs + kWave - 1) / kWave), kThreads);
    a.sum_groups = grid - static_cast<int>(zeros);
    a.parts = w.parts;
    hipStream_t st = as_stream(stream);
    if (n) a.from = sort(a, w, st);
    with_type(d_out_dtype, [&](auto e) {
        with_type(table_dtype, [&](auto t) {
            using E = decltype(e);
            using T_ = decltype(t);
            constexpr int kN = 16 / sizeof(E);
            if (small) {
                (narrow ? sum_runs<E, T_, 1> : sum_runs<E, T_, kN>)<<<grid, kRunThreads, 0, st>>>(a);
                HSN_HIP(hipGetLastError());
                return;
            }
            (narrow        ? sum_chunks<E, T_, 16, 1>
             : lanes == 16 ? sum_chunks<E, T_, 16, kN>
                           : sum_chunks<E, T_, kWave, kN>)<<<grid, kThreads, 0, st>>>(a);
            HSN_HIP(hipGetLastError());
            if (!joins) return;
            Args j = a;
            j.slices = (packs + kWave - 1) / kWave;
            (narrow ? join_chunks<T_, 1> : join_chunks<T_, kN>)<<<joins, kThreads, 0, st>>>(j);
            HSN_HIP(hipGetLastError());
        });
    });
    HSN_ABI_END
}
