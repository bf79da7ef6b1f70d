// The global norm of many gradients and clipping by it (include/hsn_clip.h): a launch that sums squares,
// and a launch that scales, each over a list of tensors in its kernel arguments.
//
// The list is one sequence of chunks of 4096 elements. A workgroup takes a run of chunks that lie one
// after the other, so it looks its first tensor up once and steps on from there. Squares are taken and
// summed in float64 (a square of an fp32 number is exact there, and none overflows); every workgroup
// leaves one partial sum, and every workgroup of the second launch adds all of them in the same order
// before it scales, which costs it less than a third launch.
//
// What bounds it is memory: the list is read twice, the second time from the last-level cache where it
// fits, and written once. A run is scaled from its end, which was read last, and long lists are stored past
// the cache: 64 tensors of 4 M fp32 elements take 596 us, 615 from the begin and with ordinary stores.
#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/hsn_clip.h"
#include "abi_util.h"
#include "packs.cuh"

// Allowed to contract, the compiler also joins two narrowings into one, with float64 to fp16 in some
// twenty integer instructions.
#pragma clang fp contract(off)

namespace hsn {
namespace clip {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kChunk = 4096;    // elements
constexpr int kPartials = 2048;  // workgroups over all launches of a pass, at most (but kFewest a launch)
constexpr int kFewest = 32;
constexpr double kEps = 1e-6;

// The tensors of a launch: an address is 48 bits, the elements of the last chunk less one 12 of the next
// ones and the type the highest two, so that 201 tensors of two operands fit the 4 KiB of kernel
// arguments and the usual small model's list is one launch.
template <int ROWS>
struct List {
    static constexpr int kTensors = (4096 - 64) / (8 * ROWS + 4);
    uint64_t at[ROWS][kTensors];
    uint32_t first[kTensors];  // the tensor's first chunk
    int n;
    uint32_t chunks;
    double* partials;  // this launch's (squares), or all of them (scale)
    double* result;
    double max_norm;
    int n_partials;
    bool writes_result, in_place;
};
static_assert(sizeof(List<1>) <= 4096 && sizeof(List<2>) <= 4096, "kernel arguments take 4 KiB");

constexpr uint64_t kAddress = (uint64_t(1) << 48) - 1;

// A workgroup's run of chunks and the tensor it is at; everything is uniform.
template <int ROWS>
struct Walk {
    const List<ROWS>& l;
    uint32_t c, end;
    int t;
    // from the run's first chunk on, or (`backward`) from its last
    __device__ Walk(const List<ROWS>& list, bool backward = false) : l(list) {
        c = static_cast<uint32_t>(uint64_t(blockIdx.x) * l.chunks / gridDim.x);
        end = static_cast<uint32_t>(uint64_t(blockIdx.x + 1) * l.chunks / gridDim.x);
        if (backward) {
            const uint32_t last = end;
            end = c;
            c = last;
        }
        int lo = 0, hi = l.n;  // the last tensor that begins at or before chunk c
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (l.first[mid] <= (backward ? c - 1 : c))
                lo = mid;
            else
                hi = mid;
        }
        t = lo;
    }
    __device__ __forceinline__ bool more() {
        if (c >= end) return false;
        if (t + 1 < l.n && c >= l.first[t + 1]) ++t;  // (no tensor is without a chunk)
        return true;
    }
    __device__ __forceinline__ bool back() {
        if (c <= end) return false;
        if (--c < l.first[t]) --t;
        return true;
    }
    __device__ __forceinline__ int type() const { return static_cast<int>(l.at[0][t] >> 62); }
    __device__ __forceinline__ int count() const {
        const uint32_t next = t + 1 < l.n ? l.first[t + 1] : l.chunks;
        return c + 1 < next ? kChunk : static_cast<int>(l.at[0][t] >> 48 & 0xfff) + 1;
    }
    template <typename E>
    __device__ __forceinline__ E* base(int row) const {
        using Global = __attribute__((address_space(1))) E;  // not a generic address
        return (E*)(Global*)(l.at[row][t] & kAddress) + int64_t(c - l.first[t]) * kChunk;
    }
};

template <typename E>
__device__ __forceinline__ void add_squares(const E* p, int count, double (&sum)[2]) {
    constexpr int kN = Pack<E>::kN, kPacks = kChunk / (kThreads * kN);
    if (count == kChunk) {
        Pack<E> v[kPacks];
#pragma unroll
        for (int i = 0; i < kPacks; ++i) v[i] = load_pack(p + (i * kThreads + threadIdx.x) * kN);
#pragma unroll
        for (int i = 0; i < kPacks; ++i)
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const double g = v[i][j];
                sum[j % 2] = __builtin_fma(g, g, sum[j % 2]);
            }
        return;
    }
    for (int o = threadIdx.x * kN; o < count; o += kThreads * kN) {
        if (o + kN <= count) {
            const Pack<E> v = load_pack(p + o);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const double g = v[j];
                sum[j % 2] = __builtin_fma(g, g, sum[j % 2]);
            }
        } else {
            for (int j = o; j < count; ++j) {
                const double g = to_f32(p[j]);
                sum[0] = __builtin_fma(g, g, sum[0]);
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void squares(const List<1> l) {
    __shared__ double s[kWaves];
    double sum[2] = {0.0, 0.0};
    for (Walk<1> w(l); w.more(); ++w.c) {
        if (w.type() == HSN_DTYPE_F32)
            add_squares(w.base<float>(0), w.count(), sum);
        else if (w.type() == HSN_DTYPE_F16)
            add_squares(w.base<_Float16>(0), w.count(), sum);
        else
            add_squares(w.base<bf16_t>(0), w.count(), sum);
    }
    const double total = block_sum<kWaves>(sum[0] + sum[1], s);
    if (threadIdx.x == 0) l.partials[blockIdx.x] = total;
}

// The product in float64, as the trainer's own clip rounds it; a 16-bit type's from its fp32.
template <typename E>
__device__ __forceinline__ E scaled(float g, double by) {
    return from_f32<E>(static_cast<float>(static_cast<double>(g) * by));
}

template <bool STREAM, typename E>
__device__ __forceinline__ void scale_chunk(const E* p, E* q, int count, double by) {
    constexpr int kN = Pack<E>::kN, kPacks = kChunk / (kThreads * kN);
    if (count == kChunk) {
        Pack<E> v[kPacks];
#pragma unroll
        for (int i = 0; i < kPacks; ++i) v[i] = load_pack(p + (i * kThreads + threadIdx.x) * kN);
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
#pragma unroll
            for (int j = 0; j < kN; ++j) v[i].e[j] = scaled<E>(v[i][j], by);
            store_pack<STREAM>(q + (i * kThreads + threadIdx.x) * kN, v[i]);
        }
        return;
    }
    for (int o = threadIdx.x * kN; o < count; o += kThreads * kN) {
        if (o + kN <= count) {
            Pack<E> v = load_pack(p + o);
#pragma unroll
            for (int j = 0; j < kN; ++j) v.e[j] = scaled<E>(v[j], by);
            store_pack<false>(q + o, v);
        } else {
            for (int j = o; j < count; ++j) q[j] = scaled<E>(to_f32(p[j]), by);
        }
    }
}

// STREAM: what is written goes past the cache.
template <bool STREAM>
__global__ __launch_bounds__(kThreads) void scale(const List<2> l) {
    __shared__ double s[kWaves];
    double sum = 0.0;
    for (int i = threadIdx.x; i < l.n_partials; i += kThreads) sum += l.partials[i];
    const double norm = __builtin_sqrt(block_sum<kWaves>(sum, s));
    double by = l.max_norm / (norm + kEps);
    if (!(by < 1.0) || !(norm < __builtin_inf())) by = 1.0;  // (NaN: 1)
    if (l.writes_result && blockIdx.x == 0 && threadIdx.x == 0) {
        l.result[0] = norm;
        l.result[1] = by;
    }
    if (l.in_place && by == 1.0) return;
    for (Walk<2> w(l, true); w.back();) {
        if (w.type() == HSN_DTYPE_F32)
            scale_chunk<STREAM>(w.base<const float>(0), w.base<float>(1), w.count(), by);
        else if (w.type() == HSN_DTYPE_F16)
            scale_chunk<STREAM>(w.base<const _Float16>(0), w.base<_Float16>(1), w.count(), by);
        else
            scale_chunk<STREAM>(w.base<const bf16_t>(0), w.base<bf16_t>(1), w.count(), by);
    }
}

// ------------------------------------------------------------------------------------------
// The launches of a pass.
// ------------------------------------------------------------------------------------------

constexpr int64_t kMostChunks = (int64_t(1) << 32) - 1;  // of a list

int launches_of(int n, int tensors) { return std::max(1, (n + tensors - 1) / tensors); }
// Workgroups of a launch, of so many.
int grid_of(uint32_t chunks, int launches) {
    return static_cast<int>(std::min<uint32_t>(chunks, std::max(kFewest, kPartials / launches)));
}
int most_partials(int n) {
    const int launches = launches_of(n, List<1>::kTensors);
    return std::max(kPartials, kFewest * launches);
}

template <int ROWS>
void append(List<ROWS>& l, const void* const (&rows)[ROWS], int64_t numel, int dtype) {
    const uint64_t last = static_cast<uint64_t>((numel - 1) % kChunk);
    for (int r = 0; r < ROWS; ++r)
        l.at[r][l.n] = reinterpret_cast<uintptr_t>(rows[r]) | last << 48 | uint64_t(dtype) << 62;
    l.first[l.n++] = l.chunks;
    l.chunks += static_cast<uint32_t>((numel + kChunk - 1) / kChunk);
}

int64_t size_of(int dtype) { return dtype == HSN_DTYPE_F32 ? 4 : 2; }

struct Range {
    uintptr_t from, to;
    int j;
    bool operator<(const Range& o) const { return from < o.from; }
};

// What is written lies apart from everything else, a tensor's own gradient in place aside.
void check_apart(const void* const* grads, void* const* outs, const int64_t* numels, const int* dtypes, int n) {
    std::vector<Range> written;
    written.reserve(n);
    bool sorted = true;
    for (int j = 0; j < n; ++j)
        if (numels[j]) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(outs[j]);
            sorted = sorted && (written.empty() || written.back().from <= at);
            written.push_back({at, at + static_cast<uintptr_t>(numels[j] * size_of(dtypes[j])), j});
        }
    if (written.empty()) return;
    if (!sorted) std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        HSN_REQUIRE(written[i].from >= written[i - 1].to, HSN_ERR_INVALID_ARGUMENT,
                    "tensors " + std::to_string(written[i - 1].j) + " and " + std::to_string(written[i].j) +
                        " to be written overlap");
    const uintptr_t first = written.front().from, last = written.back().to;
    for (int j = 0; j < n; ++j) {
        if (!numels[j] || grads[j] == outs[j]) continue;
        const uintptr_t from = reinterpret_cast<uintptr_t>(grads[j]);
        const uintptr_t to = from + static_cast<uintptr_t>(numels[j] * size_of(dtypes[j]));
        if (to <= first || from >= last) continue;
        auto it = std::lower_bound(written.begin(), written.end(), Range{to, 0, 0});  // begins at or after the end
        HSN_REQUIRE(it == written.begin() || std::prev(it)->to <= from, HSN_ERR_INVALID_ARGUMENT,
                    "a tensor to be written overlaps gradient " + std::to_string(j));
    }
}

}  // namespace
}  // namespace clip
}  // namespace hsn

using namespace hsn;
using namespace hsn::clip;

extern "C" int hsn_clip_workspace(const int64_t* numels, int n, int64_t* bytes) {
    HSN_ABI_BEGIN
    HSN_REQUIRE(n >= 0 && (n == 0 || numels), HSN_ERR_INVALID_ARGUMENT, "bad tensor list");
    HSN_REQUIRE(bytes, HSN_ERR_INVALID_ARGUMENT, "bytes must not be NULL");
    *bytes = 8 * int64_t(most_partials(n));
    HSN_ABI_END
}

extern "C" int hsn_clip(const void* const* grads, void* const* outs, const int64_t* numels, const int* dtypes,
                        int n, double max_norm, double* result, void* workspace, int64_t workspace_bytes,
                        void* stream) {
    HSN_ABI_BEGIN
    HSN_REQUIRE(n >= 0 && (n == 0 || (grads && numels && dtypes)), HSN_ERR_INVALID_ARGUMENT, "bad tensor list");
    HSN_REQUIRE(result && workspace, HSN_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
    HSN_REQUIRE(max_norm >= 0.0, HSN_ERR_INVALID_ARGUMENT, "max_norm >= 0");
    HSN_REQUIRE(workspace_bytes >= 8 * int64_t(most_partials(n)), HSN_ERR_INVALID_ARGUMENT,
                "the workspace is too small");
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, HSN_ERR_INVALID_ARGUMENT,
                "the workspace must be aligned to 8 bytes");
    bool in_place = true;
    int filled = 0;  // tensors with an element
    int64_t chunks = 0, written_bytes = 0;
    for (int j = 0; j < n; ++j) {
        HSN_REQUIRE(dtypes[j] == HSN_DTYPE_F32 || dtypes[j] == HSN_DTYPE_F16 || dtypes[j] == HSN_DTYPE_BF16,
                    HSN_ERR_UNSUPPORTED_DTYPE, "a gradient must be F32, F16 or BF16");
        HSN_REQUIRE(numels[j] >= 0, HSN_ERR_INVALID_ARGUMENT, "a tensor's element count is negative");
        if (!numels[j]) continue;
        const uintptr_t g = reinterpret_cast<uintptr_t>(grads[j]);
        const uintptr_t o = outs ? reinterpret_cast<uintptr_t>(outs[j]) : g;
        HSN_REQUIRE(g && o, HSN_ERR_INVALID_ARGUMENT, "a tensor's address is NULL");
        HSN_REQUIRE((g | o) <= kAddress && (g | o) % size_of(dtypes[j]) == 0, HSN_ERR_INVALID_ARGUMENT,
                    "a tensor's address is not aligned to its type");
        in_place = in_place && g == o;
        chunks += (numels[j] - 1) / kChunk + 1;
        HSN_REQUIRE(chunks <= kMostChunks, HSN_ERR_SIZE_OVERFLOW, "the list has 2^44 elements or more");
        written_bytes += numels[j] * size_of(dtypes[j]);
        ++filled;
    }
    if (outs) check_apart(grads, outs, numels, dtypes, n);
    hipStream_t st = as_stream(stream);
    double* const partials = static_cast<double*>(workspace);
    int n_partials = 0;
    List<1> l;
    l.n = 0, l.chunks = 0;
    const int launches = launches_of(filled, List<1>::kTensors);
    for (int j = 0, left = filled; left; ++j) {
        if (!numels[j]) continue;
        append<1>(l, {grads[j]}, numels[j], dtypes[j]);
        if (--left && l.n < List<1>::kTensors) continue;
        l.partials = partials + n_partials;
        const int grid = grid_of(l.chunks, launches);
        squares<<<grid, kThreads, 0, st>>>(l);
        HSN_HIP(hipGetLastError());
        n_partials += grid;
        l.n = 0, l.chunks = 0;
    }
    List<2> m;
    m.n = 0, m.chunks = 0;
    m.partials = partials, m.n_partials = n_partials, m.max_norm = max_norm, m.result = result;
    m.in_place = in_place && outs;
    m.writes_result = true;
    const auto kernel = outs && written_bytes > kStream ? scale<true> : scale<false>;
    if (!outs || !filled) {
        kernel<<<1, kThreads, 0, st>>>(m);
        HSN_HIP(hipGetLastError());
        return HSN_OK;
    }
    const int writes = launches_of(filled, List<2>::kTensors);
    for (int j = 0, left = filled; left; ++j) {
        if (!numels[j]) continue;
        append<2>(m, {grads[j], outs[j]}, numels[j], dtypes[j]);
        if (--left && m.n < List<2>::kTensors) continue;
        kernel<<<grid_of(m.chunks, writes), kThreads, 0, st>>>(m);
        HSN_HIP(hipGetLastError());
        m.n = 0, m.chunks = 0;
        m.writes_result = false;
    }
    HSN_ABI_END
}
