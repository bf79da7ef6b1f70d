// A whole layer of routed units for a few tokens (include/hsn_units_layer.h).
//
//   route    (token, four units): the router's products, a wave a unit.
//   choose   (token): the K units; where the tokens are few, in the first product instead.
//   product  (column tile and split of the rows, slot): z = x W1[e] for the tokens that chose the
//            slot's unit e, as fp32 sums of the split's rows.
//   product  the same for v W2[e], where v is made from the first product's sums on the way.
//   combine  (token, 64 columns): the weighted sum over the token's units, in a fixed order.
//
// What bounds it is one read of the chosen units' weights, so the products stream them from HBM into
// registers once, 16 bytes a lane, as they lie ([in, out]), and give them to the matrix cores with up
// to 16 tokens as the other operand. A wave takes 32 rows and 16 lanes' columns a step, lane group g =
// lane / 16 the rows 8 g .. 8 g + 7: eight loads of one row each. In 16-bit storage a lane then
// holds 8 columns of 8 consecutive rows; byte permutes pair neighbouring rows into the operands of 8
// products 16x16x32, the m-th with the columns c0 + m of the lanes. Rows are split over a workgroup's
// waves and, where units and column tiles are few, over workgroups, so that some 512 workgroups
// keep the loads of two steps each in flight.
// One token, 8 of 64 gated units of 2048 x 1024 in bf16: 35 us, the products 16.1 and 11.8 (4.2 and 2.8
// TB/s); 256 workgroups a product are as fast, 1024 take 40 us, and 48 with one step a wave. 32 such
// tokens: 175 us, the products 100 and 61 (5.3 and 4.3 TB/s). One launch for both products and the
// sum, its workgroups waiting for one another through memory, measured 35 to 37 us against 34.4 for the one
// token, 13.1 against 16.0 for one of 2 of 8 units of 256 x 512 in fp32, and 31.3 against 33.4 for 5 tokens of
// 3 of 12 units of 999 x 1234 in fp16; where it would begin to lose is not measured, and no rule takes it.
//
// x enters the first product exactly, and so does v the second. v is fp32: 16-bit weights multiply it on
// the 16-bit matrix cores as the sum of three bf16 (8 bits each, all 24 of v's; two would lose up to 2^-16
// of v, which shows in bf16 results as a rounding the other way here and there), fp16 weights as two bf16
// themselves (8 and 3 of their 11 bits), since fp16 has not the range of an unscaled v and fp32 products
// of widened weights take four times the matrix cores' time. A value's parts have its sign and none is 0
// unless the value is (2^-126 stands in for a part without bits), so that an infinity on either side gives
// an infinity and not a NaN. A workgroup makes v for its rows in LDS, 512 rows at a time, with the
// first weights in flight.
#include <algorithm>
#include <type_traits>

#include "../../include/hsn_units_layer.h"
#include "abi_util.h"
#include "common.cuh"
#include "unit_math.cuh"

namespace hsn {
namespace units_layer {
namespace {

constexpr int kMaxUnits = HSN_UNITS_MAX, kMaxChosen = HSN_UNITS_MAX_CHOSEN;
constexpr int kMaxTokens = HSN_UNITS_MAX_TOKENS;
constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kRows = 32;    // rows of a step
constexpr int kTokens = 16;  // tokens of a product
constexpr int kStage = 512;  // rows of v in LDS

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// One of the two products: [pairs, rows] times [M, rows, cols] by the pairs' units.
struct Product {
    const void* W;
    float* sums;  // [splits, pairs, cols]
    int rows, cols, tiles, splits, split_rows;
};

struct Args {
    const void *x, *router, *b1, *b2;
    void* y;
    int64_t x_row;
    float* logit;  // [n, M]
    int* unit;     // [n, K] the choice
    float* share;  // [n, K]
    Product up, down;
    int n, M, K, d_in, H, d_out, activation;
    bool choose_inline;  // the first product chooses
};

// 16 bytes from any element's address (one load; the GPU takes global addresses unaligned).
template <typename E>
__device__ __forceinline__ v4u load16(const E* p) {
    v4u r;
    __builtin_memcpy(&r, p, 16);
    return r;
}

// --------------------------------------------------------------------------------------------
// The router.
// --------------------------------------------------------------------------------------------

// The units of up to kThreads / M tokens from their products, a thread a unit of a token: a unit's rank
// is the number of units before it (larger, or equal and lower), and the first K are chosen. Every
// thread of the workgroup calls it; `units` and `shares` (LDS) get [tokens, K].
struct ChoiceLds {
    uint32_t key[kThreads + 4];
    float logit[kThreads];
    int unit[kThreads];
    float share[kThreads];
};
static_assert(kThreads >= kMaxUnits && kMaxChosen <= 16, "a token's units, a thread each");

__device__ __forceinline__ void choose_units(ChoiceLds& lds, int M, int K, int tokens, float logit) {
    const int tid = threadIdx.x, i = tid / M, m = tid % M;
    const uint32_t key = score_key(logit);
    if (i < tokens) lds.key[tid] = key;
    __syncthreads();
    int rank = 0;
    if (i < tokens) {
        const uint32_t* others = lds.key + i * M;
        int j = 0;
        for (; j + 8 <= M; j += 8) {
            uint32_t other[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) other[k] = others[j + k];
#pragma unroll
            for (int k = 0; k < 8; ++k) rank += other[k] > key || (other[k] == key && j + k < m);
        }
        for (; j < M; ++j) rank += others[j] > key || (others[j] == key && j < m);
    }
    const bool chosen = i < tokens && rank < K;
    if (chosen) lds.unit[i * K + rank] = m, lds.logit[i * K + rank] = logit;
    __syncthreads();
    const int first = tid / K * K;
    if (tid < tokens * K) lds.share[tid] = expf(lds.logit[tid] - lds.logit[first]);
    __syncthreads();
    if (tid < tokens * K) {
        float sum = 0.0f;
        for (int k = 0; k < K; ++k) sum += lds.share[first + k];
        lds.logit[tid] = lds.share[tid] / sum;
    }
    __syncthreads();
    if (tid < tokens * K) lds.share[tid] = lds.logit[tid];
}

// A thread writes what it wrote to LDS.
__device__ __forceinline__ void write_choice(const Args& a, const ChoiceLds& lds, int first_token,
                                             int tokens) {
    const int tid = threadIdx.x;
    if (tid >= tokens * a.K) return;
    a.unit[first_token * a.K + tid] = lds.unit[tid];
    a.share[first_token * a.K + tid] = lds.share[tid];
}

template <typename E>
__global__ __launch_bounds__(kThreads) void route(Args a) {
    constexpr int kVec = 16 / sizeof(E), kStep = kWave * kVec;
    const int i = blockIdx.x, lane = threadIdx.x % kWave;
    const int m = blockIdx.y * kWaves + threadIdx.x / kWave;
    if (m >= a.M) return;
    const E* x = static_cast<const E*>(a.x) + i * a.x_row;
    const E* w = static_cast<const E*>(a.router) + int64_t(m) * a.d_in;
    float sum = 0.0f;
    int k = lane * kVec;
#pragma unroll 4
    for (; k + kVec <= a.d_in; k += kStep) {
        const v4u xv = load16(x + k), wv = load16(w + k);
        E xe[kVec], we[kVec];
        __builtin_memcpy(xe, &xv, 16);
        __builtin_memcpy(we, &wv, 16);
#pragma unroll
        for (int j = 0; j < kVec; ++j) sum = __builtin_fmaf(to_f32(xe[j]), to_f32(we[j]), sum);
    }
    for (; k < a.d_in; ++k)  // the last, incomplete pack is one lane's
        sum = __builtin_fmaf(to_f32(x[k]), to_f32(w[k]), sum);
    for (int d = 1; d < kWave; d *= 2) sum += wave_shfl_xor(sum, d);
    if (lane == 0) a.logit[i * a.M + m] = sum;
}

__global__ __launch_bounds__(kThreads) void choose(Args a) {
    __shared__ ChoiceLds lds;
    const int i = blockIdx.x;
    choose_units(lds, a.M, a.K, 1,
                 int(threadIdx.x) < a.M ? a.logit[i * a.M + threadIdx.x] : 0.0f);
    write_choice(a, lds, i, 1);
}

// --------------------------------------------------------------------------------------------
// The products.
// --------------------------------------------------------------------------------------------

// Eight rows of the left operand: pair's rows k0 + 8 g .. + 7 (0 from `end` on).
template <typename E>
__device__ __forceinline__ void load_x(const Args& a, int pair, int k, int end, E (&to)[8]) {
    const E* x = static_cast<const E*>(a.x) + (pair / a.K) * a.x_row + k;
    if (k + 8 <= end) {
        __builtin_memcpy(to, x, sizeof(to));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) to[j] = k + j < end ? x[j] : from_f32<E>(0.0f);
    }
}

// Eight of a pair's first-product values: the splits' sums, then the bias.
template <typename E>
__device__ __forceinline__ void load_z(const Args& a, int pair, int unit, int col, int count,
                                       float (&z)[8]) {
    const int64_t stride = int64_t(a.n) * a.K * a.up.cols;
    const float* at = a.up.sums + int64_t(pair) * a.up.cols + col;
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = 0.0f;
    for (int s = 0; s < a.up.splits; ++s, at += stride)
        if (count == 8) {
            float v[8];
            __builtin_memcpy(v, at, sizeof(v));
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] += v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < count) z[j] += at[j];
        }
    if (a.b1) {
        const E* b = static_cast<const E*>(a.b1) + int64_t(unit) * a.up.cols + col;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) z[j] += to_f32(b[j]);
    }
}

template <typename E>
__device__ __forceinline__ void load_hidden(const Args& a, int pair, int unit, int k, int end,
                                            float (&v)[8]) {
    const int count = min(8, max(0, end - k));
    float z[8];
    load_z<E>(a, pair, unit, k, count, z);
    if (a.activation == HSN_UNITS_SWIGLU) {
        float g[8];
        load_z<E>(a, pair, unit, a.H + k, count, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = z[j] * act_sigmoid(z[j]) * g[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = units::gelu(z[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < count ? v[j] : 0.0f;
}

__device__ __forceinline__ v4f mfma(v8bf a, v8bf b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(float a, float b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// The upper and the lower halves of two words, as one word.
__device__ __forceinline__ uint32_t upper(uint32_t lo, uint32_t hi) {
    return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
__device__ __forceinline__ uint32_t lower(uint32_t lo, uint32_t hi) {
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// Column m of the lane's eight rows as the eight-row operand of a 16-bit product.
template <typename V8>
__device__ __forceinline__ V8 column(const v4u (&row)[8], int m) {
    v4u r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t even = row[2 * i][m / 2], odd = row[2 * i + 1][m / 2];
        r[i] = m % 2 ? upper(even, odd) : lower(even, odd);
    }
    return __builtin_bit_cast(V8, r);
}

template <typename E>
__device__ __forceinline__ float element(v4u row, int m) {
    E e[16 / sizeof(E)];
    __builtin_memcpy(e, &row, 16);
    return to_f32(e[m]);
}

// The upper 8 significant bits of a value, which are a bf16.
__device__ __forceinline__ float top_bits(float v) {
    return __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}

// What is left of a value after its upper bits, or what stands in for it.
__device__ __forceinline__ float left_bits(float from, float value) {
    const float left = from - top_bits(from);  // NaN of an infinity
    return __builtin_fabsf(left) > 0.0f ? left : __builtin_amdgcn_fmed3f(value, -0x1p-126f, 0x1p-126f);
}

// Column m of fp16 rows as two bf16 operands: the upper 8 bits of each and the rest.
__device__ __forceinline__ void column_halves(const v4u (&row)[8], int m, v8bf& hi, v8bf& lo) {
    v4u h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t whole[2], rest[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            whole[k] = __float_as_uint(element<_Float16>(row[2 * i + k], m));
            const float w = __uint_as_float(whole[k]);
            rest[k] = __float_as_uint(left_bits(w, w));
        }
        h[i] = upper(whole[0], whole[1]);
        l[i] = upper(rest[0], rest[1]);
    }
    hi = __builtin_bit_cast(v8bf, h);
    lo = __builtin_bit_cast(v8bf, l);
}

// v in LDS: fp32, or three bf16 with 8 of its bits each, the upper ones first. The rows are padded by
// 16 bytes, so that 16 tokens' packs lie in different banks.
constexpr int kParts = 3;
template <bool kSplit>
struct Hidden {
    float v[kTokens][kStage + 4];
    __device__ __forceinline__ void put(int t, int k, const float (&x)[8]) {
        __builtin_memcpy(&v[t][k], x, sizeof(x));
    }
};
template <>
struct Hidden<true> {
    uint16_t part[kParts][kTokens][kStage + 8];
    __device__ __forceinline__ void put(int t, int k, const float (&x)[8]) {
        float rest[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            v4u pack;
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                pack[j / 2] = upper(__float_as_uint(rest[j]), __float_as_uint(rest[j + 1]));
            __builtin_memcpy(&part[i][t][k], &pack, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) rest[j] = left_bits(rest[j], x[j]);
        }
    }
};

template <typename E, bool kDown>
__global__ __launch_bounds__(kThreads, 2) void product(Args a) {
    constexpr int kCols = 16 / sizeof(E);   // of a lane
    constexpr int kTileCols = 16 * kCols;
    constexpr bool kBf16 = __is_same(E, bf16_t), kF32 = __is_same(E, float);
    __shared__ union {
        float red[kWaves][kTokens][kTileCols];
        Hidden<!kF32> hidden;
        ChoiceLds choice;
    } lds;
    __shared__ uint32_t mask[kMaxUnits / 32];
    __shared__ int list[kMaxTokens], listed;
    const Product& p = kDown ? a.down : a.up;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int pairs = a.n * a.K, slot = blockIdx.y;
    const int* units = a.unit;
    if constexpr (!kDown)
        if (a.choose_inline) {  // every workgroup chooses, the first writes the choice down
            choose_units(lds.choice, a.M, a.K, a.n, tid < a.n * a.M ? a.logit[tid] : 0.0f);
            if (blockIdx.x == 0 && slot == 0) write_choice(a, lds.choice, 0, a.n);
            units = lds.choice.unit;
        }
    // the slot's unit, the slot-th of the chosen ones, and its pairs (at most one a token)
    int unit, count = 1;
    if (a.n == 1) {
        unit = uniform(units[slot]);
        if (tid == 0) list[0] = slot;
        __syncthreads();
    } else {
        if (tid < kMaxUnits / 32) mask[tid] = 0;
        __syncthreads();
        for (int i = tid; i < pairs; i += kThreads) atomicOr(&mask[units[i] / 32], 1u << units[i] % 32);
        __syncthreads();
        unit = -1;
        for (int w = 0, seen = 0; w < kMaxUnits / 32; ++w) {
            uint32_t bits = uniform(mask[w]);
            const int here = __popc(bits);
            if (unit < 0 && seen + here > slot) {
                for (int k = seen; k < slot; ++k) bits &= bits - 1;
                unit = w * 32 + __ffs(bits) - 1;
            }
            seen += here;
        }
        if (unit < 0) return;
        if (wave == 0) {
            int n = 0;
            for (int base = 0; base < pairs; base += kWave) {
                const bool hit = base + lane < pairs && units[base + lane] == unit;
                const uint64_t hits = ballot(hit);
                if (hit) list[n + lanes_below(hits)] = base + lane;
                n += __popcll(hits);
            }
            if (lane == 0) listed = n;
        }
        __syncthreads();
        count = listed;
    }
    const int tile = blockIdx.x % p.tiles, split = blockIdx.x / p.tiles;
    const int begin = split * p.split_rows, end = min(p.rows, begin + p.split_rows);
    const int group = lane / 16, col_lane = lane % 16;
    // a lane's columns end with the row: the last lanes share the last columns
    auto first_col = [&](int l) { return max(0, min(tile * kTileCols + l * kCols, p.cols - kCols)); };
    const E* W = static_cast<const E*>(p.W) + int64_t(unit) * p.rows * p.cols + first_col(col_lane);
    const bool narrow = p.cols < kCols;

    auto load_rows = [&](int k0, v4u (&row)[8]) {
        const int k = k0 + 8 * group;
        const E* at = W + int64_t(k) * p.cols;
        if (k0 + kRows <= end && !narrow) {
#pragma unroll
            for (int j = 0; j < 8; ++j) row[j] = load16(at + int64_t(j) * p.cols);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                E e[kCols];
                row[j] = v4u{};
                if (k + j >= end) continue;
                if (!narrow) {
                    row[j] = load16(at + int64_t(j) * p.cols);
                    continue;
                }
#pragma unroll
                for (int m = 0; m < kCols; ++m)
                    e[m] = m < p.cols ? at[int64_t(j) * p.cols + m] : from_f32<E>(0.0f);
                __builtin_memcpy(&row[j], e, 16);
            }
        }
    };

    for (int t0 = 0; t0 < count; t0 += kTokens) {
        const int here = min(kTokens, count - t0);
        const int pair = list[t0 + min(col_lane, here - 1)];
        int stage = begin;
        v4f acc[kCols];
#pragma unroll
        for (int m = 0; m < kCols; ++m) acc[m] = v4f{};
        auto multiply = [&](int k0, const v4u (&row)[8]) {
            const int k = k0 + 8 * group, t = min(col_lane, here - 1);
            if constexpr (kF32) {
                float left[8];
                if constexpr (kDown)
                    __builtin_memcpy(left, &lds.hidden.v[t][k - stage], sizeof(left));
                else
                    load_x<E>(a, pair, k, end, left);
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int m = 0; m < kCols; ++m)
                        acc[m] = mfma(left[j], element<E>(row[j], m), acc[m]);
            } else if constexpr (kDown) {
                v8bf v[kParts];
#pragma unroll
                for (int i = 0; i < kParts; ++i)
                    __builtin_memcpy(&v[i], &lds.hidden.part[i][t][k - stage], 16);
#pragma unroll
                for (int m = 0; m < kCols; ++m) {
                    if constexpr (kBf16) {
                        const v8bf w = column<v8bf>(row, m);
#pragma unroll
                        for (int i = kParts - 1; i >= 0; --i) acc[m] = mfma(v[i], w, acc[m]);
                    } else {
                        v8bf w, rest;
                        column_halves(row, m, w, rest);
#pragma unroll
                        for (int i = kParts - 1; i >= 0; --i) {
                            acc[m] = mfma(v[i], rest, acc[m]);
                            acc[m] = mfma(v[i], w, acc[m]);
                        }
                    }
                }
            } else {
                using V8 = typename std::conditional<kBf16, v8bf, v8h>::type;
                E x[8];
                load_x<E>(a, pair, k, end, x);
                const V8 left = __builtin_bit_cast(V8, x);
#pragma unroll
                for (int m = 0; m < kCols; ++m) acc[m] = mfma(left, column<V8>(row, m), acc[m]);
            }
        };
        // the next step's rows in flight
        v4u even[8], odd[8];
        constexpr int kStep = kWaves * kRows;
        static_assert(kStage % (2 * kStep) == 0, "a stage begins with an even step");
        int k0 = begin + wave * kRows;
        if (k0 < end) load_rows(k0, even);
        for (stage = begin; stage < end; stage += kDown ? kStage : end) {
            const int stage_end = kDown ? min(end, stage + kStage) : end;
            if constexpr (kDown) {
                __syncthreads();
                // to the end of the last step; 0 after the last row
                const int filled = stage + (stage_end - stage + kRows - 1) / kRows * kRows;
                for (int i = tid; i < here * (kStage / 8); i += kThreads) {
                    const int t = i / (kStage / 8), k = stage + i % (kStage / 8) * 8;
                    if (k >= filled) continue;
                    float v[8];
                    load_hidden<E>(a, list[t0 + t], unit, k, end, v);
                    lds.hidden.put(t, k - stage, v);
                }
                __syncthreads();
            }
            while (k0 < stage_end) {
                if (k0 + kStep < end) load_rows(k0 + kStep, odd);
                multiply(k0, even);
                k0 += kStep;
                if (k0 >= stage_end) break;  // only at the rows' end
                if (k0 + kStep < end) load_rows(k0 + kStep, even);
                multiply(k0, odd);
                k0 += kStep;
            }
        }
        __syncthreads();
        // the waves' sums, in their order; a lane has the tokens 4 group + i
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * group + i < here)
#pragma unroll
                for (int m = 0; m < kCols; ++m)
                    lds.red[wave][4 * group + i][col_lane * kCols + m] = acc[m][i];
        __syncthreads();
        for (int i = tid; i < here * kTileCols; i += kThreads) {
            const int t = i / kTileCols, c = i % kTileCols;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += lds.red[w][t][c];
            const int col = first_col(c / kCols) + c % kCols;
            if (col < p.cols)
                p.sums[(int64_t(split) * pairs + list[t0 + t]) * p.cols + col] = sum;
        }
        __syncthreads();
    }
}

// Wave w takes the token's units w, w + 4, ..: their sums over the splits, four loads in flight.
template <typename E>
__global__ __launch_bounds__(kThreads) void combine(Args a) {
    __shared__ float part[kWaves][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, i = blockIdx.y;
    const int col = blockIdx.x * kWave + lane, from = min(col, a.d_out - 1);
    const int64_t stride = int64_t(a.n) * a.K * a.d_out;
    float y = 0.0f;
    for (int k = wave; k < a.K; k += kWaves) {
        const int pair = i * a.K + k;
        const float* at = a.down.sums + int64_t(pair) * a.d_out + from;
        float z = 0.0f;
        for (int s = 0; s < a.down.splits; s += 4) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = s + j < a.down.splits ? at[(s + j) * stride] : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) z += v[j];
        }
        if (a.b2)
            z += to_f32(static_cast<const E*>(a.b2)[int64_t(a.unit[pair]) * a.d_out + from]);
        y = __builtin_fmaf(a.share[pair], z, y);
    }
    part[wave][lane] = y;
    __syncthreads();
    if (wave != 0 || col >= a.d_out) return;
    for (int w = 1; w < kWaves; ++w) y += part[w][lane];
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

// How a product's rows are split: some 512 workgroups (two a compute unit), but at least two steps a
// wave.
Product plan(const void* W, int rows, int cols, int slots, int size) {
    Product p{};
    p.W = W, p.rows = rows, p.cols = cols;
    p.tiles = (cols + 16 * (16 / size) - 1) / (16 * (16 / size));
    const int most = std::max(1, rows / (2 * kWaves * kRows));
    const int splits = std::min(most, std::max(1, 512 / (slots * p.tiles)));
    p.split_rows = ((rows + splits - 1) / splits + kRows - 1) / kRows * kRows;
    p.splits = (rows + p.split_rows - 1) / p.split_rows;
    return p;
}

// Fills `a`'s products and its parts of the workspace; returns the workspace's bytes.
int64_t layout(Args& a, const void* W1, const void* W2, char* base, int size) {
    const int slots = std::min(a.n * a.K, a.M);
    const int64_t pairs = int64_t(a.n) * a.K;
    a.up = plan(W1, a.d_in, a.activation == HSN_UNITS_SWIGLU ? 2 * a.H : a.H, std::max(1, slots), size);
    a.down = plan(W2, a.H, a.d_out, std::max(1, slots), size);
    int64_t at = 0;
    auto take = [&](int64_t count) {
        char* p = base + at;
        at += (4 * count + 255) / 256 * 256;
        return p;
    };
    a.logit = reinterpret_cast<float*>(take(int64_t(a.n) * a.M));
    a.unit = reinterpret_cast<int*>(take(pairs));
    a.share = reinterpret_cast<float*>(take(pairs));
    a.up.sums = reinterpret_cast<float*>(take(a.up.splits * pairs * a.up.cols));
    a.down.sums = reinterpret_cast<float*>(take(a.down.splits * pairs * a.down.cols));
    return at;
}

template <typename E>
void launch(Args a, hipStream_t st) {
    // The choice is the first product's where all tokens' units are a thread each, which saves a
    // kernel of 4.7 us, else a launch of its own.
    a.choose_inline = a.n * a.M <= kThreads;
    route<E><<<dim3(a.n, (a.M + kWaves - 1) / kWaves), kThreads, 0, st>>>(a);
    if (!a.choose_inline) choose<<<a.n, kThreads, 0, st>>>(a);
    const int slots = std::min(a.n * a.K, a.M);
    product<E, false><<<dim3(a.up.tiles * a.up.splits, slots), kThreads, 0, st>>>(a);
    product<E, true><<<dim3(a.down.tiles * a.down.splits, slots), kThreads, 0, st>>>(a);
    combine<E><<<dim3((a.d_out + kWave - 1) / kWave, a.n), kThreads, 0, st>>>(a);
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
    Args a{};
    a.n = n, a.M = M, a.K = K, a.d_in = d_in, a.H = H, a.d_out = d_out, a.activation = activation;
    *bytes = layout(a, nullptr, nullptr, nullptr, dtype == HSN_DTYPE_F32 ? 4 : 2);
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
    HSN_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, HSN_ERR_INVALID_ARGUMENT,
                "the workspace must be aligned to 16 bytes");
    Args a{};
    a.x = x, a.x_row = x_row, a.router = router, a.b1 = b1, a.b2 = b2, a.y = y;
    a.n = n, a.M = M, a.K = K, a.d_in = d_in, a.H = H, a.d_out = d_out, a.activation = activation;
    HSN_REQUIRE(workspace_bytes >= layout(a, W1, W2, static_cast<char*>(workspace),
                                          dtype == HSN_DTYPE_F32 ? 4 : 2),
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
