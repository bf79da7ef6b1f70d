// Packs of 16 bytes at any element's address, and sums over a workgroup.
//
// Global memory takes 16-byte accesses at any address on gfx950, so a pack is addressed as E and a row
// or tensor that starts off a 16-byte boundary needs no other path: its packs are the same ones, some
// of them across two cache lines.
#pragma once

#include "common.cuh"
#include "dpp.cuh"

namespace hsn {

template <typename E>
struct Pack {
    static constexpr int kN = 16 / sizeof(E);
    E e[kN];
    __device__ __forceinline__ float operator[](int j) const { return to_f32(e[j]); }
};

template <typename E>
__device__ __forceinline__ Pack<E> load_pack(const E* p) {
    Pack<E> v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// Outputs beyond half of the last-level cache are stored past it, which leaves it to what is read again (the
// logits' second reading, say): see the kernels for what each gains. Smaller ones stay in it for whoever
// reads them next (a gradient of 60 MB: 31.3 us, past the cache 32.2).
constexpr int64_t kStream = int64_t(128) << 20;

template <int BYTES>
__device__ __forceinline__ void stream_bytes(void* p, const void* v) {
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
    static_assert(BYTES % 16 == 0, "packs");
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
        words w;
        __builtin_memcpy(&w, static_cast<const char*>(v) + 16 * i, 16);
        __builtin_nontemporal_store(w, reinterpret_cast<words*>(static_cast<char*>(p) + 16 * i));
    }
}

// (A template: of two branches that store the same, the compiler makes one ordinary store.)
template <bool STREAM, typename E>
__device__ __forceinline__ void store_pack(E* p, const Pack<E>& v) {
    if constexpr (STREAM)
        stream_bytes<16>(p, &v);
    else
        __builtin_memcpy(p, &v, 16);
}

// Between a wave's accesses to LDS by different lanes: a wave's LDS instructions are carried out in their
// order, so it is enough that the compiler keeps it. (A fence would wait for loads in flight as well.)
__device__ __forceinline__ void wave_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// A double's halves through the lanes (an LDS shuffle costs five times as much).
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, uint64_t(dpp_u32<CTRL>(static_cast<uint32_t>(u >> 32))) << 32 |
                                          dpp_u32<CTRL>(static_cast<uint32_t>(u)));
}
__device__ __forceinline__ double rows_sum(RowPair lo, RowPair hi) {
    return __builtin_bit_cast(double, uint64_t(hi.lo) << 32 | lo.lo) +
           __builtin_bit_cast(double, uint64_t(hi.hi) << 32 | lo.hi);
}
// The sum over the lanes of a wave whose numbers differ by multiples of G, in each of them.
template <int G = 1>
__device__ __forceinline__ double wave_sum(double v) {
    if constexpr (G <= 1) v += dpp_f64<dpp::kXor1>(v);
    if constexpr (G <= 2) v += dpp_f64<dpp::kXor2>(v);
    if constexpr (G <= 4) v += dpp_f64<0x124>(v);  // row_ror:4
    if constexpr (G <= 8) v += dpp_f64<dpp::kRor8>(v);
    if constexpr (G <= 16) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        v = rows_sum(pair16(static_cast<uint32_t>(u)), pair16(static_cast<uint32_t>(u >> 32)));
    }
    if constexpr (G <= 32) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        v = rows_sum(pair32(static_cast<uint32_t>(u)), pair32(static_cast<uint32_t>(u >> 32)));
    }
    return v;
}

// The sum over a workgroup of WAVES waves, in every thread and in a fixed order. `s`: WAVES doubles of LDS.
template <int WAVES>
__device__ __forceinline__ double block_sum(double v, double* s) {
    v = wave_sum(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = v;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += s[w];
    return total;
}

}  // namespace hsn
