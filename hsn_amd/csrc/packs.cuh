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
template <typename E>
__device__ __forceinline__ void store_pack(E* p, const Pack<E>& v) {
    __builtin_memcpy(p, &v, 16);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int mask = 32; mask; mask >>= 1) v += __shfl_xor(v, mask, kWave);
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
