// Rows of logits: ordered keys of their values and reductions over a block.
#pragma once
#include "act.h"

namespace asca {

constexpr float LOG2E = 1.44269504f;
constexpr double LN2 = 0.693147180559945309;

// A key that orders values descending by value, then ascending by place: the larger of two
// keys is the larger value, or the lower place of equal ones (0 and -0 are equal).  Values
// that are never listed (NaN, -inf) have the key 0.
ASCA_DEV uint64_t logit_key(float v, unsigned place) {
    if (!(v > -INFINITY)) return 0;
    const unsigned b = __float_as_uint(v + 0.0f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (~place);
}
ASCA_DEV float key_value(uint64_t k) {
    const unsigned b = (unsigned)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
ASCA_DEV unsigned key_place(uint64_t k) { return ~(unsigned)k; }

template <typename T>
ASCA_DEV T wave_max_t(T x) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
        const T y = __shfl_xor(x, s, 64);
        x = y > x ? y : x;
    }
    return x;
}
template <typename T>
ASCA_DEV T wave_sum_t(T x) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) x += __shfl_xor(x, s, 64);
    return x;
}

// The largest (the sum) over a block of 64 NW threads, in every thread; `lds` holds NW values.
template <int NW, typename T>
ASCA_DEV T block_max_t(T x, T* lds) {
    x = wave_max_t(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) x = lds[w] > x ? lds[w] : x;
    return x;
}
template <int NW, typename T>
ASCA_DEV T block_sum_t(T x, T* lds) {
    x = wave_sum_t(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) x += lds[w];
    return x;
}

}  // namespace asca
