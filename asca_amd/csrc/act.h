// Activation rows in f32 or bf16: typed loads and stores of the kernels that
// take either (all arithmetic is in 32 bits; a bf16 result is rounded once, to
// nearest even, when it is stored).
#pragma once
#include <stdint.h>

#include "common.h"
#include "runtime.h"

namespace asca {

typedef uint16_t bf16_t;  // raw bits

ASCA_DEV float act_value(float x) { return x; }
ASCA_DEV float act_value(bf16_t x) { return __uint_as_float((unsigned)x << 16); }
template <typename E>
ASCA_DEV float act_load(const E* p) { return act_value(*p); }
ASCA_DEV void act_store(float* p, float x) { *p = x; }
ASCA_DEV void act_store(bf16_t* p, float x) { *p = __builtin_bit_cast(bf16_t, (__bf16)x); }

// V neighbouring values as one access (V = 4: 16 bytes of f32, 8 of bf16, aligned to
// that; V = 1: any address)
template <int V, typename E>
struct ActRaw {
    typedef E type;
};
template <>
struct ActRaw<4, float> {
    typedef f32x4 type;
};
template <>
struct ActRaw<4, bf16_t> {
    typedef uint2 type;
};
template <int V, typename E>
using act_raw = typename ActRaw<V, E>::type;

template <int V, typename E>
ASCA_DEV act_raw<V, E> act_load_raw(const E* p) { return *reinterpret_cast<const act_raw<V, E>*>(p); }

ASCA_DEV void act_values(float r, float* v) { v[0] = r; }
ASCA_DEV void act_values(bf16_t r, float* v) { v[0] = act_value(r); }
ASCA_DEV void act_values(f32x4 r, float* v) { v[0] = r[0], v[1] = r[1], v[2] = r[2], v[3] = r[3]; }
ASCA_DEV void act_values(uint2 r, float* v) {
    v[0] = __uint_as_float(r.x << 16), v[1] = __uint_as_float(r.x & 0xffff0000u);
    v[2] = __uint_as_float(r.y << 16), v[3] = __uint_as_float(r.y & 0xffff0000u);
}

template <int V>
ASCA_DEV void act_store_n(float* p, const float* v) {
    if constexpr (V == 1)
        *p = v[0];
    else
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
}
template <int V>
ASCA_DEV void act_store_n(bf16_t* p, const float* v) {
    if constexpr (V == 1) {
        act_store(p, v[0]);
    } else {
        bf16_t b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) act_store(b + k, v[k]);
        *reinterpret_cast<uint2*>(p) = make_uint2(b[0] | (unsigned)b[1] << 16, b[2] | (unsigned)b[3] << 16);
    }
}

// Whether a matrix (NULL: none) allows accesses of 4 values at multiples of 4 columns
inline bool act_vec_ok(const void* p, long ld, int dtype) {
    return !p || (ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (dtype == ASCA_F32 ? 16 : 8) == 0);
}

// 1 / (1 + exp(-v)): the exponential is of a value <= 0, so nothing overflows.
ASCA_DEV float act_sigmoid(float v) {
    const float t = __builtin_amdgcn_exp2f(-fabsf(v) * 1.44269504f);
    const float s = __builtin_amdgcn_rcpf(1.0f + t);   // to one unit of the last place
    return v >= 0.0f ? s : t * s;
}

// Calls f with a null pointer of the element type that `dtype` names.
template <typename F>
int act_dispatch(int dtype, F f) {
    if (dtype == ASCA_F32) return f((float*)nullptr);
    if (dtype == ASCA_BF16) return f((bf16_t*)nullptr);
    return fail(ASCA_ERR_UNSUPPORTED, "element type %d (ASCA_F32 or ASCA_BF16)", dtype);
}

}  // namespace asca
