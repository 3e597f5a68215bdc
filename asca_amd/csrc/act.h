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
