// Rows of logits: ordered keys of their values and reductions over a block.
#pragma once
#include "act.h"

namespace asca {

constexpr float LOG2E = 1.44269504f;
constexpr double LN2 = 0.693147180559945309;

// Temperatures that entry points take: log2(e) / tau is finite (its products with logits need not
// be: where they are large, differences of logits are formed first)
inline bool logits_temperature(float tau) { return tau >= 1e-30f && tau < INFINITY; }

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

// exp(x) of a double, to f32's precision: the argument's rounding is put back
ASCA_DEV float exp_d(double x) {
    const double y = x * 1.4426950408889634;
    const float h = (float)y;
    return h > -INFINITY ? __builtin_amdgcn_exp2f(h) * (1.0f + (float)(y - h) * 0.693147181f) : h == -INFINITY ? 0.0f : h;
}
// log(x): to 2^-24 (not relative to a large result), or to 1e-10, where small differences of
// logarithms or scores next to each other count
ASCA_DEV double log_d(float x) {
    float m = __builtin_amdgcn_frexp_mantf(x);   // 0.5 to 1
    int e = __builtin_amdgcn_frexp_expf(x);
    if (m < 0.70710678f) m *= 2.0f, --e;
    return ((double)e + (double)__builtin_amdgcn_logf(m)) * LN2;
}
// 2 artanh(a / b), |a / b| < 0.177: its odd powers up to the 11th (the 13th is 2.6e-11 there)
ASCA_DEV double artanh2(double a, double b) {
    double r = __builtin_amdgcn_rcp(b);
    r = fma(fma(-b, r, 1.0), r, r);
    const double t = a * r, q = t * t;
    double v = 2.0 / 11;
    v = fma(v, q, 2.0 / 9), v = fma(v, q, 2.0 / 7), v = fma(v, q, 2.0 / 5), v = fma(v, q, 2.0 / 3), v = fma(v, q, 2.0);
    return v * t;
}
ASCA_DEV double log_exact(float x, bool near = false, double a = 0.0, double b = 1.0) {   // near: 2 artanh(a / b)
    float m = __builtin_amdgcn_frexp_mantf(x);
    int e = __builtin_amdgcn_frexp_expf(x);
    if (m < 0.70710678f) m *= 2.0f, --e;
    const double l = artanh2(near ? a : (double)m - 1.0, near ? b : (double)m + 1.0);   // log m
    return near ? l : x > 0.0f && x < INFINITY ? fma((double)e, LN2, l) : (double)__builtin_amdgcn_logf(x);
}

// ------------------------------------------------------ lanes of a wave

// The wave's number in its block, in a scalar register with all that follows from it
ASCA_DEV int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// What lane ^ M holds, M = 1, 2, 4 or 8
template <int M>
ASCA_DEV float lane_xor(float x) {
    if constexpr (M == 1) return dpp<DPP_QUAD_XOR1>(x);
    if constexpr (M == 2) return dpp<DPP_QUAD_XOR2>(x);
    if constexpr (M == 4) return dpp<DPP_HALF_MIRROR>(dpp<0x1B>(x));   // ^3 (quad_perm [3,2,1,0]), then ^7
    return dpp<DPP_ROW_ROR8>(x);
}
// The larger of x and what lane ^ M holds with c = inf, the smaller with c = -inf: the median
// with it, one instruction (no NaN; max and min would each first quiet theirs).
template <int M>
ASCA_DEV float lane_pick(float x, float c) {
    if constexpr (M >= 16) {   // the swap leaves the pair in both lanes, in either order
        const unsigned u = __float_as_uint(x);
        auto r = M == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                         : __builtin_amdgcn_permlane32_swap(u, u, false, false);
        return __builtin_amdgcn_fmed3f(__uint_as_float(r[0]), __uint_as_float(r[1]), c);
    } else {
        return __builtin_amdgcn_fmed3f(x, lane_xor<M>(x), c);
    }
}
// The larger of two, or NaN where either is (one instruction for three of them; a maximum that
// leaves a NaN out quiets each operand first)
ASCA_DEV float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The largest of the wave's values, NaN where one is
ASCA_DEV float wave_max(float x) {
    x = max_or_nan(x, lane_xor<1>(x));
    x = max_or_nan(x, lane_xor<2>(x));
    x = max_or_nan(x, dpp<DPP_HALF_MIRROR>(x));   // four lanes hold the same
    x = max_or_nan(x, dpp<DPP_ROW_MIRROR>(x));
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = max_or_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_or_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

ASCA_DEV double lane_value(double x, int lane) {
    const uint64_t u = __double_as_longlong(x);
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)u, lane), hi = __builtin_amdgcn_readlane((unsigned)(u >> 32), lane);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
ASCA_DEV float lane_value(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }

// The sums of four values over the wave together: a third of the steps that they take apart
ASCA_DEV void wave_sum4(float& a, float& b, float& c, float& d) {
    const float x = group_sum<16>(tsum16(tsum32(a, b), tsum32(c, d)));
    a = lane_value(x, 0), c = lane_value(x, 16), b = lane_value(x, 32), d = lane_value(x, 48);
}

template <int M>
ASCA_DEV float lane_step(float x) { return lane_pick<M>(x, threadIdx.x & M ? -INFINITY : INFINITY); }
// The steps of a bitonic network that sort runs of N lanes, the largest first
template <int N>
ASCA_DEV float lane_merge(float x) {
    if constexpr (N >= 64) x = lane_step<32>(x);
    if constexpr (N >= 32) x = lane_step<16>(x);
    if constexpr (N >= 16) x = lane_step<8>(x);
    if constexpr (N >= 8) x = lane_step<4>(x);
    if constexpr (N >= 4) x = lane_step<2>(x);
    return lane_step<1>(x);
}
// x, or -x in the lanes of `bits`
ASCA_DEV float lane_flip(float x, unsigned bits) { return __uint_as_float(__float_as_uint(x) ^ (bits ? 0x80000000u : 0u)); }
// The wave's values, the largest in lane 0: every other run of a stage is sorted the other
// way round, as the largest first of -x
ASCA_DEV float lane_sort(float x) {
    const unsigned l = threadIdx.x, d = l ^ l >> 1;   // bit k of d: bits k and k + 1 differ
    x = lane_merge<2>(lane_flip(x, l & 2));
    x = lane_merge<4>(lane_flip(x, d & 2));
    x = lane_merge<8>(lane_flip(x, d & 4));
    x = lane_merge<16>(lane_flip(x, d & 8));
    x = lane_merge<32>(lane_flip(x, d & 16));
    return lane_merge<64>(lane_flip(x, l & 32));
}

template <typename T>
ASCA_DEV T wave_max_t(T x) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
        const T y = __shfl_xor(x, s, 64);
        x = y > x ? y : x;
    }
    return x;
}
// The largest over a block of 64 NW threads, in every thread; `lds` holds NW values.
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

// ------------------------------------------------------------ row pieces

// A row's n elements as pieces of B bytes (16 or 8): `head` elements before the first whole
// piece of the address space, nb pieces of W, fewer than W after them.  `fixed`: the pieces begin
// at the row's first element, at any address of one, so that which thread has what, and with it
// the rounding of a sum over the row, is the same wherever the row lies.
template <int B>
struct PieceRaw {
    typedef uint4 type;
};
template <>
struct PieceRaw<8> {
    typedef uint2 type;
};
template <typename E, int B = 16>
struct Pieces {
    static constexpr int W = B / sizeof(E);
    typedef typename PieceRaw<B>::type Raw;
    const E* p;
    int n, head, nb;
    // (without pieces all of up to 2 W - 1 elements are at the edges)
    ASCA_DEV Pieces(const E* row, int len, bool pieces = true, bool fixed = false) : p(row), n(len) {
        const int off = fixed ? 0 : (int)(reinterpret_cast<uintptr_t>(row) / sizeof(E) % W);
        head = min(off ? W - off : 0, n);
        nb = pieces ? (n - head) / W : 0;
    }
    ASCA_DEV Raw piece(int i) const {
        Raw r;
        __builtin_memcpy(&r, p + head + (long)i * W, B);   // one load, at any address of an element
        return r;
    }
    ASCA_DEV int col(int i) const { return head + i * W; }   // the first column of a piece
    // the column outside the pieces that thread t takes, or -1: one of the first 2 W, of the first 32
    // without pieces
    ASCA_DEV int edge(int t) const {
        if (t < head) return t;
        const int c = head + nb * W + t - W;
        return t >= W && c < n ? c : -1;
    }
    ASCA_DEV int edge_thread(int c) const { return c < head ? c : c - head - nb * W + W; }
};

// A piece that is nothing but -inf
template <typename E, int B = 16>
ASCA_DEV typename PieceRaw<B>::type piece_none() {
    const unsigned w = sizeof(E) == 4 ? 0xff800000u : 0xff80ff80u;
    if constexpr (B == 16) return make_uint4(w, w, w, w);
    else return make_uint2(w, w);
}
// -inf in the places of the bits that are set
ASCA_DEV void piece_mask(uint4& r, unsigned bits4, float) {
    r.x = bits4 & 1 ? 0xff800000u : r.x, r.y = bits4 & 2 ? 0xff800000u : r.y;
    r.z = bits4 & 4 ? 0xff800000u : r.z, r.w = bits4 & 8 ? 0xff800000u : r.w;
}
ASCA_DEV void piece_mask(uint4& r, unsigned bits8, bf16_t) {
    auto two = [](unsigned v, unsigned b) {
        v = b & 1 ? (v & 0xffff0000u) | 0xff80u : v;
        return b & 2 ? (v & 0xffffu) | 0xff800000u : v;
    };
    r.x = two(r.x, bits8), r.y = two(r.y, bits8 >> 2), r.z = two(r.z, bits8 >> 4), r.w = two(r.w, bits8 >> 6);
}
// The values of a piece
ASCA_DEV void piece_values(uint4 r, float (&v)[4], float) {
    v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
}
ASCA_DEV void piece_values(uint2 r, float (&v)[2], float) { v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y); }
ASCA_DEV void piece_values(uint2 r, float (&v)[4], bf16_t) { act_values(r, v); }
ASCA_DEV void piece_values(uint4 r, float (&v)[8], bf16_t) {
    act_values(make_uint2(r.x, r.y), v);
    act_values(make_uint2(r.z, r.w), v + 4);
}
// What is made of a piece after this is made anew: the compiler would keep the 32-bit values
// of an earlier look at it, in twice its registers (bf16).
ASCA_DEV void piece_again(uint4& r) { asm("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); }
ASCA_DEV void piece_again(uint2& r) { asm("" : "+v"(r.x), "+v"(r.y)); }

}  // namespace asca
