// The norms around a block fused with its gate and residual scale, per row
// (rms(a) = a i(a), i(a) = 1 / sqrt(mean(a^2) + eps)):
//   u = y o silu(z);  r = x + s o rms(u) o w1;  n = rms(r) o w2
// and back from dr, dn:
//   dR = dr + i2 (w2 dn - rh mean(w2 dn rh)), rh = rms(r);  dx = dR
//   dp = s o dR;  du = i1 (w1 dp - uh mean(w1 dp uh)), uh = rms(u)
//   dy = du silu(z);  dz = du y silu'(z);  dw1 = sum dp uh, ds = sum dR w1 uh,
//   dw2 = sum dn rh
// A row stays in the registers of 64 WPR threads, so each operand is read once
// and each result written once, in either direction; what the backward needs of
// the forward it computes again from x, y and z.  Bound by memory: 16384 x 512 f32
// forward 26 us, backward 47 us (6.5 and 5.7 TB/s, some of it from the last-level
// cache), 16384 x 2048 bf16 71 and 116 us (4.7 and 4.6 TB/s).  Rows that cannot be loaded
// four values at a time are loaded one at a time: 16384 x 2047 bf16 85 and 207 us (2048,
// with the sums' launch too: 71 and 128), 16384 x 511 f32 28 and 57 (26 and 51).
#include <algorithm>

#include "act.h"
#include "parts.h"

namespace asca {

struct NormArgs {
    const void *x, *y, *z, *dr, *dn;
    long ldx, ldy, ldz, lddr, lddn;
    const float *w1, *s, *w2;
    void *r, *n, *dx, *dy, *dz;
    long ldr, ldn, lddx, lddy, lddz;
    float* part;   // (blocks, 3, cols): dw1, ds, dw2
    long rows;
    int cols;
    float eps;
};

// An operand of the rows, or in the place of one that is not given another's, whose
// values are replaced by zeros once they are there.  All loads of a row are issued
// before any is looked at: none sits under a condition or is converted on the way,
// as either would wait for it (16384 x 2048 bf16 backward 307 -> 177 us).
template <typename E>
struct NormOp {
    const E* m;
    long ld;
    bool on;
    ASCA_DEV NormOp(const void* a, long la, const void* other, long lo)
        : m(static_cast<const E*>(a ? a : other)), ld(a ? la : lo), on(a != nullptr) {}
    template <int VEC>
    ASCA_DEV act_raw<VEC, E> load(long row, int c, int cols) const {
        return act_load_raw<VEC>(m + row * ld + min(c, cols - VEC));
    }
    // values at column c (zeros past the row's end)
    template <int VEC>
    ASCA_DEV void values(act_raw<VEC, E> r, int c, int cols, float* v) const {
        act_values(r, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = on && c < cols ? v[k] : 0.0f;
    }
};

template <int VEC, typename E>
ASCA_DEV void row_store(E* row, int c, int cols, const float* v) {
    if (c < cols) act_store_n<VEC>(row + c, v);
}

// Sum over the threads of a row
template <int WPR>
ASCA_DEV float row_sum(float x, float* lds) {
    x = wave_sum(x);
    if constexpr (WPR > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) x += lds[w];
    }
    return x;
}

template <int CTRL>
ASCA_DEV double dpp_d(double x) {
    const uint2 u = __builtin_bit_cast(uint2, x);
    return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_mov_dpp((int)u.x, CTRL, 0xF, 0xF, true),
                                                 __builtin_amdgcn_mov_dpp((int)u.y, CTRL, 0xF, 0xF, true)));
}

// Sums over the wave of 8 values, in every lane: scattered over the lanes' low three
// bits while there are several, added over the others, read back by lane.
ASCA_DEV void wave_sums8(double (&v)[8]) {
    const int lane = threadIdx.x & 63;
    double a[4], b[2], x;
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = (lane & 4 ? v[k + 4] : v[k]) + dpp_d<DPP_HALF_MIRROR>(lane & 4 ? v[k] : v[k + 4]);
#pragma unroll
    for (int k = 0; k < 2; ++k) b[k] = (lane & 2 ? a[k + 2] : a[k]) + dpp_d<DPP_QUAD_XOR2>(lane & 2 ? a[k] : a[k + 2]);
    x = (lane & 1 ? b[1] : b[0]) + dpp_d<DPP_QUAD_XOR1>(lane & 1 ? b[0] : b[1]);
    x += dpp_d<DPP_ROW_ROR8>(x);
    x += __shfl_xor(x, 16, 64);
    x += __shfl_xor(x, 32, 64);
    const uint2 u = __builtin_bit_cast(uint2, x);
#pragma unroll
    for (int k = 0; k < 8; ++k)
        v[k] = __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_readlane(u.x, k), __builtin_amdgcn_readlane(u.y, k)));
}

// The same over the threads of a row; `turn` alternates from call to call
template <int WPR>
ASCA_DEV void row_sums8(double (&v)[8], double (*lds)[WPR][8], int turn) {
    wave_sums8(v);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < 8; ++k) lds[turn & 1][threadIdx.x >> 6][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = lds[turn & 1][0][k];
#pragma unroll
            for (int w = 1; w < WPR; ++w) v[k] += lds[turn & 1][w][k];
        }
    }
}

template <int WPR>
constexpr int bn_threads() { return WPR == 1 ? 256 : 64 * WPR; }

// VEC values of a parameter (ones where there is none; past the row's end any that
// exist: they meet zeros)
template <int VEC>
ASCA_DEV void par_load(const float* m, int c, int cols, float* v) {
    if (m) {
        act_values(act_load_raw<VEC>(m + min(c, cols - VEC)), v);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = 1.0f;
    }
}

template <typename E, int VEC, int NV, int WPR>
__global__ __launch_bounds__(bn_threads<WPR>()) void block_norm_fwd_k(NormArgs p) {
    __shared__ float lds[WPR];
    constexpr int NE = VEC * NV, RPB = bn_threads<WPR>() / (64 * WPR);
    const long row = (long)blockIdx.x * RPB + threadIdx.x / (64 * WPR);
    const int tid = threadIdx.x % (64 * WPR);
    if (row >= p.rows) return;
    const void* any = p.x ? p.x : p.y;
    const long la = p.x ? p.ldx : p.ldy;
    const NormOp<E> ox(p.x, p.ldx, any, la), oy(p.y, p.ldy, any, la), oz(p.z, p.ldz, any, la);
    act_raw<VEC, E> rx[NV], ry[NV], rz[NV];
    float w1[NE], s[NE], w2[NE], r[NE], u[NE], z[NE], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + tid) * VEC;
        rx[i] = ox.template load<VEC>(row, c, p.cols);
        ry[i] = oy.template load<VEC>(row, c, p.cols);
        rz[i] = oz.template load<VEC>(row, c, p.cols);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + tid) * VEC;
        par_load<VEC>(p.w1, c, p.cols, w1 + i * VEC);
        par_load<VEC>(p.s, c, p.cols, s + i * VEC);
        par_load<VEC>(p.w2, c, p.cols, w2 + i * VEC);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + tid) * VEC;
        ox.template values<VEC>(rx[i], c, p.cols, r + i * VEC);
        oy.template values<VEC>(ry[i], c, p.cols, u + i * VEC);
        oz.template values<VEC>(rz[i], c, p.cols, z + i * VEC);
    }
    if (p.y) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            if (p.z) u[e] *= z[e] * act_sigmoid(z[e]);
            ss = fmaf(u[e], u[e], ss);
        }
        const float i1 = 1.0f / sqrtf(row_sum<WPR>(ss, lds) / (float)p.cols + p.eps);
#pragma unroll
        for (int e = 0; e < NE; ++e) r[e] = fmaf(s[e], u[e] * i1 * w1[e], r[e]);
    }
    if (p.r)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            row_store<VEC>(static_cast<E*>(p.r) + row * p.ldr, (i * 64 * WPR + tid) * VEC, p.cols, r + i * VEC);
    if (!p.n) return;
    ss = 0.0f;
#pragma unroll
    for (int e = 0; e < NE; ++e) ss = fmaf(r[e], r[e], ss);
    const float i2 = 1.0f / sqrtf(row_sum<WPR>(ss, lds) / (float)p.cols + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + tid) * VEC;
        float v[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = r[i * VEC + k] * i2 * w2[i * VEC + k];
        row_store<VEC>(static_cast<E*>(p.n) + row * p.ldn, c, p.cols, v);
    }
}

// All sums that a row needs are sums of products of its inputs: with q = s w1 u,
// k = w2 dn and r = x + i1 q,
//   sum r^2 = sum x^2 + 2 i1 sum x q + i1^2 sum q^2,  sum k r = sum k x + i1 sum k q,
//   sum dR q = sum dr q + i2 (sum k q - m2 (sum x q + i1 sum q^2)),
// so one pass and one exchange between the threads give seven of them, and nothing
// waits for a second.  They are taken in 64 bits, as k - r m2 and t - u m1 are:
// these cancel where the gradient is near a multiple of the row (always in a row of
// one column), and products of two f32 values are exact there.
// Adds an element's products to the seven sums: c = s w1, k = w2 dn
ASCA_DEV void norm_sums(double (&v)[8], float x, float u, float c, float k, float dr) {
    const double ud = u, q = (double)c * ud, kd = k, xd = x;
    v[0] = fma(ud, ud, v[0]);
    v[1] = fma(xd, xd, v[1]);
    v[2] = fma(xd, q, v[2]);
    v[3] = fma(q, q, v[3]);
    v[4] = fma(kd, xd, v[4]);
    v[5] = fma(kd, q, v[5]);
    v[6] = fma((double)dr, q, v[6]);
}

// What a row's sums come to
struct NormStats {
    double i1, i2, m1, m2;
    float i1f, i2f;
    ASCA_DEV NormStats(const NormArgs& p, const double (&v)[8]) {
        const double in = 1.0 / p.cols;
        i1 = p.y ? 1.0 / sqrt(fma(v[0], in, (double)p.eps)) : 0.0;   // without y not of eps alone, which may be 0
        const double rq = fma(i1, v[3], v[2]);
        i2 = p.dn ? 1.0 / sqrt(fma(fma(i1, v[2] + rq, v[1]), in, (double)p.eps)) : 0.0;
        m2 = fma(i1, v[5], v[4]) * in * (i2 * i2);
        m1 = fma(i2, v[5] - m2 * rq, v[6]) * in * (i1 * i1);
        i1f = (float)i1, i2f = (float)i2;
    }
};

// An element's dR, du, dR uh and rms(r)
struct NormGrad {
    double dR;
    float du, ru, rh;
    ASCA_DEV NormGrad(const NormStats& n, float x, float u, float c, float k, float dr) {
        const double r = fma(n.i1, (double)c * (double)u, (double)x);
        dR = fma(n.i2, fma(-r, n.m2, (double)k), (double)dr);
        du = n.i1f * (float)fma(-(double)u, n.m1, dR * c);
        ru = (float)dR * (u * n.i1f);
        rh = (float)r * n.i2f;
    }
};

template <typename E, int VEC, int NV, int WPR>
__global__ __launch_bounds__(bn_threads<WPR>()) void block_norm_bwd_k(NormArgs p) {
    constexpr int NE = VEC * NV, NT = bn_threads<WPR>(), RPB = NT / (64 * WPR);
    __shared__ double lds[2][WPR][8];
    __shared__ float acc[RPB > 1 ? NT * NE : 1];
    const int sub = threadIdx.x / (64 * WPR), tid = threadIdx.x % (64 * WPR);
    float g1[NE], gs[NE], g2[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) g1[e] = gs[e] = g2[e] = 0.0f;
    int turn = 0;
    const void* any = p.x ? p.x : p.y;
    const long la = p.x ? p.ldx : p.ldy;
    const NormOp<E> ox(p.x, p.ldx, any, la), oy(p.y, p.ldy, any, la), oz(p.z, p.ldz, any, la), odr(p.dr, p.lddr, any, la),
        odn(p.dn, p.lddn, any, la);
    // the parameters stay; a row's operands are loaded while the row before is worked on
    float w1[NV][VEC], s[NV][VEC], w2[NV][VEC];
    act_raw<VEC, E> rx[NV], ry[NV], rz[NV], rdr[NV], rdn[NV];
    auto load = [&](long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * WPR + tid) * VEC;
            rx[i] = ox.template load<VEC>(row, c, p.cols);
            ry[i] = oy.template load<VEC>(row, c, p.cols);
            rz[i] = oz.template load<VEC>(row, c, p.cols);
            rdr[i] = odr.template load<VEC>(row, c, p.cols);
            rdn[i] = odn.template load<VEC>(row, c, p.cols);
        }
    };
    load(min((long)blockIdx.x * RPB + sub, p.rows - 1));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + tid) * VEC;
        par_load<VEC>(p.w1, c, p.cols, w1[i]);
        par_load<VEC>(p.s, c, p.cols, s[i]);
        par_load<VEC>(p.w2, c, p.cols, w2[i]);
#pragma unroll
        for (int m = 0; m < VEC; ++m) asm volatile("" : "+v"(w1[i][m]), "+v"(s[i][m]), "+v"(w2[i][m]));
    }
    for (long row = (long)blockIdx.x * RPB + sub; row < p.rows; row += (long)gridDim.x * RPB, ++turn) {
        float x[NV][VEC], y[NV][VEC], z[NV][VEC], dr[NV][VEC], dn[NV][VEC], sg[NV][VEC];
        double v[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
        auto values = [&](int i) {
            const int c = (i * 64 * WPR + tid) * VEC;
            ox.template values<VEC>(rx[i], c, p.cols, x[i]);
            oy.template values<VEC>(ry[i], c, p.cols, y[i]);
            oz.template values<VEC>(rz[i], c, p.cols, z[i]);
            odr.template values<VEC>(rdr[i], c, p.cols, dr[i]);
            odn.template values<VEC>(rdn[i], c, p.cols, dn[i]);
        };
        auto gates = [&](int i) {
#pragma unroll
            for (int m = 0; m < VEC; ++m) sg[i][m] = p.z ? act_sigmoid(z[i][m]) : 1.0f;
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) values(i);
        load(min(row + (long)gridDim.x * RPB, p.rows - 1));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            gates(i);
#pragma unroll
            for (int m = 0; m < VEC; ++m) {
                const float u = p.z ? y[i][m] * (z[i][m] * sg[i][m]) : y[i][m];
                norm_sums(v, x[i][m], u, s[i][m] * w1[i][m], dn[i][m] * w2[i][m], dr[i][m]);
            }
        }
        row_sums8<WPR>(v, lds, turn);
        // the 64-bit copies are made again below rather than kept over the exchange
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int m = 0; m < VEC; ++m)
                asm volatile("" : "+v"(x[i][m]), "+v"(y[i][m]), "+v"(dr[i][m]), "+v"(dn[i][m]), "+v"(sg[i][m]));
        const NormStats n(p, v);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * WPR + tid) * VEC;
            float vx[VEC], vy[VEC], vz[VEC];
#pragma unroll
            for (int m = 0; m < VEC; ++m) {
                const int e = i * VEC + m;
                const float zz = z[i][m], sz = sg[i][m], gate = p.z ? zz * sz : 1.0f;
                const NormGrad g(n, x[i][m], y[i][m] * gate, s[i][m] * w1[i][m], dn[i][m] * w2[i][m], dr[i][m]);
                g2[e] = fmaf(dn[i][m], g.rh, g2[e]);
                gs[e] = fmaf(g.ru, w1[i][m], gs[e]);
                g1[e] = fmaf(g.ru, s[i][m], g1[e]);
                vx[m] = (float)g.dR;
                vy[m] = g.du * gate;
                vz[m] = p.z ? g.du * y[i][m] * (sz * fmaf(zz, 1.0f - sz, 1.0f)) : 0.0f;
            }
            if (p.dx) row_store<VEC>(static_cast<E*>(p.dx) + row * p.lddx, c, p.cols, vx);
            if (p.dy) row_store<VEC>(static_cast<E*>(p.dy) + row * p.lddy, c, p.cols, vy);
            if (p.dz) row_store<VEC>(static_cast<E*>(p.dz) + row * p.lddz, c, p.cols, vz);
        }
    }
    if (!p.part) return;
    // the block's rows' sums, then one row of partial sums for the block
    auto put = [&](int which, float* g) {
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < NE; ++e) acc[e * NT + threadIdx.x] = g[e];
            __syncthreads();
            if (sub == 0)
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    g[e] = acc[e * NT + tid];
                    for (int k = 1; k < RPB; ++k) g[e] += acc[e * NT + k * 64 * WPR + tid];
                }
        }
        if (sub == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 64 * WPR + tid) * VEC;
                float* dst = p.part + ((long)blockIdx.x * 3 + which) * p.cols;
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (c + k < p.cols) dst[c + k] = g[i * VEC + k];
            }
    };
    put(0, g1);
    put(1, gs);
    put(2, g2);
}

// Rows of any width: a block of BW_NT threads walks the row and reads it again for
// each further sum (from a cache), and the backward adds to its own row of partial
// sums in memory.
constexpr int BW_NT = 512;

template <typename E, int VEC>
struct NormWide {
    const NormArgs& p;
    long row;
    NormOp<E> ox, oy, oz;
    ASCA_DEV NormWide(const NormArgs& a, long r)
        : p(a), row(r), ox(a.x, a.ldx, a.x ? a.x : a.y, a.x ? a.ldx : a.ldy),
          oy(a.y, a.ldy, a.x ? a.x : a.y, a.x ? a.ldx : a.ldy), oz(a.z, a.ldz, a.x ? a.x : a.y, a.x ? a.ldx : a.ldy) {}
    // x, y, z and u = y silu(z) at column c
    ASCA_DEV void at(int c, float* x, float* y, float* z, float* sg, float* u) const {
        const auto rx = ox.template load<VEC>(row, c, p.cols), ry = oy.template load<VEC>(row, c, p.cols),
                   rz = oz.template load<VEC>(row, c, p.cols);
        ox.template values<VEC>(rx, c, p.cols, x);
        oy.template values<VEC>(ry, c, p.cols, y);
        oz.template values<VEC>(rz, c, p.cols, z);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            sg[k] = p.z ? act_sigmoid(z[k]) : 1.0f;
            u[k] = p.z ? y[k] * (z[k] * sg[k]) : y[k];
        }
    }
};

template <typename E, int VEC>
__global__ __launch_bounds__(BW_NT) void block_norm_fwd_wide_k(NormArgs p) {
    __shared__ float lds[BW_NT / 64];
    const NormWide<E, VEC> w(p, blockIdx.x);
    float x[VEC], y[VEC], z[VEC], sg[VEC], u[VEC], w1[VEC], s[VEC], i1 = 0.0f;
    if (p.y) {
        float ss = 0.0f;
        for (int c = threadIdx.x * VEC; c < p.cols; c += BW_NT * VEC) {
            w.at(c, x, y, z, sg, u);
#pragma unroll
            for (int k = 0; k < VEC; ++k) ss = fmaf(u[k], u[k], ss);
        }
        i1 = 1.0f / sqrtf(row_sum<BW_NT / 64>(ss, lds) / (float)p.cols + p.eps);
    }
    auto r_at = [&](int c, float* r) {
        w.at(c, r, y, z, sg, u);
        par_load<VEC>(p.w1, c, p.cols, w1);
        par_load<VEC>(p.s, c, p.cols, s);
#pragma unroll
        for (int k = 0; k < VEC; ++k) r[k] = p.y ? fmaf(s[k], u[k] * i1 * w1[k], r[k]) : r[k];
    };
    float ss = 0.0f, i2 = 0.0f;
    if (p.n) {
        for (int c = threadIdx.x * VEC; c < p.cols; c += BW_NT * VEC) {
            r_at(c, x);
#pragma unroll
            for (int k = 0; k < VEC; ++k) ss = fmaf(x[k], x[k], ss);
        }
        i2 = 1.0f / sqrtf(row_sum<BW_NT / 64>(ss, lds) / (float)p.cols + p.eps);
    }
    // r may be x: a thread overwrites only columns that it has read
    for (int c = threadIdx.x * VEC; c < p.cols; c += BW_NT * VEC) {
        r_at(c, x);
        if (p.r) row_store<VEC>(static_cast<E*>(p.r) + w.row * p.ldr, c, p.cols, x);
        if (!p.n) continue;
        par_load<VEC>(p.w2, c, p.cols, w1);
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] *= i2 * w1[k];
        row_store<VEC>(static_cast<E*>(p.n) + w.row * p.ldn, c, p.cols, x);
    }
}

template <typename E, int VEC>
__global__ __launch_bounds__(BW_NT) void block_norm_bwd_wide_k(NormArgs p) {
    __shared__ double lds[2][BW_NT / 64][8];
    int turn = 0;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x, ++turn) {
        const NormWide<E, VEC> w(p, row);
        const NormOp<E> odr(p.dr, p.lddr, p.x ? p.x : p.y, p.x ? p.ldx : p.ldy),
            odn(p.dn, p.lddn, p.x ? p.x : p.y, p.x ? p.ldx : p.ldy);
        float x[VEC], y[VEC], z[VEC], sg[VEC], u[VEC], dr[VEC], dn[VEC], w1[VEC], s[VEC], w2[VEC];
        auto at = [&](int c) {
            const auto rdr = odr.template load<VEC>(row, c, p.cols), rdn = odn.template load<VEC>(row, c, p.cols);
            w.at(c, x, y, z, sg, u);
            odr.template values<VEC>(rdr, c, p.cols, dr);
            odn.template values<VEC>(rdn, c, p.cols, dn);
            par_load<VEC>(p.w1, c, p.cols, w1);
            par_load<VEC>(p.s, c, p.cols, s);
            par_load<VEC>(p.w2, c, p.cols, w2);
        };
        double v[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
        for (int c = threadIdx.x * VEC; c < p.cols; c += BW_NT * VEC) {
            at(c);
#pragma unroll
            for (int m = 0; m < VEC; ++m) norm_sums(v, x[m], u[m], s[m] * w1[m], dn[m] * w2[m], dr[m]);
        }
        row_sums8<BW_NT / 64>(v, lds, turn);
        const NormStats n(p, v);
        const bool first = row == blockIdx.x;
        for (int c = threadIdx.x * VEC; c < p.cols; c += BW_NT * VEC) {
            at(c);
            float vx[VEC], vy[VEC], vz[VEC];
#pragma unroll
            for (int m = 0; m < VEC; ++m) {
                const NormGrad g(n, x[m], u[m], s[m] * w1[m], dn[m] * w2[m], dr[m]);
                vx[m] = (float)g.dR;
                vy[m] = p.z ? g.du * (z[m] * sg[m]) : g.du;
                vz[m] = g.du * y[m] * (sg[m] * fmaf(z[m], 1.0f - sg[m], 1.0f));
                if (p.part && c + m < p.cols) {
                    float* t = p.part + (long)blockIdx.x * 3 * p.cols + c + m;
                    const float a[3] = {g.ru * s[m], g.ru * w1[m], dn[m] * g.rh};
#pragma unroll
                    for (int k = 0; k < 3; ++k) t[(long)k * p.cols] = first ? a[k] : t[(long)k * p.cols] + a[k];
                }
            }
            if (p.dx) row_store<VEC>(static_cast<E*>(p.dx) + row * p.lddx, c, p.cols, vx);
            if (p.dy) row_store<VEC>(static_cast<E*>(p.dy) + row * p.lddy, c, p.cols, vy);
            if (p.dz) row_store<VEC>(static_cast<E*>(p.dz) + row * p.lddz, c, p.cols, vz);
        }
    }
}

}  // namespace asca

using namespace asca;

// Columns of the kernels that hold a row in registers; wider rows are walked.
static int bn_held(bool bwd) { return bwd ? 2048 : 4096; }

// Calls f with (element type, VEC, NV, WPR), NV = 0 for wide rows: 16-byte (bf16:
// 8-byte) access where every row and the parameters allow it; a row has as few waves
// as its values a lane allow, 8, or 16 in the forward's widest.
template <bool BWD, typename F>
static int bn_dispatch(int dtype, int cols, bool vec, F f) {
    return act_dispatch(dtype, [&](auto* e) {
        using std::integral_constant;
        auto go = [&](auto ne, auto wpr) {
            constexpr int NE = decltype(ne)::value;
            return vec ? f(e, integral_constant<int, 4>{}, integral_constant<int, NE / 4>{}, wpr)
                       : f(e, integral_constant<int, 1>{}, integral_constant<int, NE>{}, wpr);
        };
        const integral_constant<int, 0> n0;
        const integral_constant<int, 1> c1;
        const integral_constant<int, 2> c2;
        const integral_constant<int, 4> c4;
        const integral_constant<int, 8> c8;
        const integral_constant<int, 16> c16;
        if (cols > bn_held(BWD)) return go(n0, c1);
        if (cols <= 256) return go(c4, c1);
        if (cols <= 512) return go(c8, c1);
        if (cols <= 1024) return go(c8, c2);
        if constexpr (BWD) {
            return go(c8, c4);
        } else {
            if (cols <= 2048) return go(c8, c4);
            return go(c16, c4);
        }
    });
}

static int bn_row_check(const char* fn, const char* what, const void* a, long ld, int cols) {
    if (!a || ld >= cols) return ASCA_OK;
    return fail(ASCA_ERR_INVALID, "%s: row stride %s=%ld below its %d columns", fn, what, ld, cols);
}

extern "C" {

int asca_block_norm_fwd(const void* x, long ldx, const void* y, long ldy, const void* z, long ldz, const float* w_post,
                        const float* scale, const float* w_pre, void* r, long ldr, void* n, long ldn, long rows,
                        int cols, float eps, int dtype, void* stream) {
    const char* fn = "asca_block_norm_fwd";
    if (rows < 0 || cols < 0) return fail(ASCA_ERR_INVALID, "%s: negative shape", fn);
    if (!(eps >= 0.0f)) return fail(ASCA_ERR_INVALID, "%s: eps=%g", fn, (double)eps);
    int rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; });
    if (rc) return rc;
    if (!y && (z || w_post || scale)) return fail(ASCA_ERR_INVALID, "%s: z, w_post or scale without y", fn);
    if (!n && w_pre) return fail(ASCA_ERR_INVALID, "%s: w_pre without n", fn);
    if (rows == 0 || cols == 0) return ASCA_OK;
    if ((!x && !y) || (!r && !n)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if ((rc = bn_row_check(fn, "ldx", x, ldx, cols)) || (rc = bn_row_check(fn, "ldy", y, ldy, cols)) ||
        (rc = bn_row_check(fn, "ldz", z, ldz, cols)) || (rc = bn_row_check(fn, "ldr", r, ldr, cols)) ||
        (rc = bn_row_check(fn, "ldn", n, ldn, cols)))
        return rc;
    bool vec = cols % 4 == 0;
    auto rows_ok = [&](const void* a, long ld) { return act_vec_ok(a, ld, dtype); };
    auto par_ok = [&](const float* a) { return reinterpret_cast<uintptr_t>(a) % 16 == 0; };
    vec = vec && rows_ok(x, ldx) && rows_ok(y, ldy) && rows_ok(z, ldz) && rows_ok(r, ldr) && rows_ok(n, ldn) &&
          par_ok(w_post) && par_ok(scale) && par_ok(w_pre);
    NormArgs p{};
    p.x = x, p.y = y, p.z = z, p.ldx = ldx, p.ldy = ldy, p.ldz = ldz, p.w1 = w_post, p.s = scale, p.w2 = w_pre;
    p.r = r, p.n = n, p.ldr = ldr, p.ldn = ldn, p.rows = rows, p.cols = cols, p.eps = eps;
    const int rpb = cols <= 512 ? 4 : 1;
    const long blocks = (rows + rpb - 1) / rpb;
    return bn_dispatch<false>(dtype, cols, vec, [&](auto* e, auto v, auto nv, auto wpr) {
        using E = std::remove_pointer_t<decltype(e)>;
        constexpr int V = decltype(v)::value, NV = decltype(nv)::value, WPR = decltype(wpr)::value;
        if (!grid_fits(blocks, NV ? bn_threads<WPR>() : BW_NT)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows", fn);
        int q = pre_launch("block_norm_fwd");
        if (q) return q;
        const hipStream_t st = as_stream(stream);
        if constexpr (NV == 0)
            hipLaunchKernelGGL((block_norm_fwd_wide_k<E, V>), dim3((unsigned)blocks), dim3(BW_NT), 0, st, p);
        else
            hipLaunchKernelGGL((block_norm_fwd_k<E, V, NV, WPR>), dim3((unsigned)blocks), dim3(bn_threads<WPR>()), 0, st, p);
        return post_launch("block_norm_fwd");
    });
}

int asca_block_norm_bwd(const void* x, long ldx, const void* y, long ldy, const void* z, long ldz, const float* w_post,
                        const float* scale, const float* w_pre, const void* dr, long lddr, const void* dn, long lddn,
                        void* dx, long lddx, void* dy, long lddy, void* dz, long lddz, float* dw_post, float* dscale,
                        float* dw_pre, long rows, int cols, float eps, int dtype, void* stream) {
    const char* fn = "asca_block_norm_bwd";
    if (rows < 0 || cols < 0) return fail(ASCA_ERR_INVALID, "%s: negative shape", fn);
    if (!(eps >= 0.0f)) return fail(ASCA_ERR_INVALID, "%s: eps=%g", fn, (double)eps);
    int rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; });
    if (rc) return rc;
    if (!y && (z || w_post || scale)) return fail(ASCA_ERR_INVALID, "%s: z, w_post or scale without y", fn);
    if ((dx && !x) || (dy && !y) || (dz && !z) || (dw_post && !w_post) || (dscale && !scale) || (dw_pre && !w_pre))
        return fail(ASCA_ERR_INVALID, "%s: a gradient of an input that is NULL", fn);
    if (cols == 0) return ASCA_OK;
    if (rows > 0 && ((!x && !y) || (!dr && !dn))) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if ((rc = bn_row_check(fn, "ldx", x, ldx, cols)) || (rc = bn_row_check(fn, "ldy", y, ldy, cols)) ||
        (rc = bn_row_check(fn, "ldz", z, ldz, cols)) || (rc = bn_row_check(fn, "lddr", dr, lddr, cols)) ||
        (rc = bn_row_check(fn, "lddn", dn, lddn, cols)) || (rc = bn_row_check(fn, "lddx", dx, lddx, cols)) ||
        (rc = bn_row_check(fn, "lddy", dy, lddy, cols)) || (rc = bn_row_check(fn, "lddz", dz, lddz, cols)))
        return rc;
    auto rows_ok = [&](const void* a, long ld) { return act_vec_ok(a, ld, dtype); };
    auto par_ok = [&](const float* a) { return reinterpret_cast<uintptr_t>(a) % 16 == 0; };
    const bool vec = cols % 4 == 0 && rows_ok(x, ldx) && rows_ok(y, ldy) && rows_ok(z, ldz) && rows_ok(dr, lddr) &&
                     rows_ok(dn, lddn) && rows_ok(dx, lddx) && rows_ok(dy, lddy) && rows_ok(dz, lddz) && par_ok(w_post) &&
                     par_ok(scale) && par_ok(w_pre);
    const hipStream_t st = as_stream(stream);
    NormArgs p{};
    p.x = x, p.y = y, p.z = z, p.ldx = ldx, p.ldy = ldy, p.ldz = ldz, p.w1 = w_post, p.s = scale, p.w2 = w_pre;
    p.dr = dr, p.dn = dn, p.lddr = lddr, p.lddn = lddn, p.dx = dx, p.dy = dy, p.dz = dz;
    p.lddx = lddx, p.lddy = lddy, p.lddz = lddz, p.rows = rows, p.cols = cols, p.eps = eps;
    const int rpb = cols <= 512 ? 4 : 1;
    // what the CUs hold at once: each block is two waves a SIMD's registers allow
    const long held = cols > 512 && cols <= 1024 ? 1024 : 512;
    const long blocks = std::min((rows + rpb - 1) / rpb, held);
    const bool sums = dw_post || dscale || dw_pre;
    StreamScratch sc;
    if (sums && (rc = sc.get((size_t)blocks * 3 * cols, st))) return rc;
    p.part = sc.ws.p;
    if (blocks)
        rc = bn_dispatch<true>(dtype, cols, vec, [&](auto* e, auto v, auto nv, auto wpr) {
            using E = std::remove_pointer_t<decltype(e)>;
            constexpr int V = decltype(v)::value, NV = decltype(nv)::value, WPR = decltype(wpr)::value;
            int q = pre_launch("block_norm_bwd");
            if (q) return q;
            if constexpr (NV == 0)
                hipLaunchKernelGGL((block_norm_bwd_wide_k<E, V>), dim3((unsigned)blocks), dim3(BW_NT), 0, st, p);
            else
                hipLaunchKernelGGL((block_norm_bwd_k<E, V, NV, WPR>), dim3((unsigned)blocks), dim3(bn_threads<WPR>()), 0,
                                   st, p);
            return post_launch("block_norm_bwd");
        });
    if (rc || !sums) return rc;
    return sum_parts_launch(p.part, blocks, PartsOut{{dw_post, dscale, dw_pre}, {cols, cols, cols}}, st);
}

}  // extern "C"
