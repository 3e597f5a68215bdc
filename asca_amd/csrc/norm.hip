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
// the forward it computes again from x, y and z.  Bound by memory.
#include <algorithm>

#include "act.h"
#include "parts.h"

namespace asca {

constexpr int BN_MAX = 16384;   // columns: 16 waves of 16 values a lane

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

// VEC values at column c of a row (zeros past its end; cols is a multiple of VEC)
template <int VEC, typename E>
ASCA_DEV void row_load(const E* row, int c, int cols, float* v) {
    if (VEC == 1 || c >= cols) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = c < cols ? act_load(row + c + k) : 0.0f;
    } else if constexpr (sizeof(E) == 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(row + c);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = a[k & 3];
    } else {
        const uint2 a = *reinterpret_cast<const uint2*>(row + c);
        v[0] = __uint_as_float(a.x << 16);
        if constexpr (VEC == 4) {
            v[1] = __uint_as_float(a.x & 0xffff0000u);
            v[2] = __uint_as_float(a.y << 16);
            v[3] = __uint_as_float(a.y & 0xffff0000u);
        }
    }
}

template <int VEC, typename E>
ASCA_DEV void row_store(E* row, int c, int cols, const float* v) {
    if (c >= cols) return;
    if constexpr (VEC == 1) {
        act_store(row + c, v[0]);
    } else if constexpr (sizeof(E) == 4) {
        *reinterpret_cast<f32x4*>(row + c) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
        bf16_t b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) act_store(b + k, v[k]);
        *reinterpret_cast<uint2*>(row + c) = make_uint2(b[0] | (unsigned)b[1] << 16, b[2] | (unsigned)b[3] << 16);
    }
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

// The same in 64 bits
template <int WPR>
ASCA_DEV double row_sum(double x, double* lds) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) x += __shfl_xor(x, s, 64);
    if constexpr (WPR > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0;
#pragma unroll
        for (int w = 0; w < WPR; ++w) x += lds[w];
    }
    return x;
}

template <int WPR>
constexpr int bn_threads() { return WPR == 1 ? 256 : 64 * WPR; }

// A row: u, r, y, silu(z), z and the two inverse norms.  The backward takes the
// sums of its rows in 64 bits: k - uh mean(k uh) cancels where k is near a multiple
// of uh (always in a row of one column), and the products of f32 values are exact there.
template <typename S, int NE>
struct BnRow {
    float u[NE], r[NE], y[NE], sz[NE], z[NE];
    S i1, i2;
};

template <typename S, typename E, int VEC, int NV, int WPR>
ASCA_DEV void bn_row(const NormArgs& p, long row, int tid, bool second, S* lds, BnRow<S, VEC * NV>& o) {
    constexpr int NE = VEC * NV;
    S ss = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + tid) * VEC;
        if (p.x) row_load<VEC>(static_cast<const E*>(p.x) + row * p.ldx, c, p.cols, o.r + i * VEC);
        if (p.y) row_load<VEC>(static_cast<const E*>(p.y) + row * p.ldy, c, p.cols, o.y + i * VEC);
        if (p.z) row_load<VEC>(static_cast<const E*>(p.z) + row * p.ldz, c, p.cols, o.z + i * VEC);
    }
    if (!p.x)
#pragma unroll
        for (int e = 0; e < NE; ++e) o.r[e] = 0.0f;
    if (p.y) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            o.sz[e] = p.z ? o.z[e] * act_sigmoid(o.z[e]) : 1.0f;
            o.u[e] = o.y[e] * o.sz[e];
            ss += (S)o.u[e] * (S)o.u[e];
        }
        o.i1 = 1 / sqrt(row_sum<WPR>(ss, lds) / (S)p.cols + (S)p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * WPR + tid) * VEC;
            float w1[VEC], s[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) w1[k] = s[k] = 1.0f;
            if (p.w1) row_load<VEC>(p.w1, c, p.cols, w1);
            if (p.s) row_load<VEC>(p.s, c, p.cols, s);
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                o.r[i * VEC + k] = fmaf(s[k], o.u[i * VEC + k] * (float)o.i1 * w1[k], o.r[i * VEC + k]);
        }
    }
    if (second) {
        ss = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) ss += (S)o.r[e] * (S)o.r[e];
        o.i2 = 1 / sqrt(row_sum<WPR>(ss, lds) / (S)p.cols + (S)p.eps);
    }
}

template <typename E, int VEC, int NV, int WPR>
__global__ __launch_bounds__(bn_threads<WPR>()) void block_norm_fwd_k(NormArgs p) {
    __shared__ float lds[16];
    constexpr int RPB = bn_threads<WPR>() / (64 * WPR);
    const long row = (long)blockIdx.x * RPB + threadIdx.x / (64 * WPR);
    const int tid = threadIdx.x % (64 * WPR);
    if (row >= p.rows) return;
    BnRow<float, VEC * NV> o;
    bn_row<float, E, VEC, NV, WPR>(p, row, tid, p.n != nullptr, lds, o);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + tid) * VEC;
        if (p.r) row_store<VEC>(static_cast<E*>(p.r) + row * p.ldr, c, p.cols, o.r + i * VEC);
        if (p.n) {
            float w2[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) w2[k] = 1.0f;
            if (p.w2) row_load<VEC>(p.w2, c, p.cols, w2);
#pragma unroll
            for (int k = 0; k < VEC; ++k) w2[k] *= o.r[i * VEC + k] * o.i2;
            row_store<VEC>(static_cast<E*>(p.n) + row * p.ldn, c, p.cols, w2);
        }
    }
}

template <typename E, int VEC, int NV, int WPR>
__global__ __launch_bounds__(bn_threads<WPR>()) void block_norm_bwd_k(NormArgs p) {
    constexpr int NE = VEC * NV, NT = bn_threads<WPR>(), RPB = NT / (64 * WPR);
    __shared__ double lds[16];
    __shared__ float acc[RPB > 1 ? NT * NE : 1];
    const int sub = threadIdx.x / (64 * WPR), tid = threadIdx.x % (64 * WPR);
    float g1[NE], gs[NE], g2[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) g1[e] = gs[e] = g2[e] = 0.0f;
    for (long row = (long)blockIdx.x * RPB + sub; row < p.rows; row += (long)gridDim.x * RPB) {
        BnRow<double, NE> o;
        float dr[NE], dn[NE];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * WPR + tid) * VEC;
            if (p.dr) row_load<VEC>(static_cast<const E*>(p.dr) + row * p.lddr, c, p.cols, dr + i * VEC);
            if (p.dn) row_load<VEC>(static_cast<const E*>(p.dn) + row * p.lddn, c, p.cols, dn + i * VEC);
        }
        if (!p.dr)
#pragma unroll
            for (int e = 0; e < NE; ++e) dr[e] = 0.0f;
        bn_row<double, E, VEC, NV, WPR>(p, row, tid, p.dn != nullptr, lds, o);
        if (p.dn) {
            const float i2 = (float)o.i2;
            double m = 0.0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 64 * WPR + tid) * VEC;
                float w2[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) w2[k] = 1.0f;
                if (p.w2) row_load<VEC>(p.w2, c, p.cols, w2);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = i * VEC + k;
                    g2[e] = fmaf(dn[e], o.r[e] * i2, g2[e]);
                    dn[e] *= w2[k];
                    m = fma((double)dn[e], (double)o.r[e], m);
                }
            }
            m = row_sum<WPR>(m, lds) / p.cols * (o.i2 * o.i2);
#pragma unroll
            for (int e = 0; e < NE; ++e) dr[e] = fmaf(i2, (float)fma(-(double)o.r[e], m, (double)dn[e]), dr[e]);
        }
        if (p.dx)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                row_store<VEC>(static_cast<E*>(p.dx) + row * p.lddx, (i * 64 * WPR + tid) * VEC, p.cols, dr + i * VEC);
        if (p.y) {
            const float i1 = (float)o.i1;
            double m = 0.0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 64 * WPR + tid) * VEC;
                float w1[VEC], s[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) w1[k] = s[k] = 1.0f;
                if (p.w1) row_load<VEC>(p.w1, c, p.cols, w1);
                if (p.s) row_load<VEC>(p.s, c, p.cols, s);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = i * VEC + k;
                    const float ru = dr[e] * (o.u[e] * i1);
                    gs[e] = fmaf(ru, w1[k], gs[e]);
                    g1[e] = fmaf(ru, s[k], g1[e]);
                    dr[e] *= s[k] * w1[k];
                    m = fma((double)dr[e], (double)o.u[e], m);
                }
            }
            m = row_sum<WPR>(m, lds) / p.cols * (o.i1 * o.i1);
#pragma unroll
            for (int e = 0; e < NE; ++e) dr[e] = i1 * (float)fma(-(double)o.u[e], m, (double)dr[e]);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 64 * WPR + tid) * VEC;
                float v[VEC];
                if (p.dy) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) v[k] = dr[i * VEC + k] * o.sz[i * VEC + k];
                    row_store<VEC>(static_cast<E*>(p.dy) + row * p.lddy, c, p.cols, v);
                }
                if (p.z && p.dz) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        const float z = o.z[i * VEC + k], sg = act_sigmoid(z);
                        v[k] = dr[i * VEC + k] * o.y[i * VEC + k] * (sg * fmaf(z, 1.0f - sg, 1.0f));
                    }
                    row_store<VEC>(static_cast<E*>(p.dz) + row * p.lddz, c, p.cols, v);
                }
            }
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

}  // namespace asca

using namespace asca;

// Calls f with (element type, VEC, NV, WPR): 16-byte (bf16: 8-byte) access where
// every row and the parameters allow it, a wave a row up to 1024 columns, 4 up to
// 4096, else 16.
template <typename F>
static int bn_dispatch(int dtype, int cols, bool vec, F f) {
    return act_dispatch(dtype, [&](auto* e) {
        auto go = [&](auto v, auto nv, auto wpr) { return f(e, v, nv, wpr); };
        using std::integral_constant;
        const integral_constant<int, 1> c1;
        const integral_constant<int, 2> c2;
        const integral_constant<int, 4> c4;
        const integral_constant<int, 16> c16;
        if (vec) {
            if (cols <= 256) return go(c4, c1, c1);
            if (cols <= 512) return go(c4, c2, c1);
            if (cols <= 1024) return go(c4, c4, c1);
            if (cols <= 4096) return go(c4, c4, c4);
            return go(c4, c4, c16);
        }
        if (cols <= 256) return go(c1, c4, c1);
        if (cols <= 1024) return go(c1, c16, c1);
        if (cols <= 4096) return go(c1, c16, c4);
        return go(c1, c16, c16);
    });
}

// Rows a block takes for `cols` columns
static int bn_rpb(int cols) { return cols <= 1024 ? 4 : 1; }

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
    int rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; });
    if (rc) return rc;
    if (cols > BN_MAX) return fail(ASCA_ERR_UNSUPPORTED, "%s: cols=%d above %d", fn, cols, BN_MAX);
    if (!y && (z || w_post || scale)) return fail(ASCA_ERR_INVALID, "%s: z, w_post or scale without y", fn);
    if (!n && w_pre) return fail(ASCA_ERR_INVALID, "%s: w_pre without n", fn);
    if (rows == 0 || cols == 0) return ASCA_OK;
    if ((!x && !y) || (!r && !n)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if ((rc = bn_row_check(fn, "ldx", x, ldx, cols)) || (rc = bn_row_check(fn, "ldy", y, ldy, cols)) ||
        (rc = bn_row_check(fn, "ldz", z, ldz, cols)) || (rc = bn_row_check(fn, "ldr", r, ldr, cols)) ||
        (rc = bn_row_check(fn, "ldn", n, ldn, cols)))
        return rc;
    const size_t size = dtype == ASCA_F32 ? 4 : 2;
    bool vec = cols % 4 == 0;
    auto rows_ok = [&](const void* a, long ld) {
        return !a || (ld % 4 == 0 && reinterpret_cast<uintptr_t>(a) % (4 * size) == 0);
    };
    auto par_ok = [&](const float* a) { return reinterpret_cast<uintptr_t>(a) % 16 == 0; };
    vec = vec && rows_ok(x, ldx) && rows_ok(y, ldy) && rows_ok(z, ldz) && rows_ok(r, ldr) && rows_ok(n, ldn) &&
          par_ok(w_post) && par_ok(scale) && par_ok(w_pre);
    NormArgs p{};
    p.x = x, p.y = y, p.z = z, p.ldx = ldx, p.ldy = ldy, p.ldz = ldz, p.w1 = w_post, p.s = scale, p.w2 = w_pre;
    p.r = r, p.n = n, p.ldr = ldr, p.ldn = ldn, p.rows = rows, p.cols = cols, p.eps = eps;
    const long blocks = (rows + bn_rpb(cols) - 1) / bn_rpb(cols);
    if (blocks > 0x7fffffffL) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows", fn);
    return bn_dispatch(dtype, cols, vec, [&](auto* e, auto v, auto nv, auto wpr) {
        using E = std::remove_pointer_t<decltype(e)>;
        constexpr int V = decltype(v)::value, NV = decltype(nv)::value, WPR = decltype(wpr)::value;
        int q = pre_launch("block_norm_fwd");
        if (q) return q;
        hipLaunchKernelGGL((block_norm_fwd_k<E, V, NV, WPR>), dim3((unsigned)blocks), dim3(bn_threads<WPR>()), 0,
                           as_stream(stream), p);
        return post_launch("block_norm_fwd");
    });
}

int asca_block_norm_bwd(const void* x, long ldx, const void* y, long ldy, const void* z, long ldz, const float* w_post,
                        const float* scale, const float* w_pre, const void* dr, long lddr, const void* dn, long lddn,
                        void* dx, long lddx, void* dy, long lddy, void* dz, long lddz, float* dw_post, float* dscale,
                        float* dw_pre, long rows, int cols, float eps, int dtype, void* stream) {
    const char* fn = "asca_block_norm_bwd";
    if (rows < 0 || cols < 0) return fail(ASCA_ERR_INVALID, "%s: negative shape", fn);
    int rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; });
    if (rc) return rc;
    if (cols > BN_MAX) return fail(ASCA_ERR_UNSUPPORTED, "%s: cols=%d above %d", fn, cols, BN_MAX);
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
    const size_t size = dtype == ASCA_F32 ? 4 : 2;
    auto rows_ok = [&](const void* a, long ld) {
        return !a || (ld % 4 == 0 && reinterpret_cast<uintptr_t>(a) % (4 * size) == 0);
    };
    auto par_ok = [&](const float* a) { return reinterpret_cast<uintptr_t>(a) % 16 == 0; };
    const bool vec = cols % 4 == 0 && rows_ok(x, ldx) && rows_ok(y, ldy) && rows_ok(z, ldz) && rows_ok(dr, lddr) &&
                     rows_ok(dn, lddn) && rows_ok(dx, lddx) && rows_ok(dy, lddy) && rows_ok(dz, lddz) && par_ok(w_post) &&
                     par_ok(scale) && par_ok(w_pre);
    const hipStream_t st = as_stream(stream);
    NormArgs p{};
    p.x = x, p.y = y, p.z = z, p.ldx = ldx, p.ldy = ldy, p.ldz = ldz, p.w1 = w_post, p.s = scale, p.w2 = w_pre;
    p.dr = dr, p.dn = dn, p.lddr = lddr, p.lddn = lddn, p.dx = dx, p.dy = dy, p.dz = dz;
    p.lddx = lddx, p.lddy = lddy, p.lddz = lddz, p.rows = rows, p.cols = cols, p.eps = eps;
    const long blocks = std::min((rows + bn_rpb(cols) - 1) / bn_rpb(cols), 1024L);
    const bool sums = dw_post || dscale || dw_pre;
    StreamScratch sc;
    if (sums && (rc = sc.get((size_t)blocks * 3 * cols, st))) return rc;
    p.part = sc.ws.p;
    if (blocks)
        rc = bn_dispatch(dtype, cols, vec, [&](auto* e, auto v, auto nv, auto wpr) {
            using E = std::remove_pointer_t<decltype(e)>;
            constexpr int V = decltype(v)::value, NV = decltype(nv)::value, WPR = decltype(wpr)::value;
            int q = pre_launch("block_norm_bwd");
            if (q) return q;
            hipLaunchKernelGGL((block_norm_bwd_k<E, V, NV, WPR>), dim3((unsigned)blocks), dim3(bn_threads<WPR>()), 0, st,
                               p);
            return post_launch("block_norm_bwd");
        });
    if (rc || !sums) return rc;
    return sum_parts_launch(p.part, blocks, PartsOut{{dw_post, dscale, dw_pre}, {cols, cols, cols}}, st);
}

}  // extern "C"
