// Selective state space scan: forward, backward, and one row for many sequences.
//
//   e = softplus(dt + dt_bias);  h_tn = exp(e_t A_n) h_{t-1,n} + e_t x_t B_tn
//   y_t = sum_n C_tn h_tn + Dk x_t          (per channel d; n = 0 .. N-1)
// and back, with the carry c_tn = exp(e_{t+1} A_n) g_{t+1,n}:
//   g_tn = C_tn dy_t + c_tn;  dC_tn = sum_d dy_t h_tn;  dB_tn = sum_d g_tn e_t x_t
//   dx_t = e_t sum_n g_tn B_tn + Dk dy_t;  p_tn = exp(e_t A_n) g_tn h_{t-1,n}
//   de_t = x_t sum_n g_tn B_tn + sum_n A_n p_tn;  dA_n = sum_t e_t p_tn
//   ddt = de sigmoid(v);  ddt_bias = sum ddt;  dDk = sum dy x
// The decay depends on channel, state and row together, so no product of
// matrices appears: the work is an exponential (a quarter-rate instruction) and
// a few multiply-adds for each of them, on the vector unit.
//
// A wave holds 16 channels by 4 groups of states: lane (q, c) = 16 q + c has the
// NS = ceil(N/4) states q NS .. of channel c in registers.  Rows go in blocks of K:
//   - x, dt (dy) of a quad of rows 4i .. 4i+3 are read with lane group q on row
//     4i + q, so softplus and its like are computed once per (row, channel); two
//     kinds of row swap (v_permlane32/16_swap) give every group all four rows.
//   - B and C of a block lie across the 16 lanes of a group, value v = row NS +
//     state on lane v % 16 of register v / 16, and reach the arithmetic as a DPP
//     row broadcast.
//   - sums over states (y, sum g B, sum A p) end on the group that owns the row:
//     a transposed pair sum, three swaps for four rows.
//   - sums over channels (dB, dC) are scattered over the 16 lanes as they are
//     formed, then added over the block's waves through LDS; the tiles' partial
//     sums are added by a second kernel in a fixed order.
// The forward leaves the state before every K-th row; the backward computes a
// block's states and decays again from it and keeps them in registers.
#include <algorithm>
#include <utility>

#include "act.h"
#include "parts.h"

namespace asca {

constexpr int SSM_NW = 4;              // waves a block: 64 channels of one group
constexpr int SSM_CH = 16 * SSM_NW;
constexpr float LOG2E = 1.44269504088896341f;

// Rows a block of the scan (and between two kept states): with NS states a lane,
// the backward's registers hold 2 K NS floats of them.
constexpr int ssm_k(int NS) { return NS <= 4 ? 16 : NS == 8 ? 8 : 4; }

struct SsmArgs {
    const void *x, *dt, *Bm, *Cm, *dy;
    long ldx, lddt, ldb, ldc, lddy;
    const float *dt_bias, *A, *Dk, *h0, *dh_out;
    const int32_t* lens;
    void *y, *dx, *ddt;
    long ldy, lddx, ldddt;
    float *h_out, *dh0;
    float* ck;                         // kept states (B, ceil(T/K), 4 NS, D)
    float* pP;                         // partial dA, dDk, ddt_bias (B, (N + 2) D)
    float* pBC;                        // partial dB, dC (tiles, B*T, G, 2, N)
    int T, D, N, G, Dg, tiles, softplus;
};

template <int I>
ASCA_DEV float row_bcast(float x) {   // lane I of the lane's 16 to all of them
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + I, 0xF, 0xF, true));
}

// out[q'] = the value that lane group q' holds, in every group
ASCA_DEV void spread4(float v, float* out) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const auto a = __builtin_amdgcn_permlane32_swap(r[0], r[0], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(r[1], r[1], false, false);
    out[0] = __uint_as_float(a[0]);
    out[1] = __uint_as_float(b[0]);
    out[2] = __uint_as_float(a[1]);
    out[3] = __uint_as_float(b[1]);
}

// Sum over the four groups of v[q'], on group q'
ASCA_DEV float gather4(const float* v) { return tsum16(tsum32(v[0], v[2]), tsum32(v[1], v[3])); }

// Sums over a group's 16 lanes of 16 values: lane i has that of v[i]
ASCA_DEV float scatter16(const float* v, int c) {
    float a[8], b[4], d[2];
    const bool h8 = c & 8, h4 = c & 4, h2 = c & 2, h1 = c & 1;
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = (h8 ? v[k + 8] : v[k]) + dpp<DPP_ROW_ROR8>(h8 ? v[k] : v[k + 8]);
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = (h4 ? a[k + 4] : a[k]) + dpp<DPP_HALF_MIRROR>(h4 ? a[k] : a[k + 4]);
#pragma unroll
    for (int k = 0; k < 2; ++k) d[k] = (h2 ? b[k + 2] : b[k]) + dpp<DPP_QUAD_XOR2>(h2 ? b[k] : b[k + 2]);
    return (h1 ? d[1] : d[0]) + dpp<DPP_QUAD_XOR1>(h1 ? d[0] : d[1]);
}

template <typename F, int... I>
ASCA_DEV void unroll_(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
ASCA_DEV void unroll(F f) {
    unroll_(f, std::make_integer_sequence<int, N>{});
}

// softplus(v) = max(v, 0) + log(1 + t), t = exp(-|v|).  log(w) t / (w - 1) with
// w = 1 + t rounded is log(1 + t) to the last bits also where t is small (w - 1
// is exact); t where w is 1.
ASCA_DEV float softplus_f(float v) {
    const float t = __builtin_amdgcn_exp2f(-fabsf(v) * LOG2E);
    const float w = 1.0f + t, m = w - 1.0f;
    const float l = __builtin_amdgcn_logf(w) * 0.693147180559945f * t * __builtin_amdgcn_rcpf(m);
    return fmaxf(v, 0.0f) + (m == 0.0f ? t : l);
}

// What a lane is and reads from
struct SsmLane {
    int b, g, tile, lane, q, c, d, w, len;
    bool live;                         // its channel exists
};

ASCA_DEV SsmLane ssm_lane(const SsmArgs& p) {
    SsmLane l;
    unsigned u = blockIdx.x;
    l.tile = u % p.tiles;
    u /= p.tiles;
    l.g = u % p.G;
    l.b = u / p.G;
    l.lane = threadIdx.x & 63;
    l.w = threadIdx.x >> 6;
    l.q = l.lane >> 4;
    l.c = l.lane & 15;
    const int ch = l.tile * SSM_CH + l.w * 16 + l.c;
    l.live = ch < p.Dg;
    l.d = l.g * p.Dg + min(ch, p.Dg - 1);
    l.len = p.lens ? min(max(p.lens[l.b], 0), p.T) : p.T;
    return l;
}

// One block's B or C: value v = r 16 + c is row t0 + v / NS, state q NS + v % NS
template <typename E, int NS, int K>
ASCA_DEV void load_bc(const SsmArgs& p, const SsmLane& l, const void* m, long ld, int t0, float* out) {
#pragma unroll
    for (int r = 0; r < K * NS / 16; ++r) {
        const int v = r * 16 + l.c, t = t0 + v / NS, n = l.q * NS + v % NS;
        out[r] = t < l.len && n < p.N
                     ? act_load(static_cast<const E*>(m) + ((long)l.b * p.T + t) * ld + (long)l.g * p.N + n)
                     : 0.0f;
    }
}

template <typename E, int NS>
__global__ __launch_bounds__(64 * SSM_NW) void ssm_fwd_k(SsmArgs p) {
    constexpr int K = ssm_k(NS), NP = 4 * NS;
    const SsmLane l = ssm_lane(p);
    const long row0 = (long)l.b * p.T;
    const int nblk = (p.T + K - 1) / K;
    float A2[NS], h[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const int n = l.q * NS + j;
        A2[j] = n < p.N ? p.A[(long)n * p.D + l.d] * LOG2E : 0.0f;
        h[j] = p.h0 && n < p.N ? p.h0[((long)l.b * p.N + n) * p.D + l.d] : 0.0f;
    }
    const float bias = p.dt_bias ? p.dt_bias[l.d] : 0.0f, Dk = p.Dk ? p.Dk[l.d] : 0.0f;
    for (int k = 0; k < nblk; ++k) {
        const int t0 = k * K;
        if (p.ck && l.live)
#pragma unroll
            for (int j = 0; j < NS; ++j) p.ck[(((long)l.b * nblk + k) * NP + l.q * NS + j) * p.D + l.d] = h[j];
        float Bv[K * NS / 16], Cv[K * NS / 16], x[K / 4], e[K / 4];
        load_bc<E, NS, K>(p, l, p.Bm, p.ldb, t0, Bv);
        load_bc<E, NS, K>(p, l, p.Cm, p.ldc, t0, Cv);
#pragma unroll
        for (int i = 0; i < K / 4; ++i) {
            const int t = t0 + 4 * i + l.q;
            const bool in = t < l.len;
            x[i] = in ? act_load(static_cast<const E*>(p.x) + (row0 + t) * p.ldx + l.d) : 0.0f;
            e[i] = in ? act_load(static_cast<const E*>(p.dt) + (row0 + t) * p.lddt + l.d) : 0.0f;
        }
        unroll<K / 4>([&](auto I) {
            constexpr int i = I;
            const int t = t0 + 4 * i + l.q;
            // past the sequence's end e = 0: the state stays
            const float v = e[i] + bias, ei = t < l.len ? (p.softplus ? softplus_f(v) : v) : 0.0f;
            float es[4], xs[4], ys[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            spread4(ei, es);
            spread4(ei * x[i], xs);
            unroll<4 * NS>([&](auto V) {
                constexpr int tt = V / NS, j = V % NS, at = i * 4 * NS + V;
                const float a = __builtin_amdgcn_exp2f(es[tt] * A2[j]);
                h[j] = fmaf(a, h[j], row_bcast<at % 16>(Bv[at / 16]) * xs[tt]);
                ys[tt] = fmaf(row_bcast<at % 16>(Cv[at / 16]), h[j], ys[tt]);
            });
            const float y = gather4(ys) + Dk * x[i];
            if (l.live && t < p.T) act_store(static_cast<E*>(p.y) + (row0 + t) * p.ldy + l.d, t < l.len ? y : 0.0f);
        });
    }
    if (p.h_out && l.live)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int n = l.q * NS + j;
            if (n < p.N) p.h_out[((long)l.b * p.N + n) * p.D + l.d] = h[j];
        }
}

template <typename E, int NS>
__global__ __launch_bounds__(64 * SSM_NW) void ssm_bwd_k(SsmArgs p) {
    constexpr int K = ssm_k(NS), NP = 4 * NS, KR = K * NS / 16;
    __shared__ float red[2][SSM_NW][KR * 64];
    const SsmLane l = ssm_lane(p);
    const long row0 = (long)l.b * p.T;
    const int nblk = (p.T + K - 1) / K;
    float A2[NS], cy[NS], dA[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const int n = l.q * NS + j;
        A2[j] = n < p.N ? p.A[(long)n * p.D + l.d] * LOG2E : 0.0f;
        cy[j] = p.dh_out && n < p.N ? p.dh_out[((long)l.b * p.N + n) * p.D + l.d] : 0.0f;
        dA[j] = 0.0f;
    }
    const float bias = p.dt_bias ? p.dt_bias[l.d] : 0.0f, Dk = p.Dk ? p.Dk[l.d] : 0.0f;
    float dD = 0.0f, db = 0.0f;
    for (int k = nblk - 1; k >= 0; --k) {
        const int t0 = k * K;
        float Bv[KR], Cv[KR], x[K / 4], e[K / 4], v[K / 4], dy[K / 4], h0[NS], h[K * NS], a[K * NS];
        load_bc<E, NS, K>(p, l, p.Bm, p.ldb, t0, Bv);
        load_bc<E, NS, K>(p, l, p.Cm, p.ldc, t0, Cv);
#pragma unroll
        for (int i = 0; i < K / 4; ++i) {
            const int t = t0 + 4 * i + l.q;
            const bool in = t < l.len;
            x[i] = in ? act_load(static_cast<const E*>(p.x) + (row0 + t) * p.ldx + l.d) : 0.0f;
            v[i] = in ? act_load(static_cast<const E*>(p.dt) + (row0 + t) * p.lddt + l.d) : 0.0f;
            dy[i] = in ? act_load(static_cast<const E*>(p.dy) + (row0 + t) * p.lddy + l.d) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NS; ++j) h0[j] = p.ck[(((long)l.b * nblk + k) * NP + l.q * NS + j) * p.D + l.d];
        // the block's states and decays again
        unroll<K / 4>([&](auto I) {
            constexpr int i = I;
            v[i] += bias;
            e[i] = t0 + 4 * i + l.q < l.len ? (p.softplus ? softplus_f(v[i]) : v[i]) : 0.0f;
            float es[4], xs[4];
            spread4(e[i], es);
            spread4(e[i] * x[i], xs);
            unroll<4 * NS>([&](auto V) {
                constexpr int tt = V / NS, j = V % NS, at = i * 4 * NS + V;
                a[at] = __builtin_amdgcn_exp2f(es[tt] * A2[j]);
                h[at] = fmaf(a[at], at < NS ? h0[j] : h[at < NS ? 0 : at - NS], row_bcast<at % 16>(Bv[at / 16]) * xs[tt]);
            });
        });
        float vB[K * NS], vC[K * NS], dAk[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) dAk[j] = 0.0f;
        unroll<K / 4>([&](auto I) {
            constexpr int i = K / 4 - 1 - I;
            float es[4], xs[4], dys[4], gB[4] = {0.0f, 0.0f, 0.0f, 0.0f}, pA[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            spread4(e[i], es);
            spread4(e[i] * x[i], xs);
            spread4(dy[i], dys);
            unroll<4 * NS>([&](auto V) {
                constexpr int tt = 3 - V / NS, j = V % NS, at = (i * 4 + tt) * NS + j;
                const float g = fmaf(row_bcast<at % 16>(Cv[at / 16]), dys[tt], cy[j]);
                vC[at] = dys[tt] * h[at];
                vB[at] = g * xs[tt];
                gB[tt] = fmaf(row_bcast<at % 16>(Bv[at / 16]), g, gB[tt]);
                cy[j] = a[at] * g;
                const float pp = cy[j] * (at < NS ? h0[j] : h[at < NS ? 0 : at - NS]);
                pA[tt] = fmaf(A2[j], pp, pA[tt]);
                dAk[j] = fmaf(es[tt], pp, dAk[j]);
            });
            const int t = t0 + 4 * i + l.q;
            const bool in = t < l.len;
            const float sB = gather4(gB), sA = gather4(pA) * (1.0f / LOG2E);
            const float de = fmaf(x[i], sB, sA), ddt = p.softplus ? de * act_sigmoid(v[i]) : de;
            if (l.live && t < p.T) {
                act_store(static_cast<E*>(p.dx) + (row0 + t) * p.lddx + l.d, in ? fmaf(e[i], sB, Dk * dy[i]) : 0.0f);
                act_store(static_cast<E*>(p.ddt) + (row0 + t) * p.ldddt + l.d, in ? ddt : 0.0f);
            }
            dD = fmaf(dy[i], x[i], dD);
            db += in ? ddt : 0.0f;
        });
#pragma unroll
        for (int j = 0; j < NS; ++j) dA[j] += dAk[j];
        // dB, dC of the block: over the wave's channels, then the waves'
        __syncthreads();
#pragma unroll
        for (int r = 0; r < KR; ++r) {
            // a channel that does not exist adds nothing
            if (!l.live)
#pragma unroll
                for (int i = 0; i < 16; ++i) vB[r * 16 + i] = vC[r * 16 + i] = 0.0f;
            red[0][l.w][r * 64 + l.lane] = scatter16(vB + r * 16, l.c);
            red[1][l.w][r * 64 + l.lane] = scatter16(vC + r * 16, l.c);
        }
        __syncthreads();
        for (int o = threadIdx.x; o < 2 * KR * 64; o += 64 * SSM_NW) {
            const int s = o / (KR * 64), u = o % (KR * 64), vv = u / 64 * 16 + (u & 15);
            const int t = t0 + vv / NS, n = ((u >> 4) & 3) * NS + vv % NS;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < SSM_NW; ++w) sum += red[s][w][u];
            if (t < p.T && n < p.N)
                p.pBC[(((((long)l.tile * (gridDim.x / (p.tiles * p.G)) + l.b) * p.T + t) * p.G + l.g) * 2 + s) * p.N + n] =
                    t < l.len ? sum : 0.0f;
        }
    }
    dD = add_xor32(add_xor16(dD));
    db = add_xor32(add_xor16(db));
    if (l.live) {
        float* part = p.pP + (long)l.b * (p.N + 2) * p.D + l.d;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int n = l.q * NS + j;
            if (n < p.N) {
                part[(long)n * p.D] = dA[j];
                if (p.dh0) p.dh0[((long)l.b * p.N + n) * p.D + l.d] = cy[j];
            }
        }
        if (l.q == 0) {
            part[(long)p.N * p.D] = dD;
            part[(long)(p.N + 1) * p.D] = db;
        }
    }
}

// dB, dC from the tiles' partial sums
template <typename E>
__global__ __launch_bounds__(256) void ssm_fin_bc_k(const float* __restrict__ pBC, int tiles, long rows, int G, int N,
                                                   E* __restrict__ dB, long lddb, E* __restrict__ dC, long lddc) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x, per = rows * G * 2 * N;
    if (i >= per) return;
    float s = 0.0f;
    for (int k = 0; k < tiles; ++k) s += pBC[k * per + i];
    const int n = (int)(i % N), which = (int)(i / N % 2), g = (int)(i / (2 * N) % G);
    const long r = i / ((long)2 * N * G);
    if (which == 0)
        act_store(dB + r * lddb + (long)g * N + n, s);
    else
        act_store(dC + r * lddc + (long)g * N + n, s);
}

// One row for each sequence: a thread has a channel of a sequence.
template <typename E>
__global__ __launch_bounds__(256) void ssm_step_k(float* __restrict__ h, SsmArgs p) {
    const unsigned cb = (p.D + 255) / 256;
    const int d = blockIdx.x % cb * 256 + threadIdx.x;
    const long s = blockIdx.x / cb;
    if (d >= p.D) return;
    const int g = d / p.Dg;
    const float x = act_load(static_cast<const E*>(p.x) + s * p.ldx + d);
    const float v = act_load(static_cast<const E*>(p.dt) + s * p.lddt + d) + (p.dt_bias ? p.dt_bias[d] : 0.0f);
    const float e = p.softplus ? softplus_f(v) : v, ex = e * x;
    const E* Br = static_cast<const E*>(p.Bm) + s * p.ldb + (long)g * p.N;
    const E* Cr = static_cast<const E*>(p.Cm) + s * p.ldc + (long)g * p.N;
    float* hr = h + s * p.N * p.D + d;
    float y = p.Dk ? p.Dk[d] * x : 0.0f;
    for (int n = 0; n < p.N; ++n) {
        const float a = __builtin_amdgcn_exp2f(e * (p.A[(long)n * p.D + d] * LOG2E));
        const float hn = fmaf(a, hr[(long)n * p.D], act_load(Br + n) * ex);
        hr[(long)n * p.D] = hn;
        y = fmaf(act_load(Cr + n), hn, y);
    }
    act_store(static_cast<E*>(p.y) + s * p.ldy + d, y);
}

}  // namespace asca

using namespace asca;

static int ssm_ns(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

static int ssm_check(const char* fn, int B, int T, int D, int N, int G) {
    if (B < 0 || T < 0 || D < 0) return fail(ASCA_ERR_INVALID, "%s: negative shape B=%d T=%d D=%d", fn, B, T, D);
    if (N < 1 || N > 64) return fail(ASCA_ERR_UNSUPPORTED, "%s: N=%d outside 1..64", fn, N);
    if (G < 1 || D % G) return fail(ASCA_ERR_INVALID, "%s: D=%d is not a multiple of G=%d", fn, D, G);
    return ASCA_OK;
}

static int ssm_ld(const char* fn, const char* what, long ld, long cols) {
    return ld >= cols ? ASCA_OK : fail(ASCA_ERR_INVALID, "%s: row stride %s=%ld below its %ld columns", fn, what, ld, cols);
}

// Calls f with the element type and the compile-time states a lane
template <typename F>
static int ssm_dispatch(int dtype, int N, F f) {
    return act_dispatch(dtype, [&](auto* e) {
        switch (ssm_ns(N)) {
            case 1: return f(e, std::integral_constant<int, 1>{});
            case 2: return f(e, std::integral_constant<int, 2>{});
            case 4: return f(e, std::integral_constant<int, 4>{});
            case 8: return f(e, std::integral_constant<int, 8>{});
            default: return f(e, std::integral_constant<int, 16>{});
        }
    });
}

extern "C" {

int asca_ssm_ws_bytes(int B, int T, int D, int N, size_t* bytes) {
    if (!bytes) return fail(ASCA_ERR_INVALID, "null output pointer");
    int rc = ssm_check("asca_ssm_ws_bytes", B, T, D, N, 1);
    if (rc) return rc;
    const int ns = ssm_ns(N), K = ssm_k(ns);
    *bytes = (size_t)B * (((size_t)T + K - 1) / K) * 4 * ns * D * sizeof(float);
    return ASCA_OK;
}

int asca_ssm_fwd(const void* x, long ldx, const void* dt, long lddt, const float* dt_bias, const float* A,
                 const void* Bm, long ldb, const void* Cm, long ldc, const float* Dk, const float* h0,
                 const int32_t* lens, void* y, long ldy, float* h_out, void* ws, int B, int T, int D, int N, int G,
                 int softplus, int dtype, void* stream) {
    const char* fn = "asca_ssm_fwd";
    int rc = ssm_check(fn, B, T, D, N, G);
    if (rc || (rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; }))) return rc;
    if (B == 0 || D == 0) return ASCA_OK;
    const hipStream_t st = as_stream(stream);
    if (!A) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (T > 0 && (!x || !dt || !Bm || !Cm || !y)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (h_out && h_out == h0) return fail(ASCA_ERR_INVALID, "%s: h_out must not be h0", fn);
    if ((rc = ssm_ld(fn, "ldx", ldx, D)) || (rc = ssm_ld(fn, "lddt", lddt, D)) || (rc = ssm_ld(fn, "ldy", ldy, D)) ||
        (rc = ssm_ld(fn, "ldb", ldb, (long)G * N)) || (rc = ssm_ld(fn, "ldc", ldc, (long)G * N)))
        return rc;
    SsmArgs p{};
    p.x = x, p.dt = dt, p.Bm = Bm, p.Cm = Cm, p.ldx = ldx, p.lddt = lddt, p.ldb = ldb, p.ldc = ldc;
    p.dt_bias = dt_bias, p.A = A, p.Dk = Dk, p.h0 = h0, p.lens = lens, p.y = y, p.ldy = ldy, p.h_out = h_out;
    p.ck = static_cast<float*>(ws);
    p.T = T, p.D = D, p.N = N, p.G = G, p.Dg = D / G, p.softplus = softplus;
    p.tiles = (p.Dg + SSM_CH - 1) / SSM_CH;
    const long blocks = (long)B * G * p.tiles;
    if (blocks > 0x7fffffffL) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many channels", fn);
    return ssm_dispatch(dtype, N, [&](auto* e, auto ns) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r = pre_launch("ssm_fwd");
        if (r) return r;
        hipLaunchKernelGGL((ssm_fwd_k<E, decltype(ns)::value>), dim3((unsigned)blocks), dim3(64 * SSM_NW), 0, st, p);
        return post_launch("ssm_fwd");
    });
}

int asca_ssm_bwd(const void* x, long ldx, const void* dt, long lddt, const float* dt_bias, const float* A,
                 const void* Bm, long ldb, const void* Cm, long ldc, const float* Dk, const int32_t* lens,
                 const void* dy, long lddy, const float* dh_out, const void* ws, void* dx, long lddx, void* ddt,
                 long ldddt, float* ddt_bias, float* dA, void* dB, long lddb, void* dC, long lddc, float* dDk,
                 float* dh0, int B, int T, int D, int N, int G, int softplus, int dtype, void* stream) {
    const char* fn = "asca_ssm_bwd";
    int rc = ssm_check(fn, B, T, D, N, G);
    if (rc || (rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; }))) return rc;
    if (D == 0) return ASCA_OK;
    if (!A || !dA) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (B > 0 && T > 0 && (!x || !dt || !Bm || !Cm || !dy || !ws || !dx || !ddt || !dB || !dC))
        return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (dh0 && dh0 == dh_out) return fail(ASCA_ERR_INVALID, "%s: dh0 must not be dh_out", fn);
    if ((rc = ssm_ld(fn, "ldx", ldx, D)) || (rc = ssm_ld(fn, "lddt", lddt, D)) || (rc = ssm_ld(fn, "lddy", lddy, D)) ||
        (rc = ssm_ld(fn, "lddx", lddx, D)) || (rc = ssm_ld(fn, "ldddt", ldddt, D)) ||
        (rc = ssm_ld(fn, "ldb", ldb, (long)G * N)) || (rc = ssm_ld(fn, "ldc", ldc, (long)G * N)) ||
        (rc = ssm_ld(fn, "lddb", lddb, (long)G * N)) || (rc = ssm_ld(fn, "lddc", lddc, (long)G * N)))
        return rc;
    const hipStream_t st = as_stream(stream);
    SsmArgs p{};
    p.x = x, p.dt = dt, p.Bm = Bm, p.Cm = Cm, p.dy = dy;
    p.ldx = ldx, p.lddt = lddt, p.ldb = ldb, p.ldc = ldc, p.lddy = lddy;
    p.dt_bias = dt_bias, p.A = A, p.Dk = Dk, p.dh_out = dh_out, p.lens = lens;
    p.dx = dx, p.lddx = lddx, p.ddt = ddt, p.ldddt = ldddt, p.dh0 = dh0;
    p.ck = static_cast<float*>(const_cast<void*>(ws));
    p.T = T, p.D = D, p.N = N, p.G = G, p.Dg = D / G, p.softplus = softplus;
    p.tiles = (p.Dg + SSM_CH - 1) / SSM_CH;
    const long blocks = (long)B * G * p.tiles, rows = (long)B * T, per = rows * G * 2 * N, nd = (long)N * D;
    if (blocks > 0x7fffffffL || (per + 255) / 256 > 0x7fffffffL)
        return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows or channels", fn);
    StreamScratch sc;
    if ((rc = sc.get((size_t)B * (nd + 2 * D) + (size_t)p.tiles * per, st))) return rc;
    p.pP = sc.ws.p, p.pBC = p.pP + B * (nd + 2 * D);
    return ssm_dispatch(dtype, N, [&](auto* e, auto ns) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r;
        if (blocks) {
            if ((r = pre_launch("ssm_bwd"))) return r;
            hipLaunchKernelGGL((ssm_bwd_k<E, decltype(ns)::value>), dim3((unsigned)blocks), dim3(64 * SSM_NW), 0, st, p);
            if ((r = post_launch("ssm_bwd"))) return r;
        }
        if (per) {
            if ((r = pre_launch("ssm_fin_bc"))) return r;
            hipLaunchKernelGGL(ssm_fin_bc_k<E>, dim3((unsigned)((per + 255) / 256)), dim3(256), 0, st, p.pBC, p.tiles, rows,
                               G, N, static_cast<E*>(dB), lddb, static_cast<E*>(dC), lddc);
            if ((r = post_launch("ssm_fin_bc"))) return r;
        }
        return sum_parts_launch(p.pP, B, PartsOut{{dA, dDk, ddt_bias}, {nd, D, D}}, st);
    });
}

int asca_ssm_step(float* h, const void* x, long ldx, const void* dt, long lddt, const float* dt_bias, const float* A,
                  const void* Bm, long ldb, const void* Cm, long ldc, const float* Dk, void* y, long ldy, int n, int D,
                  int N, int G, int softplus, int dtype, void* stream) {
    const char* fn = "asca_ssm_step";
    int rc = ssm_check(fn, n, 1, D, N, G);
    if (rc || (rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; }))) return rc;
    if (n == 0 || D == 0) return ASCA_OK;
    if (!h || !x || !dt || !A || !Bm || !Cm || !y) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    const long blocks = (long)n * ((D + 255) / 256);
    if (blocks > 0x7fffffffL) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many channels", fn);
    if ((rc = ssm_ld(fn, "ldx", ldx, D)) || (rc = ssm_ld(fn, "lddt", lddt, D)) || (rc = ssm_ld(fn, "ldy", ldy, D)) ||
        (rc = ssm_ld(fn, "ldb", ldb, (long)G * N)) || (rc = ssm_ld(fn, "ldc", ldc, (long)G * N)))
        return rc;
    SsmArgs p{};
    p.x = x, p.dt = dt, p.Bm = Bm, p.Cm = Cm, p.ldx = ldx, p.lddt = lddt, p.ldb = ldb, p.ldc = ldc;
    p.dt_bias = dt_bias, p.A = A, p.Dk = Dk, p.y = y, p.ldy = ldy;
    p.D = D, p.N = N, p.G = G, p.Dg = D / G, p.softplus = softplus;
    return act_dispatch(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r = pre_launch("ssm_step");
        if (r) return r;
        hipLaunchKernelGGL(ssm_step_k<E>, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), h, p);
        return post_launch("ssm_step");
    });
}

}  // extern "C"
