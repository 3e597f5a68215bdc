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
// A wave holds 64 / Q channels by Q groups of states (Q = 8, or 16 where waves are few:
// ssm_split and ssm_form), each lane the NS states of its group in registers; a block has NW
// waves, CB = 64 / Q NW channels of one sequence, and takes its rows in tiles of K:
//   - a thread reads x, dt (dy) of one channel at K / Q of the tile's rows, so loads
//     are whole rows and softplus and its like are computed once per (row, channel);
//     e and e x go through LDS to the lanes that need them, B and C beside them.  The
//     next tile's loads are in flight while a tile is scanned.
//   - sums over states (y, sum g B, sum A p) and over channels (dB, dC) are scattered
//     over the lanes that they are taken across as they are formed (a row swap or a
//     DPP move and an add for each value that remains), and the results go through
//     LDS back to the thread that owns the (row, channel), or are added over the
//     waves there.
//   - one barrier a tile: everything in LDS has two copies.
// The forward leaves the state before every tile; the backward computes a tile's
// states and decays again from it and keeps them in registers.  Partial sums of dB
// and dC over a block's channels, and of the parameters' gradients over its rows,
// are added by further kernels in a fixed order.
// Where sequences and channels give too few blocks the forward's rows are split over a
// block's waves (ssm_split_k), or the rows are cut into chunks: a first pass
// leaves what a chunk makes of a zero state (carry) and its sum of e, from which every
// chunk works out what enters it, exp(A sum e) being its decay.
//
// What bounds it is the vector unit, not memory: f32, 32 x 512 x 512, N = 16, the
// forward (51 us) issues vector instructions in 73% of its cycles and the backward
// (111 us) in 83%.  A step of a wave (8 channels) takes 21 issue slots of 4 cycles
// forward, 12 of them the recurrence's own exponentials and multiply-adds, and 52
// backward, 26 of them the recurrence's and 17 the sums'.
#include <algorithm>

#include "act.h"
#include "parts.h"

namespace asca {

constexpr float LOG2E = 1.44269504088896341f;

// Rows a tile (and between two kept states): the backward keeps 2 K NS floats a lane.
constexpr int ssm_k(int NS) { return NS <= 2 ? 16 : 8; }

// The states of a channel lie on Q lane groups (8 or 16), NS to a lane; a wave has
// 64 / Q channels and a block of NW waves SSM_CB of them.
template <int Q, int NW>
constexpr int SSM_CB = 64 / Q * NW;

struct SsmArgs {
    const void *x, *dt, *Bm, *Cm, *dy;
    long ldx, lddt, ldb, ldc, lddy;
    const float *dt_bias, *A, *Dk, *h0, *dh_out;
    const int32_t* lens;
    void *y, *dx, *ddt;
    long ldy, lddx, ldddt;
    float *h_out, *dh0;
    float* ck;                         // kept states (B, ceil(T/K), N, D)
    float* pP;                         // partial dA, dDk, ddt_bias (B nch, (N + 2) D)
    float* pBC;                        // partial dB, dC (tiles, B*T, G, 2, N)
    float *cs, *ce;                    // per chunk: its own states (B, nch, N, D), sum of e (B, nch, D)
    int T, D, N, G, Dg, tiles, softplus;
    int B, nch, ctile;                 // chunks a sequence, tiles of K rows a chunk
};

// Halves n values: out[k] = a[k] (lanes with `hi`: a[k + n/2]) of this lane and of
// the lane that CTRL brings, whose `hi` is the other
template <int CTRL, int H>
ASCA_DEV void halve_dpp(const float* a, float* out, bool hi) {
#pragma unroll
    for (int k = 0; k < H; ++k) out[k] = (hi ? a[k + H] : a[k]) + dpp<CTRL>(hi ? a[k] : a[k + H]);
}

// The value of the lane whose bit 2 is the other
ASCA_DEV float xor4(float x) {
    const int u = __float_as_int(x), lo = __builtin_amdgcn_update_dpp(u, u, 0x104, 0xF, 0x5, false);   // row_shl:4
    return __int_as_float(__builtin_amdgcn_update_dpp(lo, u, 0x114, 0xF, 0xA, false));                 // row_shr:4
}

// Sums over the B lanes that differ in the lane's highest bits (4, 8 or 16: bits 4..5,
// 3..5, 2..5) of v[0 .. B M): lane l has those of v[M (l / (64 / B)) .. + M)
template <int B, int M>
ASCA_DEV void scatter_high(const float* v, int lane, float* out) {
    float a[B / 2 * M], b[B / 4 * M];
#pragma unroll
    for (int k = 0; k < B / 2 * M; ++k) a[k] = tsum32(v[k], v[k + B / 2 * M]);
#pragma unroll
    for (int k = 0; k < B / 4 * M; ++k) b[k] = tsum16(a[k], a[k + B / 4 * M]);
    if constexpr (B == 4) {
#pragma unroll
        for (int k = 0; k < M; ++k) out[k] = b[k];
    } else if constexpr (B == 8) {
        halve_dpp<DPP_ROW_ROR8, M>(b, out, lane & 8);
    } else {
        float d[2 * M];
        halve_dpp<DPP_ROW_ROR8, 2 * M>(b, d, lane & 8);
#pragma unroll
        for (int k = 0; k < M; ++k) out[k] = (lane & 4 ? d[k + M] : d[k]) + xor4(lane & 4 ? d[k] : d[k + M]);
    }
}

// The same over the lowest bits (8 or 16 lanes): lane l has those of v[M (l % B) .. + M)
template <int B, int M>
ASCA_DEV void scatter_low(const float* v, int lane, float* out) {
    float h[8 * M], a[4 * M], b[2 * M];
    if constexpr (B == 16) {
        halve_dpp<DPP_ROW_ROR8, 8 * M>(v, h, lane & 8);
    } else {
#pragma unroll
        for (int k = 0; k < 8 * M; ++k) h[k] = v[k];
    }
    halve_dpp<DPP_HALF_MIRROR, 4 * M>(h, a, lane & 4);
    halve_dpp<DPP_QUAD_XOR2, 2 * M>(a, b, lane & 2);
    halve_dpp<DPP_QUAD_XOR1, M>(b, out, lane & 1);
}

// softplus(v) and its derivative 1 / (1 + exp(-v)).  softplus(v) = max(v, 0) +
// log(1 + t), t = exp(-|v|).  log(w) t / (w - 1) with w = 1 + t rounded is log(1 + t)
// to the last bits also where t is small (w - 1 is exact); t where w is 1.
ASCA_DEV float softplus_f(float v, float* slope) {
    const float t = __builtin_amdgcn_exp2f(-fabsf(v) * LOG2E);
    const float w = 1.0f + t, m = w - 1.0f;
    const float l = __builtin_amdgcn_logf(w) * 0.693147180559945f * t * __builtin_amdgcn_rcpf(m);
    *slope = (v >= 0.0f ? 1.0f : t) * __builtin_amdgcn_rcpf(w);
    return fmaxf(v, 0.0f) + (m == 0.0f ? t : l);
}

// A block's place, and a thread's as the owner of (row, channel) pairs: channel
// tid % CB of the block's CB, rows tid / CB + Q r of a tile
template <int Q, int CB>
struct SsmPlace {
    int b, ch, g, tile, len, own_c, own_row, own_d;
    bool own_live;
    long row0;
    ASCA_DEV explicit SsmPlace(const SsmArgs& p) {
        unsigned u = blockIdx.x;
        tile = u % p.tiles;
        u /= p.tiles;
        g = u % p.G;
        u /= p.G;
        ch = u % p.nch;
        b = u / p.nch;
        own_c = threadIdx.x % CB;
        own_row = threadIdx.x / CB;
        own_live = tile * CB + own_c < p.Dg;
        own_d = g * p.Dg + min(tile * CB + own_c, p.Dg - 1);
        len = p.lens ? min(max(p.lens[b], 0), p.T) : p.T;
        row0 = (long)b * p.T;
    }
    // the tiles of K rows that the block walks: those of its chunk that hold a row of
    // the sequence
    template <int K>
    ASCA_DEV void tiles_of(const SsmArgs& p, int* k0, int* k1) const {
        *k0 = ch * p.ctile;
        *k1 = max(*k0, min(*k0 + p.ctile, (len + K - 1) / K));
    }
    // zeros in the owned channel of the chunk's rows from tile k on
    template <int K, typename E>
    ASCA_DEV void zero_rows(const SsmArgs& p, E* m, long ld, int k) const {
        if (!own_live) return;
        const int end = min((ch + 1) * p.ctile * K, p.T);
        for (int t = k * K + own_row; t < end; t += Q) act_store(m + (long)(t - own_row) * ld, 0.0f);
    }
    // channel c of wave w
    ASCA_DEV int chan(const SsmArgs& p, int w, int c, bool* live) const {
        const int d = tile * CB + w * (64 / Q) + c;
        *live = d < p.Dg;
        return g * p.Dg + min(d, p.Dg - 1);
    }
};

// A thread's place in an activation matrix: its channel of row own_row of the
// sequence.  Rows are reached from it by uniform offsets, so a tile's addresses are
// scalar products.
template <typename E, int Q, int CB>
ASCA_DEV E* own_ptr(const SsmPlace<Q, CB>& l, const void* m, long ld) {
    return static_cast<E*>(const_cast<void*>(m)) + (l.row0 + l.own_row) * ld + l.own_d;
}

// A thread's values of the tile at t0, as they are in memory; rows past the
// sequence's end read its last row again (the reader replaces them).  No load sits
// under a condition and none is converted here: either would wait for it.
template <typename E, int Q, int CB, int R>
ASCA_DEV void own_load(const SsmPlace<Q, CB>& l, const E* m, long ld, int t0, E (&out)[R]) {
    long a[R];
#pragma unroll
    for (int r = 0; r < R; ++r) a[r] = (t0 + Q * r) * ld;
    if (t0 + Q * R > l.len)
#pragma unroll
        for (int r = 0; r < R; ++r) a[r] = (long)(min(t0 + l.own_row + Q * r, max(l.len - 1, 0)) - l.own_row) * ld;
#pragma unroll
    for (int r = 0; r < R; ++r) out[r] = m[a[r]];
}

// B and C of a tile: value o = thread + 64 NW r is (B or C, row, state), so that a
// wave's are all of one matrix.
template <typename E, int NS, int Q, int NW, int K>
struct BcTile {
    static constexpr int CB = SSM_CB<Q, NW>, V = K * Q * NS, R = (2 * V + 64 * NW - 1) / (64 * NW);
    const E* m[R];
    long ld[R];
    E v[R];
    ASCA_DEV BcTile(const SsmArgs& p, const SsmPlace<Q, CB>& l) {
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool C = (w + r * NW) * 64 % (2 * V) >= V;   // a wave past the last value reads again
            const int o = (threadIdx.x + r * 64 * NW) % V;
            ld[r] = C ? p.ldc : p.ldb;
            m[r] = static_cast<const E*>(C ? p.Cm : p.Bm) + (l.row0 + o / (Q * NS)) * ld[r] + (long)l.g * p.N +
                   min(o % (Q * NS), p.N - 1);
        }
    }
    ASCA_DEV void load(const SsmPlace<Q, CB>& l, int t0) {
        long a[R];
#pragma unroll
        for (int r = 0; r < R; ++r) a[r] = t0 * ld[r];
        if (t0 + K > l.len)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int u = (threadIdx.x + r * 64 * NW) % V / (Q * NS);
                a[r] = (long)(min(t0 + u, max(l.len - 1, 0)) - u) * ld[r];
            }
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = m[r][a[r]];
    }
    // into [row][group][B's NS, C's NS], zeros for rows and states that do not exist
    ASCA_DEV void store(const SsmArgs& p, const SsmPlace<Q, CB>& l, int t0, float* lds) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int o = threadIdx.x + r * 64 * NW, u = o % V / (Q * NS), n = o % (Q * NS);
            const float x = t0 + u < l.len && n < p.N ? act_value(v[r]) : 0.0f;
            if (2 * V % (64 * NW) == 0 || o < 2 * V) lds[((u * Q + n / NS) * 2 + o / V) * NS + n % NS] = x;
        }
    }
};

// Waits for a loaded value here: one that a loop uses first would be waited for in
// every turn of it, together with the loads that the turn itself has in flight.
ASCA_DEV void settle(float& x) { asm volatile("" : "+v"(x)); }

// LDS that only one wave writes and reads: its accesses keep their order, which the
// compiler has to know where a lane reads what another wrote.
ASCA_DEV void lds_wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// Step e of a row from its raw dt (0 past the sequence's end: the state stays)
ASCA_DEV float ssm_e(const SsmArgs& p, float v, bool in, float* slope) {
    float s = v;
    *slope = 1.0f;
    if (p.softplus) s = softplus_f(v, slope);
    return in ? s : 0.0f;
}

// Many rows' decay, exp2(x), is held as its square root and met in two factors: a growing
// state's alone may pass f32's range where the state does not.  The root is held at the
// largest value, so that it leaves a zero zero, as row by row, and takes any other normal
// number past the range, as the growth that it stands for would.  NaN stays.
ASCA_DEV float decay_root(float x) {
    const float f = __builtin_amdgcn_exp2f(0.5f * x), BIG = __int_as_float(0x7f7fffff);
    return f > BIG ? BIG : f;
}
ASCA_DEV float decayed(float f, float h, float c) { return fmaf(f * h, f, c); }

// The state (or with REV the carry) that enters a chunk: the chunks before (after) it
// in turn, each as it left its own zero start and by its decay.
template <int NS, bool REV>
ASCA_DEV void fold_chunks(const SsmArgs& p, int b, int ch, int q, int d, const float* A2, float* h) {
    const int n = REV ? p.nch - 1 - ch : ch;
    for (int k = 0; k < n; ++k) {
        const long u = (long)b * p.nch + (REV ? p.nch - 1 - k : k);
        const float e = p.ce[u * p.D + d];
#pragma unroll
        for (int j = 0; j < NS; ++j)
            h[j] = decayed(decay_root(e * A2[j]), h[j], p.cs[(u * p.N + min(q * NS + j, p.N - 1)) * p.D + d]);
    }
}

// The sum of the block's e, one a channel, into ce
template <int Q, int CB>
ASCA_DEV void store_esum(const SsmArgs& p, const SsmPlace<Q, CB>& l, float esum, float (*lds)[CB]) {
    __syncthreads();
    lds[l.own_row][l.own_c] = esum;
    __syncthreads();
    if (l.own_row || !l.own_live) return;
#pragma unroll
    for (int r = 1; r < Q; ++r) esum += lds[r][l.own_c];
    p.ce[((long)l.b * p.nch + l.ch) * p.D + l.own_d] = esum;
}

// OUT: the rows' y from the state that enters the chunk; otherwise what a chunk
// makes of a zero state, and the sum of its e.  Lane = CH q + c.  Bound by the vector
// unit's issue: 8 x 4096 x 2048 bf16, N = 16, 387 us; 1 x 16384 x 1024 bf16 in 32
// chunks 62 and 84 us.
template <typename E, int NS, int Q, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW) void ssm_fwd_k(SsmArgs p) {
    constexpr int K = ssm_k(NS), R = K / Q, CB = SSM_CB<Q, NW>, CH = 64 / Q;
    constexpr int YP = CB + 4;          // R YP is CH mod 2 CH: the groups' stores of y spread over the banks
    __shared__ float2 ex[2][K][CB];
    __shared__ float bc[2][K * Q * 2 * NS];
    __shared__ float ys[2][K][YP];
    const SsmPlace<Q, CB> l(p);
    if (!OUT && l.ch == p.nch - 1) return;   // no chunk follows
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane / CH, c = lane % CH;
    bool live;
    const int d = l.chan(p, w, c, &live);
    const int ntile = (p.T + K - 1) / K;
    int k0, k1;
    l.template tiles_of<K>(p, &k0, &k1);
    float A2[NS], h[NS], esum = 0.0f, eown = 0.0f;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const int n = q * NS + j;
        A2[j] = n < p.N ? p.A[(long)n * p.D + d] * LOG2E : 0.0f;
        h[j] = OUT && p.h0 && n < p.N ? p.h0[((long)l.b * p.N + n) * p.D + d] : 0.0f;
    }
    if (OUT) fold_chunks<NS, false>(p, l.b, l.ch, q, d, A2, h);
    float bias = p.dt_bias ? p.dt_bias[l.own_d] : 0.0f, Dk = p.Dk ? p.Dk[l.own_d] : 0.0f;
    settle(bias);
    settle(Dk);
#pragma unroll
    for (int j = 0; j < NS; ++j) settle(h[j]), settle(A2[j]);
    const E *px = own_ptr<E>(l, p.x, p.ldx), *pdt = own_ptr<E>(l, p.dt, p.lddt);
    E* py = own_ptr<E>(l, p.y, p.ldy);
    BcTile<E, NS, Q, NW, K> bct(p, l);
    E rx[R], rdt[R];
    float x[R], xk[R];
    auto fetch = [&](int k) {
        own_load(l, px, p.ldx, k * K, rx);
        own_load(l, pdt, p.lddt, k * K, rdt);
        bct.load(l, k * K);
    };
    auto stage = [&](int k, int buf) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool in = k * K + l.own_row + Q * r < l.len;
            float slope;
            const float e = ssm_e(p, act_value(rdt[r]) + bias, in, &slope);
            x[r] = in ? act_value(rx[r]) : 0.0f;
            ex[buf][l.own_row + Q * r][l.own_c] = make_float2(e, e * x[r]);
            eown += e;
        }
        bct.store(p, l, k * K, bc[buf]);
    };
    auto emit = [&](int k) {
        float v[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
            v[r] = k * K + l.own_row + Q * r < l.len ? fmaf(Dk, xk[r], ys[k & 1][l.own_row + Q * r][l.own_c]) : 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (l.own_live && k * K + l.own_row + Q * r < p.T) act_store(py + (k * K + Q * r) * p.ldy, v[r]);
    };
    if (k0 < k1) {
        fetch(k0);
        stage(k0, k0 & 1);
    }
    for (int k = k0; k < k1; ++k) {
        const int buf = k & 1, next = min(k + 1, k1 - 1);   // the last tile is read twice rather than left out
        lds_barrier();                       // tile k is staged, tile k - 1's y is summed
        if (OUT && k > k0) emit(k - 1);
#pragma unroll
        for (int r = 0; r < R; ++r) xk[r] = x[r];
        esum = eown;
        fetch(next);
        if (OUT && p.ck && live)
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (q * NS + j < p.N) p.ck[(((long)l.b * ntile + k) * p.N + q * NS + j) * p.D + d] = h[j];
        // operands are read PR rows ahead: read as they are needed, each row would wait
        // for its own (8 x 4096 x 2048 bf16: 570 -> 410 us; 4 or 8 rows ahead: 428, 446)
        constexpr int PR = 2, MS = OUT ? 2 * NS : NS;
        float2 ev[2][PR];
        float m[2][PR][MS], y[K];
        auto read = [&](int g) {
#pragma unroll
            for (int u = 0; u < PR; ++u) {
                ev[g & 1][u] = ex[buf][g * PR + u][w * CH + c];
#pragma unroll
                for (int j = 0; j < MS; ++j) m[g & 1][u][j] = bc[buf][((g * PR + u) * Q + q) * 2 * NS + j];
            }
        };
        read(0);
#pragma unroll
        for (int g = 0; g < K / PR; ++g) {
            if (g + 1 < K / PR) read(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < PR; ++u)
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    const float2 e = ev[g & 1][u];
                    const float* v = m[g & 1][u];
                    h[j] = fmaf(__builtin_amdgcn_exp2f(e.x * A2[j]), h[j], v[j] * e.y);
                    if (OUT) y[g * PR + u] = j ? fmaf(v[NS + j], h[j], y[g * PR + u]) : v[NS + j] * h[j];
                }
        }
        if (OUT) {
            float s[R];
            scatter_high<Q, R>(y, lane, s);
#pragma unroll
            for (int r = 0; r < R; ++r) ys[buf][R * q + r][w * CH + c] = s[r];
        }
        stage(next, buf ^ 1);
    }
    if (OUT) {
        if (k0 < k1) {
            lds_barrier();
            emit(k1 - 1);
        }
        l.template zero_rows<K>(p, py, p.ldy, k1);
    }
    if (!OUT) {
        if (live)
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (q * NS + j < p.N) p.cs[(((long)l.b * p.nch + l.ch) * p.N + q * NS + j) * p.D + d] = h[j];
        store_esum(p, l, esum, reinterpret_cast<float(*)[CB]>(&ys[0][0][0]));
    } else if (p.h_out && live && l.ch == p.nch - 1) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (q * NS + j < p.N) p.h_out[((long)l.b * p.N + q * NS + j) * p.D + d] = h[j];
    }
}

// The forward with a sequence's rows split over a block's waves: 64 / Q channels a
// block, wave w of it takes tiles w, w + NW, ...  In a tile every row's decay and input
// are formed once and kept in registers: first they give the states that the tile makes
// of a zero state and its sum of e, which the waves exchange and each goes through, NW of
// them, for the state that enters its own tile; then the tile's states and y.  (The local
// states and the decays' products kept instead, and the true state's share added by them:
// 16 x 1024 x 512 63 us; the inputs read and formed again, 26 registers fewer: 1 x 4096 x
// 4096 120 -> 131.)  A wave owns the rows R q .. of its tile, those that it has y
// of after the sum over states, so nothing of its own passes through another wave.
// Blocks are laid out so that neighbouring channels, which share lines of x, dt and y, run
// on one XCD.  Bound by the vector unit's issue, and
// by waiting for the block's other waves where it has a CU to itself: 16 x 1024 x 512 f32,
// N = 16, 60 us; 1 x 4096 x 2048 bf16 64 us; 1 x 512 x 512 8.5 us, two rounds.
template <typename E, int NS, int Q, int NW>
__global__ __launch_bounds__(64 * NW) void ssm_split_k(SsmArgs p) {
    constexpr int CH = 64 / Q, K = ssm_k(NS), R = K / Q, V = K * Q * NS, RB = 2 * V / 64;
    __shared__ float2 ex[NW][K][CH];
    __shared__ float bc[NW][2 * V];
    __shared__ float2 agg[2][NW][64][NS];
    const unsigned nb = p.B * p.G * p.tiles, per = (nb + 7) / 8, u = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (u >= nb) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane / CH, c = lane % CH;
    const int tile = u % p.tiles, g = u / p.tiles % p.G, b = u / p.tiles / p.G;
    const bool live = tile * CH + c < p.Dg;
    const int d = g * p.Dg + min(tile * CH + c, p.Dg - 1);
    const int len = p.lens ? min(max(p.lens[b], 0), p.T) : p.T;
    const int ntile = (p.T + K - 1) / K, rounds = ((len + K - 1) / K + NW - 1) / NW;
    const long row0 = (long)b * p.T;
    float A2[NS], h[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const int n = q * NS + j;
        A2[j] = n < p.N ? p.A[(long)n * p.D + d] * LOG2E : 0.0f;
        h[j] = p.h0 && n < p.N ? p.h0[((long)b * p.N + n) * p.D + d] : 0.0f;
    }
    float bias = p.dt_bias ? p.dt_bias[d] : 0.0f, Dk = p.Dk ? p.Dk[d] : 0.0f;
    settle(bias);
    settle(Dk);
#pragma unroll
    for (int j = 0; j < NS; ++j) settle(h[j]), settle(A2[j]);
    const E* px = static_cast<const E*>(p.x) + (row0 + R * q) * p.ldx + d;
    const E* pdt = static_cast<const E*>(p.dt) + (row0 + R * q) * p.lddt + d;
    E* py = static_cast<E*>(p.y) + (row0 + R * q) * p.ldy + d;
    // B and C of the wave's tile: value lane + 64 i
    const int bn = min(lane % (Q * NS), p.N - 1), br = lane / (Q * NS);
    constexpr int BR = 64 / (Q * NS);   // rows a value of i apart
    const E* pB = static_cast<const E*>(p.Bm) + (row0 + br) * p.ldb + (long)g * p.N + bn;
    const E* pC = static_cast<const E*>(p.Cm) + (row0 + br) * p.ldc + (long)g * p.N + bn;
    E rx[R], rdt[R], rb[RB];
    auto fetch = [&](int k) {
        const int t0 = k * K;
        if (t0 + K <= len) {
#pragma unroll
            for (int r = 0; r < R; ++r) rx[r] = px[(t0 + r) * p.ldx], rdt[r] = pdt[(t0 + r) * p.lddt];
#pragma unroll
            for (int i = 0; i < RB / 2; ++i) rb[i] = pB[(t0 + BR * i) * p.ldb], rb[RB / 2 + i] = pC[(t0 + BR * i) * p.ldc];
        } else {
            const int last = max(len - 1, 0);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const long t = min(t0 + R * q + r, last) - R * q;
                rx[r] = px[t * p.ldx], rdt[r] = pdt[t * p.lddt];
            }
#pragma unroll
            for (int i = 0; i < RB / 2; ++i) {
                const long t = min(t0 + br + BR * i, last) - br;
                rb[i] = pB[t * p.ldb], rb[RB / 2 + i] = pC[t * p.ldc];
            }
        }
    };
    if (rounds) fetch(w);
    for (int o = 0; o < rounds; ++o) {
        const int k = o * NW + w, t0 = k * K, buf = o & 1;
        float x[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool in = t0 + R * q + r < len;
            float slope;
            const float e = ssm_e(p, act_value(rdt[r]) + bias, in, &slope);
            x[r] = in ? act_value(rx[r]) : 0.0f;
            ex[w][R * q + r][c] = make_float2(e, e * x[r]);
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int r = br + BR * (i % (RB / 2)), n = lane % (Q * NS);
            const float v = t0 + r < len && n < p.N ? act_value(rb[i]) : 0.0f;
            bc[w][((r * Q + n / NS) * 2 + i / (RB / 2)) * NS + n % NS] = v;
        }
        lds_wave_order();
        fetch(min(k + NW, ntile - 1));
        // the tile from a zero state and its sum of e; decays and inputs are kept
        float a[K * NS], in[K * NS];
        float hl[NS], esum = 0.0f;
#pragma unroll
        for (int j = 0; j < NS; ++j) hl[j] = 0.0f;
        {
            constexpr int PR = 2;
            float2 ev[2][PR];
            float m[2][PR][NS];
            auto read = [&](int g) {
#pragma unroll
                for (int u = 0; u < PR; ++u) {
                    ev[g & 1][u] = ex[w][g * PR + u][c];
#pragma unroll
                    for (int j = 0; j < NS; ++j) m[g & 1][u][j] = bc[w][((g * PR + u) * Q + q) * 2 * NS + j];
                }
            };
            read(0);
#pragma unroll
            for (int g = 0; g < K / PR; ++g) {
                if (g + 1 < K / PR) read(g + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < PR; ++u) {
                    const int t = g * PR + u;
                    esum += ev[g & 1][u].x;
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        a[t * NS + j] = __builtin_amdgcn_exp2f(ev[g & 1][u].x * A2[j]);
                        in[t * NS + j] = m[g & 1][u][j] * ev[g & 1][u].y;
                        hl[j] = t ? fmaf(a[t * NS + j], hl[j], in[t * NS + j]) : in[t * NS + j];
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NS; ++j)
            agg[buf][w][lane][j] = make_float2(decay_root(esum * A2[j]), hl[j]);
        lds_barrier();
        float hin[NS];
#pragma unroll
        for (int v0 = 0; v0 < NW; v0 += 4) {   // 4 at a time: registers
            float2 f[4][NS];
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int j = 0; j < NS; ++j) f[v][j] = agg[buf][v0 + v][lane][j];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                if (v0 + v == w)
#pragma unroll
                    for (int j = 0; j < NS; ++j) hin[j] = h[j];
#pragma unroll
                for (int j = 0; j < NS; ++j) h[j] = decayed(f[v][j].x, h[j], f[v][j].y);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (p.ck && live && k < ntile)
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (q * NS + j < p.N) p.ck[(((long)b * ntile + k) * p.N + q * NS + j) * p.D + d] = hin[j];
        float y[K];
#pragma unroll
        for (int t = 0; t < K; ++t)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const float C = bc[w][((t * Q + q) * 2 + 1) * NS + j];
                hin[j] = fmaf(a[t * NS + j], hin[j], in[t * NS + j]);
                y[t] = j ? fmaf(C, hin[j], y[t]) : C * hin[j];
            }
        lds_wave_order();
        float s[R];
        scatter_high<Q, R>(y, lane, s);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (live && t0 + R * q + r < p.T) act_store(py + (t0 + r) * p.ldy, t0 + R * q + r < len ? fmaf(Dk, x[r], s[r]) : 0.0f);
    }
    if (!live) return;
    for (int t = (rounds * NW + w) * K; t < p.T; t += NW * K)
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (t + R * q + r < p.T) act_store(py + (long)(t + r) * p.ldy, 0.0f);
    if (p.h_out && w == 0)
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (q * NS + j < p.N) p.h_out[((long)b * p.N + q * NS + j) * p.D + d] = h[j];
}

// What a chunk makes of a zero carry, from its end to its start, and the sum of its e.
// Lane = CH q + c.  2 x 2048 x 1024 bf16, N = 16, in 8 chunks 22 us (and 60 us behind it
// in the backward proper).
template <typename E, int NS, int Q, int NW>
__global__ __launch_bounds__(64 * NW) void ssm_carry_k(SsmArgs p) {
    constexpr int K = ssm_k(NS), R = K / Q, CB = SSM_CB<Q, NW>, CH = 64 / Q;
    __shared__ float2 ey[2][K][CB];
    __shared__ float bc[2][K * Q * 2 * NS];
    const SsmPlace<Q, CB> l(p);
    if (l.ch == 0) return;   // no chunk precedes
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane / CH, c = lane % CH;
    bool live;
    const int d = l.chan(p, w, c, &live);
    int k0, k1;
    l.template tiles_of<K>(p, &k0, &k1);
    float A2[NS], cy[NS], esum = 0.0f, eown = 0.0f;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        A2[j] = q * NS + j < p.N ? p.A[(long)(q * NS + j) * p.D + d] * LOG2E : 0.0f;
        cy[j] = 0.0f;
    }
    float bias = p.dt_bias ? p.dt_bias[l.own_d] : 0.0f;
    settle(bias);
#pragma unroll
    for (int j = 0; j < NS; ++j) settle(A2[j]);
    const E *pdy = own_ptr<E>(l, p.dy, p.lddy), *pdt = own_ptr<E>(l, p.dt, p.lddt);
    BcTile<E, NS, Q, NW, K> bct(p, l);
    E rdy[R], rdt[R];
    auto fetch = [&](int k) {
        own_load(l, pdy, p.lddy, k * K, rdy);
        own_load(l, pdt, p.lddt, k * K, rdt);
        bct.load(l, k * K);
    };
    auto stage = [&](int k, int buf) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool in = k * K + l.own_row + Q * r < l.len;
            float slope;
            const float e = ssm_e(p, act_value(rdt[r]) + bias, in, &slope);
            ey[buf][l.own_row + Q * r][l.own_c] = make_float2(e, in ? act_value(rdy[r]) : 0.0f);
            eown += e;
        }
        bct.store(p, l, k * K, bc[buf]);
    };
    if (k0 < k1) {
        fetch(k1 - 1);
        stage(k1 - 1, (k1 - 1) & 1);
    }
    for (int k = k1 - 1; k >= k0; --k) {
        const int buf = k & 1, next = max(k - 1, k0);
        lds_barrier();
        esum = eown;
        fetch(next);
#pragma unroll
        for (int t = K - 1; t >= 0; --t) {
            const float2 e = ey[buf][t][w * CH + c];
            const float* m = bc[buf] + (t * Q + q) * 2 * NS + NS;
#pragma unroll
            for (int j = 0; j < NS; ++j) cy[j] = __builtin_amdgcn_exp2f(e.x * A2[j]) * fmaf(m[j], e.y, cy[j]);
        }
        stage(next, buf ^ 1);
    }
    if (live)
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (q * NS + j < p.N) p.cs[(((long)l.b * p.nch + l.ch) * p.N + q * NS + j) * p.D + d] = cy[j];
    store_esum(p, l, esum, reinterpret_cast<float(*)[CB]>(&ey[0][0][0]));
}

// Lane = Q c + q: sums over channels (2 NS a row) by row swaps, over states (2 a row) by
// DPP.  Bound by the vector unit's issue (85% of its cycles): 8 x 4096 x 2048 bf16, N =
// 16, 857 us.
template <typename E, int NS, int Q, int NW>
__global__ __launch_bounds__(64 * NW) void ssm_bwd_k(SsmArgs p) {
    constexpr int K = ssm_k(NS), R = K / Q, CB = SSM_CB<Q, NW>, CH = 64 / Q;
    constexpr int PR = 2, YP = CB + 4, RED = K * Q * 2 * NS;   // RED sums over channels a tile and wave
    // ... in groups of CH PG: TG rows' 2 NS, or one row's
    constexpr int TG = 2 * NS < CH ? CH / (2 * NS) : 1, PG = 2 * NS < CH ? 1 : 2 * NS / CH;
    __shared__ float2 ex[2][K][CB];
    __shared__ float dys[2][K][CB];
    __shared__ float bc[2][K * Q * 2 * NS];
    __shared__ float sums[2][2][K][YP];
    __shared__ float red[2][NW][RED];
    const SsmPlace<Q, CB> l(p);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane % Q, c = lane / Q;
    bool live;
    const int d = l.chan(p, w, c, &live);
    const int ntile = (p.T + K - 1) / K;
    int k0, k1;
    l.template tiles_of<K>(p, &k0, &k1);
    float A2[NS], cy[NS], dA[NS], hn[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const int n = q * NS + j;
        A2[j] = n < p.N ? p.A[(long)n * p.D + d] * LOG2E : 0.0f;
        cy[j] = p.dh_out && n < p.N ? p.dh_out[((long)l.b * p.N + n) * p.D + d] : 0.0f;
        dA[j] = 0.0f;
    }
    fold_chunks<NS, true>(p, l.b, l.ch, q, d, A2, cy);
    float bias = p.dt_bias ? p.dt_bias[l.own_d] : 0.0f, Dk = p.Dk ? p.Dk[l.own_d] : 0.0f;
    settle(bias);
    settle(Dk);
#pragma unroll
    for (int j = 0; j < NS; ++j) settle(cy[j]), settle(A2[j]);
    E rx[R], rdt[R], rdy[R];
    float x[R], sl[R], dy[R], e[R], dD = 0.0f, db = 0.0f, xk[R], slk[R], dyk[R], ek[R];
    const E *px = own_ptr<E>(l, p.x, p.ldx), *pdt = own_ptr<E>(l, p.dt, p.lddt), *pdy = own_ptr<E>(l, p.dy, p.lddy);
    E *pdx = own_ptr<E>(l, p.dx, p.lddx), *pddt = own_ptr<E>(l, p.ddt, p.ldddt);
    BcTile<E, NS, Q, NW, K> bct(p, l);
    const float* pck = p.ck + (long)l.b * ntile * p.N * p.D + d;
    auto fetch = [&](int k) {
        own_load(l, px, p.ldx, k * K, rx);
        own_load(l, pdt, p.lddt, k * K, rdt);
        own_load(l, pdy, p.lddy, k * K, rdy);
        bct.load(l, k * K);
        // a state that does not exist takes another's: its B and C are zero, so it reaches nothing
#pragma unroll
        for (int j = 0; j < NS; ++j) hn[j] = pck[(long)k * p.N * p.D + (long)min(q * NS + j, p.N - 1) * p.D];
    };
    auto stage = [&](int k, int buf) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool in = k * K + l.own_row + Q * r < l.len;
            e[r] = ssm_e(p, act_value(rdt[r]) + bias, in, &sl[r]);
            x[r] = in ? act_value(rx[r]) : 0.0f;
            dy[r] = in ? act_value(rdy[r]) : 0.0f;
            // a channel that does not exist adds nothing to dB and dC
            ex[buf][l.own_row + Q * r][l.own_c] = make_float2(e[r], l.own_live ? e[r] * x[r] : 0.0f);
            dys[buf][l.own_row + Q * r][l.own_c] = l.own_live ? dy[r] : 0.0f;
        }
        bct.store(p, l, k * K, bc[buf]);
    };
    // sums over channels that this thread adds over the waves: value (o / 64 PG) CH PG +
    // PG c + o / 64 % PG of the tile's (row, B or C, state), c = o % 64 / Q
    constexpr int RV = (RED + 64 * NW - 1) / (64 * NW);
    float* pred[RV];
    int red_t[RV];
#pragma unroll
    for (int i = 0; i < RV; ++i) {
        const int o = (threadIdx.x + i * 64 * NW) % RED, v = o / (64 * PG) * CH * PG + PG * (o % 64 / Q) + o / 64 % PG;
        const int t = v / (2 * NS), n = o % Q * NS + v % NS;
        red_t[i] = n < p.N && threadIdx.x + i * 64 * NW < RED ? t : 1 << 30;   // others store nothing
        pred[i] = p.pBC + ((((l.tile * (long)p.B + l.b) * p.T + t) * p.G + l.g) * 2 + v / NS % 2) * p.N + n;
    }
    auto emit = [&](int k) {
        const int buf = k & 1, t0 = k * K;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = l.own_row + Q * r, t = t0 + row;
            const bool in = t < l.len;
            const float sB = sums[buf][0][row][l.own_c], sA = sums[buf][1][row][l.own_c] * (1.0f / LOG2E);
            const float de = fmaf(xk[r], sB, sA), ddt = in ? de * slk[r] : 0.0f;
            if (l.own_live && t < p.T) {
                act_store(pdx + (t0 + Q * r) * p.lddx, in ? fmaf(ek[r], sB, Dk * dyk[r]) : 0.0f);
                act_store(pddt + (t0 + Q * r) * p.ldddt, ddt);
            }
            dD = fmaf(dyk[r], xk[r], dD);
            db += ddt;
        }
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const int o = (threadIdx.x + i * 64 * NW) % RED;
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < NW; ++u) sum += red[buf][u][o];
            if (red_t[i] + t0 < l.len) pred[i][(long)t0 * (2 * p.G * p.N)] = sum;
        }
    };
    if (k0 < k1) {
        fetch(k1 - 1);
        stage(k1 - 1, (k1 - 1) & 1);
    }
    for (int k = k1 - 1; k >= k0; --k) {
        const int buf = k & 1, next = max(k - 1, k0);
        float h0[NS], h[K * NS], a[K * NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) h0[j] = hn[j], settle(h0[j]);   // before this turn's stores
        lds_barrier();                       // tile k is staged, tile k + 1's sums are there
        if (k + 1 < k1) emit(k + 1);
#pragma unroll
        for (int r = 0; r < R; ++r) xk[r] = x[r], slk[r] = sl[r], dyk[r] = dy[r], ek[r] = e[r];
        fetch(next);
        // the tile's states and decays again, operands read PR rows ahead
        {
            float2 v[2][PR];
            float m[2][PR][NS];
            auto read = [&](int g) {
#pragma unroll
                for (int u = 0; u < PR; ++u) {
                    v[g & 1][u] = ex[buf][g * PR + u][w * CH + c];
#pragma unroll
                    for (int j = 0; j < NS; ++j) m[g & 1][u][j] = bc[buf][((g * PR + u) * Q + q) * 2 * NS + j];
                }
            };
            read(0);
#pragma unroll
            for (int g = 0; g < K / PR; ++g) {
                if (g + 1 < K / PR) read(g + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < PR; ++u)
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const int t = g * PR + u, at = t * NS + j;
                        a[at] = __builtin_amdgcn_exp2f(v[g & 1][u].x * A2[j]);
                        h[at] = fmaf(a[at], t ? h[(t ? t - 1 : 0) * NS + j] : h0[j], m[g & 1][u][j] * v[g & 1][u].y);
                    }
            }
        }
        float gB[K], pA[K], dAk[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) dAk[j] = 0.0f;
        float2 v2[2][TG];
        float dy2[2][TG], m2[2][TG][2 * NS];
        auto read = [&](int tg) {
#pragma unroll
            for (int u = 0; u < TG; ++u) {
                const int t = tg * TG + u;
                v2[tg & 1][u] = ex[buf][t][w * CH + c];
                dy2[tg & 1][u] = dys[buf][t][w * CH + c];
#pragma unroll
                for (int j = 0; j < 2 * NS; ++j) m2[tg & 1][u][j] = bc[buf][(t * Q + q) * 2 * NS + j];
            }
        };
        read(K / TG - 1);
#pragma unroll
        for (int tg = K / TG - 1; tg >= 0; --tg) {
            float part[CH * PG];
            if (tg) read(tg - 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = TG - 1; u >= 0; --u) {
                const int t = tg * TG + u;
                const float2 v = v2[tg & 1][u];
                const float dyt = dy2[tg & 1][u];
                const float* m = m2[tg & 1][u];
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    const float g = fmaf(m[NS + j], dyt, cy[j]);
                    part[u * 2 * NS + j] = g * v.y;
                    part[u * 2 * NS + NS + j] = dyt * h[t * NS + j];
                    gB[t] = j ? fmaf(m[j], g, gB[t]) : m[j] * g;
                    cy[j] = a[t * NS + j] * g;
                    const float pp = cy[j] * (t ? h[(t ? t - 1 : 0) * NS + j] : h0[j]);
                    pA[t] = j ? fmaf(A2[j], pp, pA[t]) : A2[j] * pp;
                    dAk[j] = fmaf(v.x, pp, dAk[j]);
                }
            }
            float s[PG];
            scatter_high<CH, PG>(part, lane, s);
#pragma unroll
            for (int u = 0; u < PG; ++u) red[buf][w][(tg * PG + u) * 64 + lane] = s[u];
        }
#pragma unroll
        for (int j = 0; j < NS; ++j) dA[j] += dAk[j];
        float s[R];
        scatter_low<Q, R>(gB, lane, s);
#pragma unroll
        for (int r = 0; r < R; ++r) sums[buf][0][R * q + r][w * CH + c] = s[r];
        scatter_low<Q, R>(pA, lane, s);
#pragma unroll
        for (int r = 0; r < R; ++r) sums[buf][1][R * q + r][w * CH + c] = s[r];
        stage(next, buf ^ 1);
    }
    if (k0 < k1) {
        lds_barrier();
        emit(k0);
    }
    l.template zero_rows<K>(p, pdx, p.lddx, k1);
    l.template zero_rows<K>(p, pddt, p.ldddt, k1);
    float* part = p.pP + ((long)l.b * p.nch + l.ch) * (p.N + 2) * p.D;
    if (live)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int n = q * NS + j;
            if (n < p.N) {
                part[(long)n * p.D + d] = dA[j];
                if (p.dh0 && l.ch == 0) p.dh0[((long)l.b * p.N + n) * p.D + d] = cy[j];
            }
        }
    __syncthreads();
    sums[0][0][l.own_row][l.own_c] = dD;
    sums[1][0][l.own_row][l.own_c] = db;
    __syncthreads();
    if (l.own_row == 0 && l.own_live) {
#pragma unroll
        for (int r = 1; r < Q; ++r) dD += sums[0][0][r][l.own_c], db += sums[1][0][r][l.own_c];
        part[(long)p.N * p.D + l.own_d] = dD;
        part[(long)(p.N + 1) * p.D + l.own_d] = db;
    }
}

// dB, dC from the tiles' partial sums, 8 loads in flight.  Bound by memory: 8 x 4096 x
// 2048, N = 16, 32 tiles of 64 channels, 134 MB in 28 us (4.8 TB/s).
template <typename E>
__global__ __launch_bounds__(256) void ssm_fin_bc_k(const float* __restrict__ pBC, int tiles, long rows, int T, int G, int N,
                                                   const int32_t* __restrict__ lens, E* __restrict__ dB, long lddb, E* __restrict__ dC, long lddc) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x, per = rows * G * 2 * N;
    if (i >= per) return;
    const int n = (int)(i % N), which = (int)(i / N % 2), g = (int)(i / (2 * N) % G);
    const long r = i / ((long)2 * N * G);
    float s = 0.0f;
    if (!lens || (int)(r % T) < lens[r / T])   // rows past a sequence's end have no sums
        for (int k = 0; k < tiles; k += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = pBC[min(k + u, tiles - 1) * per + i];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += k + u < tiles ? v[u] : 0.0f;
        }
    if (which == 0)
        act_store(dB + r * lddb + (long)g * N + n, s);
    else
        act_store(dC + r * lddc + (long)g * N + n, s);
}

// One row for each sequence: a thread has a channel of a sequence and goes over its
// states SU at a time, all of them loaded before any is used.  Few sequences wait
// for memory once so (1 x 512, N = 16: 4.8 us one state after another, 4.7 at SU =
// 8, 3.8 at 16; 64 x 2048 8.6, 8.1, 6.2 us); many are bound by it, and keep more
// waves with 8 (512 x 2048 37, 30.6, 32.7 us; the states are 134 MB).  With B and C of
// a wave in one load each 512 x 2048 bf16 takes 24 us, 6.0 TB/s.
ASCA_DEV float lane_value(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }

template <typename E, int SU>
__global__ __launch_bounds__(256) void ssm_step_k(float* __restrict__ h, SsmArgs p) {
    const unsigned cb = (p.D + 255) / 256;
    const int ch = blockIdx.x % cb * 256 + threadIdx.x, d = min(ch, p.D - 1), lane = threadIdx.x & 63;
    const long s = blockIdx.x / cb;
    const int g = d / p.Dg;
    const E rx = static_cast<const E*>(p.x)[s * p.ldx + d], rdt = static_cast<const E*>(p.dt)[s * p.lddt + d];
    const float bias = p.dt_bias ? p.dt_bias[d] : 0.0f, Dk = p.Dk ? p.Dk[d] : 0.0f;
    const E* Br = static_cast<const E*>(p.Bm) + s * p.ldb + (long)g * p.N;
    const E* Cr = static_cast<const E*>(p.Cm) + s * p.ldc + (long)g * p.N;
    float* hr = h + s * p.N * p.D + d;
    float e = 0.0f, xe = 0.0f, y = 0.0f, slope;
    // a wave within one group has B and C across its lanes, one load each
    const bool one = __all(g == __builtin_amdgcn_readfirstlane(g));
    const E rB = Br[min(lane, p.N - 1)], rC = Cr[min(lane, p.N - 1)];
    for (int n0 = 0; n0 < p.N; n0 += SU) {
        float a[SU], hn[SU];
        E b[SU] = {}, c[SU] = {};
#pragma unroll
        for (int u = 0; u < SU; ++u) {
            const int n = min(n0 + u, p.N - 1);
            hn[u] = hr[(long)n * p.D];
            a[u] = p.A[(long)n * p.D + d];
        }
        if (!one)
#pragma unroll
            for (int u = 0; u < SU; ++u) {
                b[u] = Br[min(n0 + u, p.N - 1)];
                c[u] = Cr[min(n0 + u, p.N - 1)];
            }
        if (n0 == 0) {
            const float x = act_value(rx);
            e = ssm_e(p, act_value(rdt) + bias, true, &slope);
            xe = e * x;
            y = Dk * x;
        }
#pragma unroll
        for (int u = 0; u < SU; ++u) {
            if (n0 + u >= p.N) break;
            const float fb = one ? lane_value(act_value(rB), n0 + u) : act_value(b[u]);
            const float fc = one ? lane_value(act_value(rC), n0 + u) : act_value(c[u]);
            const float v = fmaf(__builtin_amdgcn_exp2f(e * (a[u] * LOG2E)), hn[u], fb * xe);
            y = fmaf(fc, v, y);
            if (ch < p.D) hr[(long)(n0 + u) * p.D] = v;
        }
    }
    if (ch < p.D) act_store(static_cast<E*>(p.y) + s * p.ldy + d, y);
}

}  // namespace asca

using namespace asca;

// States a lane on 8 groups.  Those that do not exist are computed with the others: N = 4
// takes what 8 does, 12 what 16 and 24 what 32 (8 x 1024 x 2048 f32, forward and backward:
// 253 and 255 us, 325 and 328, 567 and 601).
static int ssm_ns(int N) { return N <= 8 ? 1 : N <= 16 ? 2 : N <= 32 ? 4 : 8; }

static int ssm_check(const char* fn, int B, int T, int D, int N, int G) {
    if (B < 0 || T < 0 || D < 0) return fail(ASCA_ERR_INVALID, "%s: negative shape B=%d T=%d D=%d", fn, B, T, D);
    if (T > 1 << 30) return fail(ASCA_ERR_UNSUPPORTED, "%s: T=%d above 2^30", fn, T);
    if (N < 1 || N > 64) return fail(ASCA_ERR_UNSUPPORTED, "%s: N=%d outside 1..64", fn, N);
    if (G < 1 || D % G) return fail(ASCA_ERR_INVALID, "%s: D=%d is not a multiple of G=%d", fn, D, G);
    return ASCA_OK;
}

static int ssm_ld(const char* fn, const char* what, long ld, long cols) {
    return ld >= cols ? ASCA_OK : fail(ASCA_ERR_INVALID, "%s: row stride %s=%ld below its %ld columns", fn, what, ld, cols);
}

// How a call runs: Q lane groups, NW waves a block.
struct SsmForm {
    int Q, NW;
};

// Whether a forward's rows are split over the waves of a block (ssm_split_k): it goes
// through a tile's states twice and the waves wait for each other every NW tiles, but
// fills the chip with 8 (4) channels a block and reads the rows once.  Against
// ssm_fwd_k:
//   - not where that has two waves a SIMD by itself (with states in and out, 32 x 512 x 512
//     f32: 55 us against 65, 8 x 2048 x 2048 bf16 189 against 211).
//   - below, 4 waves a block fill it (bf16, N = 16: 1 x 2048 x 12288 189 -> 154 us, x 8192
//     153 -> 112, 1 x 4096 x 4096 145 -> 122), 8 where that takes a block for every CU (1 x
//     4096 x 2048 78 -> 64 us; 98 with 4).  Just past that, rows cut into chunks are ahead
//     where they are many: 1 x 4096 x 2080, in 260 blocks, takes 120 us (with 8 waves 124;
//     cut 86), x 2560 121 (125; 101), x 3584 122 (125; 130), 1 x 1000 x 2080 33 (36; 32), x
//     4032 35 (36; 44).
//   - 16 groups of one state, 16 waves a block, where 8 groups leave half of the CUs
//     without (1 x 2048 x 1024 30 -> 23.4 us, 8 groups 29.3; 1 x 512 x 512 16 -> 8.5, 8
//     groups 10.5), with 8 waves for short sequences (128 rows: 14.8 -> 5.8 us, 7.0 with 16).
//   - where blocks are few and rows many, rows cut into chunks fill more of the chip (1 x
//     16384 x 1024 146 us, split 160; 1 x 4096 x 512 36 and 41); 1 x 2048 x 512 (128
//     blocks) takes 21 and 23, 1 x 8192 x 1024 (256) 82 and 87.  N of 17 to 32, 4 states a
//     lane: from a quarter of the rows on (1 x 128 x 512 14.7 -> 7.7 us, 1 x 2048 x 8192 245
//     -> 208; 1 x 2048 x 1024 43, split 66).
//   - N above 32 only for few and short rows: a wave has its SIMD to itself (1 x 64 x 2048,
//     N = 64: 20 -> 10 us; 1 x 512 x 512 35, split 46).
static bool ssm_split(SsmArgs& p, int N, SsmForm* f) {
    const long w8 = (long)p.B * p.G * ((p.Dg + 7) / 8);
    if (w8 >= 2048) return false;
    if (N <= 8)
        *f = {8, 8};
    else if (N <= 16 && w8 <= 128)
        *f = {16, p.T < 512 ? 8 : 16};
    else
        *f = {8, N <= 32 && w8 <= 256 && p.T >= 128 ? 8 : 4};
    p.tiles = (p.Dg + 64 / f->Q - 1) / (64 / f->Q);
    const long blocks = (long)p.B * p.G * p.tiles;
    if (N > 32) return blocks <= 256 && p.T <= 256;
    return blocks > 256 || p.T < std::max(1536L, blocks * blocks / 8) / (N > 16 ? 4 : 1);
}

// Otherwise p.nch chunks a sequence.
//   - 16 groups (N of 9 to 16) give the backward twice the waves for a sixth more
//     instructions: where 8 groups give about a wave a SIMD and 16 a block a CU at most
//     (16 x 1024 x 512 161 -> 146 us, 12 x 1024 x 512 158 -> 144; 24 x 1024 x 512, in 384
//     blocks, 225 -> 277), or where few waves cannot be cut enough (1 x 512 x 512 28 -> 26
//     us).  Of fewer waves 8 groups have three chunks or more, which are ahead (10 x 1024 x
//     512 112 us, 16 groups 143; 6 x 75 and 106; at 11 x, two chunks, 157 and 143).
//   - a cut costs a second pass over the rows, so it pays only for waves that are
//     missing: below `enough`, as many chunks as give `want` (forward: 2 x 2048 x 1024, N =
//     32, in 256 waves 244 us, cut to 4096 72; 32 x 512 x 512 in 2048 waves 55 us, cut to
//     4096 82; backward: 2 x 2048 x 1024 cut to 1024 142 us, to 2048 100).
//   - the backward has 8 waves a block, which halves its partial sums of dB and dC (8 x
//     4096 x 2048 904 -> 888 us), where that leaves a block for every CU (2 x 2048 x
//     1024 without: 89.8 -> 90.8 us).
static SsmForm ssm_form(SsmArgs& p, int N, bool bwd, long enough, long want) {
    const int K = ssm_k(ssm_ns(N)), ntile = (p.T + K - 1) / K;
    const long w8 = (long)p.B * p.G * ((p.Dg + 7) / 8), cuts = std::max(1, std::min(64, ntile / 4));
    SsmForm f{8, bwd && ssm_ns(N) < 8 && (long)p.B * p.G * ((p.Dg + 63) / 64) >= 256 ? 8 : 4};
    if (bwd && ssm_ns(N) == 2 && ((w8 >= 768 && (long)p.B * p.G * ((p.Dg + 31) / 32) <= 256) || w8 * cuts < 1024)) f = {16, 8};
    const int CB = 64 / f.Q * f.NW;
    p.tiles = (p.Dg + CB - 1) / CB;
    const long waves = (long)p.B * p.G * p.tiles * f.NW;
    const long nch = waves == 0 || waves >= enough ? 1 : std::max(1L, std::min(want / waves, cuts));
    p.ctile = std::max(1, (int)((ntile + nch - 1) / nch));
    p.nch = std::max(1, (ntile + p.ctile - 1) / p.ctile);
    return f;
}
static size_t ssm_chunk_floats(const SsmArgs& p) { return p.nch > 1 ? (size_t)p.B * p.nch * (p.N + 1) * p.D : 0; }

// Calls f with the element type, the states a lane, the lane groups and the waves a block
template <bool BWD, typename F>
static int ssm_dispatch(int dtype, int N, SsmForm form, F f) {
    return act_dispatch(dtype, [&](auto* e) {
        using std::integral_constant;
        const integral_constant<int, 8> c8;
        const integral_constant<int, 4> c4;
        if constexpr (BWD)
            if (form.Q == 16) return f(e, integral_constant<int, 1>{}, integral_constant<int, 16>{}, c8);
        auto go = [&](auto ns) {
            if constexpr (BWD)
                if (form.NW == 8) return f(e, ns, c8, c8);
            return f(e, ns, c8, c4);
        };
        switch (ssm_ns(N)) {
            case 1: return go(integral_constant<int, 1>{});
            case 2: return go(integral_constant<int, 2>{});
            case 4: return go(c4);
            default: return f(e, c8, c8, c4);
        }
    });
}

extern "C" {

int asca_ssm_ws_bytes(int B, int T, int D, int N, size_t* bytes) {
    if (!bytes) return fail(ASCA_ERR_INVALID, "null output pointer");
    int rc = ssm_check("asca_ssm_ws_bytes", B, T, D, N, 1);
    if (rc) return rc;
    const int K = ssm_k(ssm_ns(N));
    *bytes = (size_t)B * (((size_t)T + K - 1) / K) * N * D * sizeof(float);
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
    p.B = B;
    SsmForm form;
    if (ssm_split(p, N, &form)) {
        const dim3 grid((unsigned)(((long)B * G * p.tiles + 7) / 8 * 8));
        return act_dispatch(dtype, [&](auto* e) {
            using E = std::remove_pointer_t<decltype(e)>;
            auto go = [&](auto kernel) {
                int r = pre_launch("ssm_split");
                if (r) return r;
                hipLaunchKernelGGL(kernel, grid, dim3(64 * form.NW), 0, st, p);
                return post_launch("ssm_split");
            };
            if (form.Q == 16) return form.NW == 16 ? go(ssm_split_k<E, 1, 16, 16>) : go(ssm_split_k<E, 1, 16, 8>);
            switch (ssm_ns(N)) {
                case 1: return go(ssm_split_k<E, 1, 8, 8>);
                case 2: return form.NW == 8 ? go(ssm_split_k<E, 2, 8, 8>) : go(ssm_split_k<E, 2, 8, 4>);
                case 4: return form.NW == 8 ? go(ssm_split_k<E, 4, 8, 8>) : go(ssm_split_k<E, 4, 8, 4>);
                default: return go(ssm_split_k<E, 8, 8, 4>);
            }
        });
    }
    form = ssm_form(p, N, false, 1024, 4096);
    const long blocks = (long)B * p.nch * G * p.tiles;
    if (!grid_fits(blocks, 64 * form.NW)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many channels", fn);
    StreamScratch sc;
    if ((rc = sc.get(ssm_chunk_floats(p), st))) return rc;
    p.cs = sc.ws.p, p.ce = p.cs + (size_t)B * p.nch * N * D;
    return ssm_dispatch<false>(dtype, N, form, [&](auto* e, auto ns, auto q, auto nw) {
        using E = std::remove_pointer_t<decltype(e)>;
        constexpr int NS = decltype(ns)::value, Q = decltype(q)::value, W = decltype(nw)::value;
        int r;
        if (p.nch > 1) {
            if ((r = pre_launch("ssm_chunk"))) return r;
            hipLaunchKernelGGL((ssm_fwd_k<E, NS, Q, W, false>), dim3((unsigned)blocks), dim3(64 * W), 0, st, p);
            if ((r = post_launch("ssm_chunk"))) return r;
        }
        if ((r = pre_launch("ssm_fwd"))) return r;
        hipLaunchKernelGGL((ssm_fwd_k<E, NS, Q, W, true>), dim3((unsigned)blocks), dim3(64 * W), 0, st, p);
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
    p.B = B;
    const SsmForm form = ssm_form(p, N, true, 2048, 2048);
    const long blocks = (long)B * p.nch * G * p.tiles, rows = (long)B * T, parts = (long)B * p.nch, per = rows * G * 2 * N, nd = (long)N * D;
    if (!grid_fits(blocks, 64 * form.NW) || !grid_fits((per + 255) / 256, 256))
        return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows or channels", fn);
    StreamScratch sc;
    if ((rc = sc.get((size_t)parts * (nd + 2 * D) + (size_t)p.tiles * per + ssm_chunk_floats(p), st))) return rc;
    p.pP = sc.ws.p, p.pBC = p.pP + parts * (nd + 2 * D), p.cs = p.pBC + p.tiles * per;
    p.ce = p.cs + (size_t)parts * N * D;
    return ssm_dispatch<true>(dtype, N, form, [&](auto* e, auto ns, auto q, auto nw) {
        using E = std::remove_pointer_t<decltype(e)>;
        constexpr int NS = decltype(ns)::value, Q = decltype(q)::value, W = decltype(nw)::value;
        int r;
        if (p.nch > 1) {
            if ((r = pre_launch("ssm_carry"))) return r;
            hipLaunchKernelGGL((ssm_carry_k<E, NS, Q, W>), dim3((unsigned)blocks), dim3(64 * W), 0, st, p);
            if ((r = post_launch("ssm_carry"))) return r;
        }
        if (blocks) {
            if ((r = pre_launch("ssm_bwd"))) return r;
            hipLaunchKernelGGL((ssm_bwd_k<E, NS, Q, W>), dim3((unsigned)blocks), dim3(64 * W), 0, st, p);
            if ((r = post_launch("ssm_bwd"))) return r;
        }
        if (per) {
            if ((r = pre_launch("ssm_fin_bc"))) return r;
            hipLaunchKernelGGL(ssm_fin_bc_k<E>, dim3((unsigned)((per + 255) / 256)), dim3(256), 0, st, p.pBC, p.tiles, rows,
                               T, G, N, lens, static_cast<E*>(dB), lddb, static_cast<E*>(dC), lddc);
            if ((r = post_launch("ssm_fin_bc"))) return r;
        }
        return sum_parts_launch(p.pP, parts, PartsOut{{dA, dDk, ddt_bias}, {nd, D, D}}, st);
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
    if (!grid_fits(blocks, 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many channels", fn);
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
        const hipStream_t st = as_stream(stream);
        if ((long)n * D < 1 << 19)
            hipLaunchKernelGGL((ssm_step_k<E, 16>), dim3((unsigned)blocks), dim3(256), 0, st, h, p);
        else
            hipLaunchKernelGGL((ssm_step_k<E, 8>), dim3((unsigned)blocks), dim3(256), 0, st, h, p);
        return post_launch("ssm_step");
    });
}

}  // extern "C"
