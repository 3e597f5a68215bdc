// Causal depthwise convolution: forward, backward, and one row for many
// sequences.  Per channel, with W taps:
//   p_t = bias + sum_j w_j x_{t-W+1+j},  y = p or silu(p)
//   g = dy (silu'(p));  dx_t = sum_j w_j g_{t+W-1-j};  dw_j = sum g_t x_{t-W+1+j}
// A thread has V neighbouring channels and a run of CV_R rows: all of a run's rows
// (and the W - 1 beside it, which a neighbour reads too) are loaded at once, then
// each is used W times from registers.  The backward forms g again for the W - 1
// rows after its run.  Bound by memory: 16 x 1024 x 512 f32, W = 4, forward 13.1 us
// (5.1 TB/s), backward 22.1 us (4.6 TB/s); 8 x 4096 x 2048 bf16 53 us (5.1) and 106 us
// (3.8: two bytes a value, and taps and sigmoid formed 11 times for 8 rows, fill part
// of the vector unit's time too).  Where four channels cannot be loaded together (a width
// or stride that is not a multiple of four, an offset) V is 1: 8 x 4096 x 2047 bf16 82 and
// 219 us, 16 x 1024 x 511 f32 15.8 and 29 (512: 12.9 and 25.5, with the sums' launch).
#include "act.h"
#include "parts.h"

namespace asca {

// Rows a run, and runs a block (the backward adds their sums).  Longer runs read and
// form less twice but hold more registers: 8 x 4096 x 2048 bf16, forward and backward,
// 175 us with 8 rows, 192 with 16, 252 with 32 forward and 24 backward.
constexpr int CV_R = 8, CV_NW = 8;

struct ConvArgs {
    const void *x, *dy;
    long ldx, lddy;
    const float *w, *bias, *state_in, *dstate_out;
    const int32_t* lens;
    void *y, *dx;
    long ldy, lddx;
    float *state_out, *dstate_in, *part;
    int B, T, D, runs, silu;
};

ASCA_DEV int conv_len(const ConvArgs& p, int b) { return p.lens ? min(max(p.lens[b], 0), p.T) : p.T; }

// A wave's run: rows t0 .. t1 of sequence b; the lane's V channels start at d
struct ConvRun {
    int b, t0, t1, len, d;
    bool live, last;     // its channels exist; it is a sequence's last
};
template <int V>
ASCA_DEV ConvRun conv_run(const ConvArgs& p, unsigned block, int w) {
    const unsigned cb = (p.D + 64 * V - 1) / (64 * V);
    const long u = (long)(block / cb) * CV_NW + w;
    ConvRun r;
    r.d = (block % cb * 64 + (threadIdx.x & 63)) * V;
    r.live = r.d < p.D && u < (long)p.B * p.runs;
    r.d = min(r.d, p.D - V);
    const long v = min(u, (long)p.B * p.runs - 1);
    r.b = (int)(v / p.runs);
    r.t0 = (int)(v % p.runs) * CV_R;
    r.last = r.t0 + CV_R >= p.T;
    r.t1 = min(r.t0 + CV_R, p.T);
    r.len = conv_len(p, r.b);
    return r;
}

// Rows t .. t + N - 1 of x: the state's before row 0, zeros from the length on
template <typename E, int W, int V, int N>
ASCA_DEV void conv_rows(const ConvArgs& p, const ConvRun& r, int t, float (&x)[N][V]) {
    const E* m = static_cast<const E*>(p.x) + (long)r.b * p.T * p.ldx + r.d;
    if (t >= 0 && t + N <= r.len) {
        act_raw<V, E> raw[N];
#pragma unroll
        for (int k = 0; k < N; ++k) raw[k] = act_load_raw<V>(m + (long)(t + k) * p.ldx);
#pragma unroll
        for (int k = 0; k < N; ++k) act_values(raw[k], x[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int u = t + k;
            if (u >= 0 && u < r.len) {
                act_values(act_load_raw<V>(m + (long)u * p.ldx), x[k]);
            } else if (u < 0 && p.state_in) {
#pragma unroll
                for (int i = 0; i < V; ++i) x[k][i] = p.state_in[((long)r.b * (W - 1) + (W - 1 + u)) * p.D + r.d + i];
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) x[k][i] = 0.0f;
            }
        }
    }
}

template <int V>
ASCA_DEV void conv_params(const float* m, int d, float* out) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = m ? m[d + i] : 0.0f;
}

template <typename E, int W, int V>
__global__ __launch_bounds__(64 * CV_NW) void conv_fwd_k(ConvArgs p) {
    const ConvRun r = conv_run<V>(p, blockIdx.x, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    if (!r.live) return;
    float w[W][V], bias[V], x[CV_R + W - 1][V];
    conv_rows<E, W, V>(p, r, r.t0 - (W - 1), x);
#pragma unroll
    for (int j = 0; j < W; ++j) conv_params<V>(p.w + (long)j * p.D, r.d, w[j]);
    conv_params<V>(p.bias, r.d, bias);
    E* y = static_cast<E*>(p.y) + (long)r.b * p.T * p.ldy + r.d;
#pragma unroll
    for (int k = 0; k < CV_R; ++k) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float a = bias[i];
#pragma unroll
            for (int j = 0; j < W; ++j) a = fmaf(w[j][i], x[k + j][i], a);
            if (p.silu) a *= act_sigmoid(a);
            o[i] = r.t0 + k < r.len ? a : 0.0f;
        }
        if (r.t0 + k < r.t1) act_store_n<V>(y + (long)(r.t0 + k) * p.ldy, o);
    }
    if (p.state_out && r.last) {
        float s[W - 1][V];
        conv_rows<E, W, V>(p, r, r.len - (W - 1), s);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) p.state_out[((long)r.b * (W - 1) + j) * p.D + r.d + i] = s[j][i];
    }
}

template <typename E, int W, int V>
__global__ __launch_bounds__(64 * CV_NW) void conv_bwd_k(ConvArgs p) {
    constexpr int N = CV_R + W - 1;
    __shared__ float red[CV_NW][W + 1][64 * V];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const ConvRun r = conv_run<V>(p, blockIdx.x, wave);
    float w[W][V], bias[V], x[N + W - 1][V], g[N][V], dw[W][V], db[V];
    // g of rows t0 .. t0 + N - 1, from x of t0 - (W - 1) on
    conv_rows<E, W, V>(p, r, r.t0 - (W - 1), x);
    const E* dy = static_cast<const E*>(p.dy) + (long)r.b * p.T * p.lddy + r.d;
    act_raw<V, E> raw[N] = {};
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (p.T > 0) raw[k] = act_load_raw<V>(dy + (long)min(r.t0 + k, max(r.len - 1, 0)) * p.lddy);
#pragma unroll
    for (int j = 0; j < W; ++j) {
        conv_params<V>(p.w + (long)j * p.D, r.d, w[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] = 0.0f;
    }
    conv_params<V>(p.bias, r.d, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) db[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        act_values(raw[k], g[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float a = bias[i];
#pragma unroll
            for (int j = 0; j < W; ++j) a = fmaf(w[j][i], x[k + j][i], a);
            if (p.silu) {
                const float s = act_sigmoid(a);
                g[k][i] *= s * fmaf(a, 1.0f - s, 1.0f);
            }
            if (r.t0 + k >= r.len) g[k][i] = 0.0f;
            if (k < CV_R) {
                db[i] += g[k][i];
#pragma unroll
                for (int j = 0; j < W; ++j) dw[j][i] = fmaf(g[k][i], x[k + j][i], dw[j][i]);
            }
        }
    }
    // dx of row t0 + k from g of rows t0 + k .. t0 + k + W - 1; the first run goes back
    // to row -(W - 1), the state's (g is zero before row 0)
    E* dx = static_cast<E*>(p.dx) + (long)r.b * p.T * p.lddx + r.d;
#pragma unroll
    for (int k = -(W - 1); k < CV_R; ++k) {
        const int t = r.t0 + k, o = t - (r.len - (W - 1));
        if (!r.live || t >= r.t1 || (k < 0 && (r.t0 > 0 || !p.dstate_in))) continue;
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (k + W - 1 - j >= 0) v[i] = fmaf(w[j][i], g[k + W - 1 - j < 0 ? 0 : k + W - 1 - j][i], v[i]);
            if (p.dstate_out && o >= 0 && o < W - 1) v[i] += p.dstate_out[((long)r.b * (W - 1) + o) * p.D + r.d + i];
            if (k >= 0 && t >= r.len) v[i] = 0.0f;
        }
        if (k >= 0)
            act_store_n<V>(dx + (long)t * p.lddx, v);
        else
#pragma unroll
            for (int i = 0; i < V; ++i) p.dstate_in[((long)r.b * (W - 1) + (W - 1 + k)) * p.D + r.d + i] = v[i];
    }
    // the block's runs' dw and db, one row of partial sums
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) red[wave][j][lane * V + i] = r.live ? dw[j][i] : 0.0f;
        red[wave][W][lane * V + i] = r.live ? db[i] : 0.0f;
    }
    __syncthreads();
    const unsigned cb = (p.D + 64 * V - 1) / (64 * V);
    float* part = p.part + (long)(blockIdx.x / cb) * (W + 1) * p.D;
    for (int o = threadIdx.x; o < (W + 1) * 64 * V; o += 64 * CV_NW) {
        const int j = o / (64 * V), d = blockIdx.x % cb * 64 * V + o % (64 * V);
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < CV_NW; ++k) s += red[k][j][o % (64 * V)];
        if (d < p.D) part[(long)j * p.D + d] = s;
    }
}

// One row for each sequence, a thread a channel of one.  512 x 2048 bf16, W = 4: 6.3 us,
// its state's 25 MB at 4.7 TB/s with the rows; 1 x 512 is a launch and a load (1.7 us).
template <typename E, int W>
__global__ __launch_bounds__(256) void conv_step_k(float* __restrict__ state, ConvArgs p) {
    const unsigned cb = (p.D + 255) / 256;
    const int d = blockIdx.x % cb * 256 + threadIdx.x;
    const long s = blockIdx.x / cb;
    if (d >= p.D) return;
    float* st = state + s * (W - 1) * p.D + d;
    float a = p.bias ? p.bias[d] : 0.0f, win[W];
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) win[j] = st[(long)j * p.D];
    win[W - 1] = act_load(static_cast<const E*>(p.x) + s * p.ldx + d);
#pragma unroll
    for (int j = 0; j < W; ++j) a = fmaf(p.w[(long)j * p.D + d], win[j], a);
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) st[(long)j * p.D] = win[j + 1];
    if (p.silu) a *= act_sigmoid(a);
    act_store(static_cast<E*>(p.y) + s * p.ldy + d, a);
}

}  // namespace asca

using namespace asca;

static int conv_check(const char* fn, int B, int T, int D, int W) {
    if (B < 0 || T < 0 || D < 0) return fail(ASCA_ERR_INVALID, "%s: negative shape B=%d T=%d D=%d", fn, B, T, D);
    if (T > 1 << 30) return fail(ASCA_ERR_UNSUPPORTED, "%s: T=%d above 2^30", fn, T);
    if (W < 2 || W > 8) return fail(ASCA_ERR_UNSUPPORTED, "%s: W=%d outside 2..8", fn, W);
    return ASCA_OK;
}

static int conv_ld(const char* fn, const char* what, long ld, int cols) {
    return ld >= cols ? ASCA_OK : fail(ASCA_ERR_INVALID, "%s: row stride %s=%ld below its %d columns", fn, what, ld, cols);
}

// Calls f with the element type, the taps and the channels a thread takes
template <typename F>
static int conv_dispatch(int dtype, int W, bool vec, F f) {
    return act_dispatch(dtype, [&](auto* e) {
        auto go = [&](auto taps) {
            return vec ? f(e, taps, std::integral_constant<int, 4>{}) : f(e, taps, std::integral_constant<int, 1>{});
        };
        switch (W) {
            case 2: return go(std::integral_constant<int, 2>{});
            case 3: return go(std::integral_constant<int, 3>{});
            case 4: return go(std::integral_constant<int, 4>{});
            case 5: return go(std::integral_constant<int, 5>{});
            case 6: return go(std::integral_constant<int, 6>{});
            case 7: return go(std::integral_constant<int, 7>{});
            default: return go(std::integral_constant<int, 8>{});
        }
    });
}

// One block of `threads` for `ch` channels of `units` units each
static int conv_grid(const char* fn, long units, int D, int ch, int threads, dim3* grid) {
    const long n = units * ((D + ch - 1) / ch);
    if (!grid_fits(n, threads)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows or channels", fn);
    *grid = dim3((unsigned)n);
    return ASCA_OK;
}

extern "C" {

int asca_conv_fwd(const void* x, long ldx, const float* w, const float* bias, const float* state_in, const int32_t* lens,
                  void* y, long ldy, float* state_out, int B, int T, int D, int W, int silu, int dtype, void* stream) {
    const char* fn = "asca_conv_fwd";
    int rc = conv_check(fn, B, T, D, W);
    if (rc || (rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; }))) return rc;
    if (B == 0 || D == 0) return ASCA_OK;
    if (!w || (T > 0 && (!x || !y))) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (state_out && state_out == state_in) return fail(ASCA_ERR_INVALID, "%s: state_out must not be state_in", fn);
    if ((rc = conv_ld(fn, "ldx", ldx, D)) || (rc = conv_ld(fn, "ldy", ldy, D))) return rc;
    ConvArgs p{};
    p.x = x, p.ldx = ldx, p.w = w, p.bias = bias, p.state_in = state_in, p.lens = lens;
    p.y = y, p.ldy = ldy, p.state_out = state_out;
    p.B = B, p.T = T, p.D = D, p.runs = T > 0 ? (T + CV_R - 1) / CV_R : 1, p.silu = silu;
    dim3 grid;
    const bool vec = D % 4 == 0 && act_vec_ok(x, ldx, dtype) && act_vec_ok(y, ldy, dtype);
    if ((rc = conv_grid(fn, ((long)B * p.runs + CV_NW - 1) / CV_NW, D, vec ? 256 : 64, 64 * CV_NW, &grid))) return rc;
    return conv_dispatch(dtype, W, vec, [&](auto* e, auto taps, auto v) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r = pre_launch("conv_fwd");
        if (r) return r;
        hipLaunchKernelGGL((conv_fwd_k<E, decltype(taps)::value, decltype(v)::value>), grid, dim3(64 * CV_NW), 0,
                           as_stream(stream), p);
        return post_launch("conv_fwd");
    });
}

int asca_conv_bwd(const void* x, long ldx, const float* w, const float* bias, const float* state_in, const int32_t* lens,
                  const void* dy, long lddy, const float* dstate_out, void* dx, long lddx, float* dw, float* dbias,
                  float* dstate_in, int B, int T, int D, int W, int silu, int dtype, void* stream) {
    const char* fn = "asca_conv_bwd";
    int rc = conv_check(fn, B, T, D, W);
    if (rc || (rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; }))) return rc;
    if (D == 0) return ASCA_OK;
    if (!w || !dw || (B > 0 && T > 0 && (!x || !dy || !dx))) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (dstate_in && dstate_in == dstate_out) return fail(ASCA_ERR_INVALID, "%s: dstate_in must not be dstate_out", fn);
    if ((rc = conv_ld(fn, "ldx", ldx, D)) || (rc = conv_ld(fn, "lddy", lddy, D)) || (rc = conv_ld(fn, "lddx", lddx, D)))
        return rc;
    const hipStream_t st = as_stream(stream);
    ConvArgs p{};
    p.x = x, p.ldx = ldx, p.w = w, p.bias = bias, p.state_in = state_in, p.lens = lens, p.dy = dy, p.lddy = lddy;
    p.dstate_out = dstate_out, p.dx = dx, p.lddx = lddx, p.dstate_in = dstate_in;
    p.B = B, p.T = T, p.D = D, p.runs = T > 0 ? (T + CV_R - 1) / CV_R : 1, p.silu = silu;
    dim3 grid;
    const long parts = ((long)B * p.runs + CV_NW - 1) / CV_NW;
    const bool vec = D % 4 == 0 && act_vec_ok(x, ldx, dtype) && act_vec_ok(dy, lddy, dtype) && act_vec_ok(dx, lddx, dtype);
    if ((rc = conv_grid(fn, parts, D, vec ? 256 : 64, 64 * CV_NW, &grid))) return rc;
    StreamScratch sc;
    if ((rc = sc.get((size_t)parts * (W + 1) * D, st))) return rc;
    p.part = sc.ws.p;
    if (parts)
        rc = conv_dispatch(dtype, W, vec, [&](auto* e, auto taps, auto v) {
            using E = std::remove_pointer_t<decltype(e)>;
            int r = pre_launch("conv_bwd");
            if (r) return r;
            hipLaunchKernelGGL((conv_bwd_k<E, decltype(taps)::value, decltype(v)::value>), grid, dim3(64 * CV_NW), 0, st, p);
            return post_launch("conv_bwd");
        });
    if (rc) return rc;
    return sum_parts_launch(p.part, parts, PartsOut{{dw, dbias, nullptr}, {(long)W * D, D, 0}}, st);
}

int asca_conv_step(float* state, const void* x, long ldx, const float* w, const float* bias, void* y, long ldy, int n,
                   int D, int W, int silu, int dtype, void* stream) {
    const char* fn = "asca_conv_step";
    int rc = conv_check(fn, n, 1, D, W);
    if (rc || (rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; }))) return rc;
    if (n == 0 || D == 0) return ASCA_OK;
    if (!state || !x || !w || !y) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    dim3 grid;
    if ((rc = conv_grid(fn, n, D, 256, 256, &grid))) return rc;
    if ((rc = conv_ld(fn, "ldx", ldx, D)) || (rc = conv_ld(fn, "ldy", ldy, D))) return rc;
    ConvArgs p{};
    p.x = x, p.ldx = ldx, p.w = w, p.bias = bias, p.y = y, p.ldy = ldy, p.D = D, p.silu = silu;
    return conv_dispatch(dtype, W, false, [&](auto* e, auto taps, auto) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r = pre_launch("conv_step");
        if (r) return r;
        hipLaunchKernelGGL((conv_step_k<E, decltype(taps)::value>), grid, dim3(256), 0,
                           as_stream(stream), state, p);
        return post_launch("conv_step");
    });
}

}  // extern "C"
