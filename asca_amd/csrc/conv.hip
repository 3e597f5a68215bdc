// Causal depthwise convolution: forward, backward, and one row for many
// sequences.  Per channel, with W taps:
//   p_t = bias + sum_j w_j x_{t-W+1+j},  y = p or silu(p)
//   g = dy (silu'(p));  dx_t = sum_j w_j g_{t+W-1-j};  dw_j = sum g_t x_{t-W+1+j}
// A thread has a channel and a run of rows, and slides a window of W rows over
// it in registers, so a row is read once (and W - 1 more at a run's edge).
// Bound by memory.
#include "act.h"
#include "parts.h"

namespace asca {

constexpr int CV_FR = 32;    // rows a run, forward
constexpr int CV_BR = 64;    // backward: a run leaves W + 1 partial sums a channel

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

// x at row t of sequence b: the state's for t < 0, zero from the length on
template <typename E, int W>
ASCA_DEV float conv_x(const ConvArgs& p, int b, int t, int len, int d) {
    if (t < 0) return p.state_in ? p.state_in[((long)b * (W - 1) + (W - 1 + t)) * p.D + d] : 0.0f;
    return t < len ? act_load(static_cast<const E*>(p.x) + ((long)b * p.T + t) * p.ldx + d) : 0.0f;
}

template <typename E, int W>
__global__ __launch_bounds__(256) void conv_fwd_k(ConvArgs p) {
    const unsigned cb = (p.D + 63) / 64;
    const int d = blockIdx.x % cb * 64 + (threadIdx.x & 63);
    const long u = (long)(blockIdx.x / cb) * 4 + (threadIdx.x >> 6);
    if (d >= p.D || u >= (long)p.B * p.runs) return;
    const int b = (int)(u / p.runs), run = (int)(u % p.runs), t0 = run * CV_FR, t1 = min(t0 + CV_FR, p.T);
    const int len = conv_len(p, b);
    float w[W], win[W];
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = p.w[(long)j * p.D + d];
    const float bias = p.bias ? p.bias[d] : 0.0f;
#pragma unroll
    for (int j = 1; j < W; ++j) win[j] = conv_x<E, W>(p, b, t0 - W + j, len, d);
    E* y = static_cast<E*>(p.y) + (long)b * p.T * p.ldy + d;
    for (int t = t0; t < t1; ++t) {
#pragma unroll
        for (int j = 0; j + 1 < W; ++j) win[j] = win[j + 1];
        win[W - 1] = conv_x<E, W>(p, b, t, len, d);
        float a = bias;
#pragma unroll
        for (int j = 0; j < W; ++j) a = fmaf(w[j], win[j], a);
        if (p.silu) a *= act_sigmoid(a);
        act_store(y + (long)t * p.ldy, t < len ? a : 0.0f);
    }
    if (p.state_out && run == 0)
#pragma unroll
        for (int j = 0; j + 1 < W; ++j)
            p.state_out[((long)b * (W - 1) + j) * p.D + d] = conv_x<E, W>(p, b, len - (W - 1) + j, len, d);
}

template <typename E, int W>
__global__ __launch_bounds__(256) void conv_bwd_k(ConvArgs p) {
    const unsigned cb = (p.D + 63) / 64;
    const int d = blockIdx.x % cb * 64 + (threadIdx.x & 63);
    const long u = (long)(blockIdx.x / cb) * 4 + (threadIdx.x >> 6);
    if (d >= p.D || u >= (long)p.B * p.runs) return;
    const int b = (int)(u / p.runs), run = (int)(u % p.runs), t0 = run * CV_BR, t1 = min(t0 + CV_BR, p.T);
    const int len = conv_len(p, b);
    float w[W], win[W], gw[W], dw[W], db = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
        w[j] = p.w[(long)j * p.D + d];
        gw[j] = dw[j] = 0.0f;
    }
    const float bias = p.bias ? p.bias[d] : 0.0f;
#pragma unroll
    for (int j = 1; j < W; ++j) win[j] = conv_x<E, W>(p, b, t0 - W + j, len, d);
    const E* dy = static_cast<const E*>(p.dy) + (long)b * p.T * p.lddy + d;
    E* dx = static_cast<E*>(p.dx) + (long)b * p.T * p.lddx + d;
    // g of rows t0 .. t1 + W - 2; dx of row t - W + 1 once row t's is known
    for (int t = t0; t < t1 + W - 1; ++t) {
#pragma unroll
        for (int j = 0; j + 1 < W; ++j) {
            win[j] = win[j + 1];
            gw[j] = gw[j + 1];
        }
        win[W - 1] = conv_x<E, W>(p, b, t, len, d);
        float a = bias, g = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) a = fmaf(w[j], win[j], a);
        if (t < len) {
            g = act_load(dy + (long)t * p.lddy);
            if (p.silu) {
                const float s = act_sigmoid(a);
                g *= s * fmaf(a, 1.0f - s, 1.0f);
            }
        }
        gw[W - 1] = g;
        if (t < t1) {
            db += g;
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j] = fmaf(g, win[j], dw[j]);
        }
        const int r = t - (W - 1);   // gw[i] is g of row r + i
        if (r < t0 && !(run == 0 && r < 0)) continue;
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) v = fmaf(w[j], gw[W - 1 - j], v);
        const int o = r - (len - (W - 1));
        if (p.dstate_out && o >= 0 && o < W - 1) v += p.dstate_out[((long)b * (W - 1) + o) * p.D + d];
        if (r >= 0)
            act_store(dx + (long)r * p.lddx, r < len ? v : 0.0f);
        else if (p.dstate_in)
            p.dstate_in[((long)b * (W - 1) + (W - 1 + r)) * p.D + d] = v;
    }
    float* part = p.part + u * (W + 1) * p.D + d;
#pragma unroll
    for (int j = 0; j < W; ++j) part[(long)j * p.D] = dw[j];
    part[(long)W * p.D] = db;
}

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
    if (W < 2 || W > 8) return fail(ASCA_ERR_UNSUPPORTED, "%s: W=%d outside 2..8", fn, W);
    return ASCA_OK;
}

static int conv_ld(const char* fn, const char* what, long ld, int cols) {
    return ld >= cols ? ASCA_OK : fail(ASCA_ERR_INVALID, "%s: row stride %s=%ld below its %d columns", fn, what, ld, cols);
}

template <typename F>
static int conv_dispatch(int dtype, int W, F f) {
    return act_dispatch(dtype, [&](auto* e) {
        switch (W) {
            case 2: return f(e, std::integral_constant<int, 2>{});
            case 3: return f(e, std::integral_constant<int, 3>{});
            case 4: return f(e, std::integral_constant<int, 4>{});
            case 5: return f(e, std::integral_constant<int, 5>{});
            case 6: return f(e, std::integral_constant<int, 6>{});
            case 7: return f(e, std::integral_constant<int, 7>{});
            default: return f(e, std::integral_constant<int, 8>{});
        }
    });
}

// One block for `ch` channels of `units` units each
static int conv_grid(const char* fn, long units, int D, int ch, dim3* grid) {
    const long n = units * ((D + ch - 1) / ch);
    if (n > 0x7fffffffL) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows or channels", fn);
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
    p.B = B, p.T = T, p.D = D, p.runs = T > 0 ? (T + CV_FR - 1) / CV_FR : 1, p.silu = silu;
    dim3 grid;
    if ((rc = conv_grid(fn, ((long)B * p.runs + 3) / 4, D, 64, &grid))) return rc;
    return conv_dispatch(dtype, W, [&](auto* e, auto taps) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r = pre_launch("conv_fwd");
        if (r) return r;
        hipLaunchKernelGGL((conv_fwd_k<E, decltype(taps)::value>), grid, dim3(256), 0, as_stream(stream), p);
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
    p.B = B, p.T = T, p.D = D, p.runs = T > 0 ? (T + CV_BR - 1) / CV_BR : 1, p.silu = silu;
    dim3 grid;
    if ((rc = conv_grid(fn, ((long)B * p.runs + 3) / 4, D, 64, &grid))) return rc;
    const long parts = (long)B * p.runs;
    StreamScratch sc;
    if ((rc = sc.get((size_t)parts * (W + 1) * D, st))) return rc;
    p.part = sc.ws.p;
    if (parts)
        rc = conv_dispatch(dtype, W, [&](auto* e, auto taps) {
            using E = std::remove_pointer_t<decltype(e)>;
            int r = pre_launch("conv_bwd");
            if (r) return r;
            hipLaunchKernelGGL((conv_bwd_k<E, decltype(taps)::value>), grid, dim3(256), 0, st, p);
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
    if ((rc = conv_grid(fn, n, D, 256, &grid))) return rc;
    if ((rc = conv_ld(fn, "ldx", ldx, D)) || (rc = conv_ld(fn, "ldy", ldy, D))) return rc;
    ConvArgs p{};
    p.x = x, p.ldx = ldx, p.w = w, p.bias = bias, p.y = y, p.ldy = ldy, p.D = D, p.silu = silu;
    return conv_dispatch(dtype, W, [&](auto* e, auto taps) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r = pre_launch("conv_step");
        if (r) return r;
        hipLaunchKernelGGL((conv_step_k<E, decltype(taps)::value>), grid, dim3(256), 0,
                           as_stream(stream), state, p);
        return post_launch("conv_step");
    });
}

}  // extern "C"
