"""Plain float64 definitions of the state space block's operators (causal
convolution, selective scan, block norms, gradient clipping), row after row, and
of their gradients by the formulas.  Test infrastructure: nothing in asca_amd/
imports it.  Shapes as in include/asca_hip.h; `lens` None means all T rows.
"""
from __future__ import annotations

import numpy as np

f8 = np.float64


def _f(a):
    return None if a is None else np.asarray(a, dtype=f8)


def sigmoid(v):
    t = np.exp(-np.abs(v))
    return np.where(v >= 0, 1 / (1 + t), t / (1 + t))


def _lens(lens, B, T):
    return [T] * B if lens is None else [min(max(int(n), 0), T) for n in lens]


# ------------------------------------------------------------- convolution


def conv(x, w, bias, B, state=None, lens=None, silu=True):
    """(y, state after the last row)."""
    W, D = w.shape
    T = x.shape[0] // max(B, 1)
    w, y, last = _f(w), np.zeros((B * T, D)), np.zeros((B, W - 1, D))
    for b, n in enumerate(_lens(lens, B, T)):
        rows = np.concatenate([np.zeros((W - 1, D)) if state is None else _f(state[b]), _f(x[b * T:b * T + n])])
        for t in range(n):
            p = (w * rows[t:t + W]).sum(0) + (0 if bias is None else _f(bias))
            y[b * T + t] = p * sigmoid(p) if silu else p
        last[b] = rows[n:]
    return y, last


def conv_bwd(x, w, bias, dy, B, state=None, lens=None, dstate_out=None, silu=True):
    """(dx, dw, dbias, dstate_in)."""
    W, D = w.shape
    T = x.shape[0] // max(B, 1)
    w = _f(w)
    dx, dw, db, ds = np.zeros((B * T, D)), np.zeros((W, D)), np.zeros(D), np.zeros((B, W - 1, D))
    for b, n in enumerate(_lens(lens, B, T)):
        rows = np.concatenate([np.zeros((W - 1, D)) if state is None else _f(state[b]), _f(x[b * T:b * T + n])])
        dr = np.zeros_like(rows)
        if dstate_out is not None:
            dr[n:] += _f(dstate_out[b])
        for t in range(n):
            p = (w * rows[t:t + W]).sum(0) + (0 if bias is None else _f(bias))
            s = sigmoid(p)
            g = _f(dy[b * T + t]) * (s * (1 + p * (1 - s)) if silu else 1.0)
            dw += g * rows[t:t + W]
            db += g
            dr[t:t + W] += w * g
        ds[b], dx[b * T:b * T + n] = dr[:W - 1], dr[W - 1:]
    return dx, dw, db, ds


# -------------------------------------------------------------------- scan


def _group(m, N, D, G):
    """(G*N) row of B or C -> (N, D)."""
    return np.repeat(_f(m).reshape(G, N).T, D // G, axis=1)


def ssm(x, dt, A, Bm, Cm, B, dt_bias=None, Dk=None, h0=None, lens=None, G=1, softplus=True, history=None):
    """(y, state after the last row); `history` (a list) receives every state before a row."""
    N, D = A.shape
    T = x.shape[0] // max(B, 1)
    A, y, last = _f(A), np.zeros((B * T, D)), np.zeros((B, N, D))
    for b, n in enumerate(_lens(lens, B, T)):
        h = np.zeros((N, D)) if h0 is None else _f(h0[b]).copy()
        hs = []
        for t in range(n):
            r = b * T + t
            v = _f(dt[r]) + (0 if dt_bias is None else _f(dt_bias))
            e = np.logaddexp(v, 0) if softplus else v
            xr = _f(x[r])
            hs.append(h)
            h = np.exp(e * A) * h + e * xr * _group(Bm[r], N, D, G)
            y[r] = (_group(Cm[r], N, D, G) * h).sum(0) + (0 if Dk is None else _f(Dk) * xr)
        hs.append(h)
        last[b] = h
        if history is not None:
            history.append(hs)
    return y, last


def ssm_bwd(x, dt, A, Bm, Cm, dy, B, dt_bias=None, Dk=None, h0=None, lens=None, G=1, softplus=True, dh_out=None):
    """dict of dx, ddt, ddt_bias, dA, dB, dC, dDk, dh0."""
    N, D = A.shape
    T = x.shape[0] // max(B, 1)
    hist: list = []
    ssm(x, dt, A, Bm, Cm, B, dt_bias, Dk, h0, lens, G, softplus, hist)
    A = _f(A)
    z = np.zeros
    o = dict(dx=z((B * T, D)), ddt=z((B * T, D)), ddt_bias=z(D), dA=z((N, D)), dB=z((B * T, G * N)), dC=z((B * T, G * N)),
             dDk=z(D), dh0=z((B, N, D)))
    fold = lambda m: m.reshape(N, G, D // G).sum(2).T.reshape(-1)  # noqa: E731
    for b, n in enumerate(_lens(lens, B, T)):
        carry = z((N, D)) if dh_out is None else _f(dh_out[b]).copy()
        for t in reversed(range(n)):
            r = b * T + t
            v = _f(dt[r]) + (0 if dt_bias is None else _f(dt_bias))
            e = np.logaddexp(v, 0) if softplus else v
            xr, g_y, bt = _f(x[r]), _f(dy[r]), _group(Bm[r], N, D, G)
            o["dC"][r] = fold(hist[b][t + 1] * g_y)
            g = carry + _group(Cm[r], N, D, G) * g_y
            o["dB"][r] = fold(g * e * xr)
            gb = (g * bt).sum(0)
            carry = g * np.exp(e * A)
            p = carry * hist[b][t]
            o["dx"][r] = e * gb + (0 if Dk is None else _f(Dk) * g_y)
            de = xr * gb + (p * A).sum(0)
            o["ddt"][r] = de * (sigmoid(v) if softplus else 1.0)
            o["dA"] += p * e
            o["dDk"] += g_y * xr
        o["dh0"][b] = carry
    o["ddt_bias"] = o["ddt"].sum(0)
    return o


# -------------------------------------------------------------- block norm


def _or1(a):
    return 1.0 if a is None else _f(a)


def block_norm(x, y=None, z=None, w_post=None, scale=None, w_pre=None, eps=1e-6):
    """(r, n)."""
    r = 0.0 if x is None else _f(x)
    if y is not None:
        u = _f(y) * (1.0 if z is None else _f(z) * sigmoid(_f(z)))
        r = r + _or1(scale) * _or1(w_post) * u / np.sqrt((u * u).mean(1, keepdims=True) + eps)
    return r, _or1(w_pre) * r / np.sqrt((r * r).mean(1, keepdims=True) + eps)


def block_norm_bwd(x, y, z, dr, dn, w_post=None, scale=None, w_pre=None, eps=1e-6):
    r, _ = block_norm(x, y, z, w_post, scale, w_pre, eps)
    g = np.zeros_like(r) if dr is None else _f(dr).copy()
    o = {}
    if dn is not None:
        i2 = 1 / np.sqrt((r * r).mean(1, keepdims=True) + eps)
        k = _f(dn) * _or1(w_pre)
        g = g + i2 * (k - r * i2 * (k * r * i2).mean(1, keepdims=True))
        o["dw_pre"] = (_f(dn) * r * i2).sum(0)
    else:
        o["dw_pre"] = np.zeros(r.shape[1])
    o["dx"] = g
    if y is not None:
        yv, s = _f(y), 1.0 if z is None else sigmoid(_f(z))
        gate = 1.0 if z is None else _f(z) * s
        u = yv * gate
        i1 = 1 / np.sqrt((u * u).mean(1, keepdims=True) + eps)
        uh = u * i1
        o["dscale"] = (g * uh * _or1(w_post)).sum(0)
        o["dw_post"] = (g * uh * _or1(scale)).sum(0)
        k = g * _or1(scale) * _or1(w_post)
        du = i1 * (k - uh * (k * uh).mean(1, keepdims=True))
        o["dy"] = du * gate
        if z is not None:
            o["dz"] = du * yv * s * (1 + _f(z) * (1 - s))
    return o


# ---------------------------------------------------------------- clipping


def clip(grads, max_norm):
    """(norm, factor, clipped)."""
    norm = float(np.sqrt(sum((_f(g) ** 2).sum() for g in grads)))
    c = min(1.0, max_norm / (norm + 1e-6))
    return norm, c, [_f(g) * c for g in grads]
