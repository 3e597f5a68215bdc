"""The float64 oracle of the state space block's operators: every gradient
formula against central differences of the forward, and identities of the
forward (a sequence cut in two, rows past a length).  CPU only."""
import numpy as np
import pytest

from oracle import ssm_oracle as so

STEP, TOL = 1e-5, 1e-8   # central differences in float64: error of step^2 and of 1e-16 / step


def _numeric(f, a, probe):
    """d f / d a along `probe`, by a central difference."""
    return (f(a + STEP * probe) - f(a - STEP * probe)) / (2 * STEP)


def _check(f, args, grads, rng):
    """Each gradient's product with a random direction against the difference."""
    for k, g in grads.items():
        d = rng.standard_normal(np.shape(args[k]))
        want = _numeric(lambda v: f({**args, k: v}), args[k], d)
        got = float((g * d).sum())
        assert abs(got - want) <= TOL * max(1.0, abs(want)) * 50, (k, got, want)


@pytest.mark.parametrize("B,T,D,W,lens,silu", [(2, 5, 3, 4, None, True), (3, 6, 2, 3, [0, 1, 6], True), (1, 2, 3, 5, None, False)])
def test_conv_gradients(B, T, D, W, lens, silu):
    rng = np.random.default_rng(W * 10 + T)
    a = dict(x=rng.standard_normal((B * T, D)), w=rng.standard_normal((W, D)), bias=rng.standard_normal(D),
             state=rng.standard_normal((B, W - 1, D)))
    dy, ds = rng.standard_normal((B * T, D)), rng.standard_normal((B, W - 1, D))

    def f(v):
        y, s = so.conv(v["x"], v["w"], v["bias"], B, v["state"], lens, silu)
        return float((y * dy).sum() + (s * ds).sum())

    dx, dw, db, dst = so.conv_bwd(a["x"], a["w"], a["bias"], dy, B, a["state"], lens, ds, silu)
    _check(f, a, dict(x=dx, w=dw, bias=db, state=dst), rng)


@pytest.mark.parametrize("B,T,D,N,G,lens,softplus", [(2, 6, 4, 3, 1, None, True), (3, 5, 6, 2, 3, [0, 1, 5], True),
                                                     (1, 4, 2, 5, 2, None, False)])
def test_ssm_gradients(B, T, D, N, G, lens, softplus):
    rng = np.random.default_rng(N * 10 + T)
    a = dict(x=rng.standard_normal((B * T, D)), dt=rng.uniform(0.1, 0.9, (B * T, D)), A=-rng.uniform(0.5, 2, (N, D)),
             Bm=rng.standard_normal((B * T, G * N)), Cm=rng.standard_normal((B * T, G * N)), dt_bias=rng.standard_normal(D) * 0.1,
             Dk=rng.standard_normal(D), h0=rng.standard_normal((B, N, D)))
    dy, dh = rng.standard_normal((B * T, D)), rng.standard_normal((B, N, D))
    run = lambda v: so.ssm(v["x"], v["dt"], v["A"], v["Bm"], v["Cm"], B, v["dt_bias"], v["Dk"], v["h0"], lens, G, softplus)  # noqa: E731

    def f(v):
        y, h = run(v)
        return float((y * dy).sum() + (h * dh).sum())

    g = so.ssm_bwd(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], dy, B, a["dt_bias"], a["Dk"], a["h0"], lens, G, softplus, dh)
    _check(f, a, dict(x=g["dx"], dt=g["ddt"], A=g["dA"], Bm=g["dB"], Cm=g["dC"], dt_bias=g["ddt_bias"], Dk=g["dDk"], h0=g["dh0"]),
           rng)


@pytest.mark.parametrize("have", ["x y z", "x y", "y z", "x"])
def test_block_norm_gradients(have):
    rng = np.random.default_rng(len(have))
    a = {k: rng.standard_normal((4, 7)) for k in have.split()}
    a.update({k: rng.standard_normal(7) + 1 for k in (("w_post", "scale", "w_pre") if "y" in a else ("w_pre",))})
    dr, dn = rng.standard_normal((4, 7)), rng.standard_normal((4, 7))
    kw = lambda v: {k: v.get(k) for k in ("w_post", "scale", "w_pre")}  # noqa: E731

    def f(v):
        r, n = so.block_norm(v.get("x"), v.get("y"), v.get("z"), **kw(v))
        return float((r * dr).sum() + (n * dn).sum())

    g = so.block_norm_bwd(a.get("x"), a.get("y"), a.get("z"), dr, dn, **kw(a))
    _check(f, a, {k: g["d" + k] for k in a}, rng)


def test_a_sequence_cut_in_two_is_the_sequence():
    rng = np.random.default_rng(3)
    T, D, N, W, k = 9, 4, 3, 4, 5
    x, dt = rng.standard_normal((T, D)), rng.standard_normal((T, D))
    A, Bm, Cm = -rng.uniform(0.5, 2, (N, D)), rng.standard_normal((T, N)), rng.standard_normal((T, N))
    y, h = so.ssm(x, dt, A, Bm, Cm, 1)
    y1, h1 = so.ssm(x[:k], dt[:k], A, Bm[:k], Cm[:k], 1)
    y2, h2 = so.ssm(x[k:], dt[k:], A, Bm[k:], Cm[k:], 1, h0=h1)
    np.testing.assert_allclose(np.concatenate([y1, y2]), y, rtol=1e-13, atol=1e-13)
    np.testing.assert_allclose(h2, h, rtol=1e-13, atol=1e-13)
    w = rng.standard_normal((W, D))
    c, s = so.conv(x, w, None, 1)
    c1, s1 = so.conv(x[:2], w, None, 1)
    c2, s2 = so.conv(x[2:], w, None, 1, state=s1)
    np.testing.assert_allclose(np.concatenate([c1, c2]), c, rtol=1e-13, atol=1e-13)
    np.testing.assert_array_equal(s2, s)


def test_clip_of_a_known_list():
    norm, c, out = so.clip([np.array([3.0]), np.array([[4.0]])], 1.0)
    assert norm == 5.0 and abs(c - 0.2) < 1e-6 and abs(out[1][0, 0] - 0.8) < 1e-6
    assert so.clip([np.array([3.0])], 10.0)[1] == 1.0
