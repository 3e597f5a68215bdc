"""GPU parity of the state space block's operators (causal convolution, selective
scan, block norms, gradient clipping) against the float64 oracle, through the
operator API and the C ABI.

Tolerances (max|d| / max|ref|, as elsewhere): 2e-5 for f32 forwards and 1e-4 for
f32 gradients; a bf16 result may be half a unit of its 8-bit significand off the
oracle's (2^-9 of itself) and is allowed twice that, 2^-8, for what f32 arithmetic
moves it over a rounding boundary."""
import ctypes as C

import numpy as np
import pytest

from oracle import ssm_oracle as so

pytestmark = pytest.mark.gpu

FWD, GRAD, BF = 2e-5, 1e-4, 2.0 ** -8


def err(got, ref):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape and np.isfinite(got).all()
    m = np.abs(ref).max() if ref.size else 0.0
    d = np.abs(got - ref).max() if ref.size else 0.0
    return d / m if m else d


class Rows:
    """Random activation rows in a type: what the device gets, and its float64 values."""

    def __init__(self, rng, bf16):
        from asca_amd import gpu

        self.rng, self.bf16, self.g = rng, bf16, gpu

    def __call__(self, *shape, scale=1.0):
        a = (self.rng.standard_normal(shape) * scale).astype(np.float32)
        return self.dev(a)

    def dev(self, a):
        return self.g.to_bf16(a) if self.bf16 else a

    def val(self, a):
        return self.g.from_bf16(a) if a is not None and a.dtype == np.uint16 else a

    def tol(self, base):
        return BF if self.bf16 else base


def check(label, pairs):
    worst = {k: err(a, b) for k, a, b, _ in pairs}
    print(f"[{label}] " + " ".join(f"{k} {v:.1e}" for k, v in worst.items()), flush=True)
    for k, _, _, tol in pairs:
        assert worst[k] <= tol, (k, worst[k], tol)


def ragged(B, T):
    """Lengths from zero and one to all of T, and values outside 0..T."""
    return [[T, 0, 1, T + 5, -3, T // 2, max(T - 1, 0)][i % 7] for i in range(B)]


# ------------------------------------------------------------- convolution

CONV = [(1, 1, 1, 4, False), (2, 3, 5, 4, True), (7, 40, 64, 4, True), (2, 70, 130, 2, True), (3, 65, 33, 3, False),
        (2, 129, 257, 4, False), (2, 33, 20, 8, True), (1, 10, 7, 5, False), (1, 9, 68, 6, True), (2, 9, 12, 7, True),
        (1, 1000, 512, 4, False), (4, 2, 16, 4, True)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,T,D,W,rag", CONV)
def test_conv(g, B, T, D, W, rag, bf16):
    print(f"[conv] B={B} T={T} D={D} W={W} ragged={rag} bf16={bf16}", flush=True)
    rng = np.random.default_rng(B * 1000 + T + D + W)
    r = Rows(rng, bf16)
    x, dy, w, bias = r(B * T, D), r(B * T, D), rng.standard_normal((W, D)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    st, ds = (rng.standard_normal((B, W - 1, D)).astype(np.float32) for _ in range(2))
    lens = ragged(B, T) if rag else None
    for silu in (True, False):
        y, s = g.conv(x, w, bias, batch=B, state=st, lens=lens, silu=silu)
        ry, rs = so.conv(r.val(x), w, bias, B, st, lens, silu)
        got = g.conv_bwd(x, w, bias, dy, batch=B, state=st, lens=lens, dstate_out=ds, silu=silu)
        ref = so.conv_bwd(r.val(x), w, bias, r.val(dy), B, st, lens, ds, silu)
        check("conv", [("y", r.val(y), ry, r.tol(FWD)), ("state", s, rs, 0.0), ("dx", r.val(got[0]), ref[0], r.tol(GRAD)),
                       ("dw", got[1], ref[1], GRAD), ("db", got[2], ref[2], GRAD), ("ds", got[3], ref[3], GRAD)])


def test_conv_without_bias_and_state(g):
    rng = np.random.default_rng(1)
    x, dy, w = (rng.standard_normal(s).astype(np.float32) for s in ((60, 33), (60, 33), (4, 33)))
    y, s = g.conv(x, w, batch=2)
    got = g.conv_bwd(x, w, None, dy, batch=2)
    ref = so.conv_bwd(x, w, None, dy, 2)
    ry, rs = so.conv(x, w, None, 2)
    check("conv plain", [("y", y, ry, FWD), ("state", s, rs, 0.0)] + [(k, a, b, GRAD) for k, a, b in zip(("dx", "dw", "db"), got, ref)])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,D,W", [(1, 1, 2), (1, 512, 4), (5, 100, 3), (70, 257, 4), (3, 36, 8)])
def test_conv_step_goes_on_from_a_prompt(g, n, D, W, bf16):
    rng = np.random.default_rng(n + D)
    r = Rows(rng, bf16)
    T = 6
    x, w, bias = r(n * T, D), rng.standard_normal((W, D)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    ref, last = so.conv(r.val(x), w, bias, n)
    from asca_amd.gpu import DevBuf

    st = DevBuf.from_host(np.zeros((n, W - 1, D), np.float32))
    for t in range(T):
        y = g.conv_step(st, np.ascontiguousarray(x.reshape(n, T, D)[:, t]), w, bias)
        check(f"conv step {t}", [("y", r.val(y), ref.reshape(n, T, D)[:, t], r.tol(FWD))])
    np.testing.assert_array_equal(st.to_host((n, W - 1, D)), last.astype(np.float32))


# -------------------------------------------------------------------- scan

SSM = [(1, 1, 1, 1, 1, False), (2, 5, 3, 4, 1, True), (1, 16, 16, 16, 1, False), (7, 33, 70, 16, 1, True),
       (2, 100, 130, 12, 2, True), (1, 257, 64, 8, 4, False), (2, 40, 65, 32, 1, True), (1, 37, 20, 64, 2, False),
       (2, 300, 48, 5, 3, False), (1, 700, 33, 16, 1, False), (2, 64, 256, 16, 1, True), (3, 21, 50, 2, 1, True),
       (1, 19, 17, 33, 1, False), (2, 1100, 64, 16, 1, True), (1, 2050, 20, 4, 1, False),
       # many channels (each width of the lane groups, 8 waves a block), long rows cut into chunks
       (8, 20, 2048, 16, 1, True), (8, 20, 2048, 7, 1, True), (8, 12, 2048, 20, 1, True), (4, 40, 2048, 10, 2, False),
       (1, 1100, 512, 16, 1, True), (1, 1100, 500, 12, 2, False), (1, 1100, 260, 33, 1, False), (2, 700, 300, 24, 3, True),
       # rows split over a block's waves (4, 8 and 16 of them), and narrow long ones in chunks
       (9, 70, 256, 16, 1, True), (1, 150, 1100, 16, 1, False), (3, 530, 36, 12, 1, True), (1, 1700, 24, 16, 1, False), (2, 1600, 10, 5, 1, True),
       (1, 200, 72, 30, 2, False), (3, 90, 800, 20, 1, True), (2, 130, 30, 50, 1, True)]


def ssm_inputs(r, rng, B, T, D, N, G):
    """Steps e of about 0.001 to 0.1 and one in twenty around 1; A near -1 .. -N."""
    e = np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), D))
    dtv = rng.standard_normal((B * T, D)) + np.where(rng.random((B * T, D)) < 0.05, 4.0, 0.0)
    return dict(x=r(B * T, D), dt=r.dev(dtv.astype(np.float32)), Bm=r(B * T, G * N), Cm=r(B * T, G * N),
                A=(-np.arange(1, N + 1)[:, None] * np.exp(0.1 * rng.standard_normal((N, D)))).astype(np.float32),
                dt_bias=np.log(np.expm1(e)).astype(np.float32), Dk=rng.standard_normal(D).astype(np.float32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,T,D,N,G,rag", SSM)
def test_ssm(g, B, T, D, N, G, rag, bf16):
    print(f"[ssm] B={B} T={T} D={D} N={N} G={G} ragged={rag} bf16={bf16}", flush=True)
    rng = np.random.default_rng(B * 1000 + T + D + N)
    r = Rows(rng, bf16)
    i = ssm_inputs(r, rng, B, T, D, N, G)
    v = {k: r.val(a) for k, a in i.items()}
    h0, dh = (rng.standard_normal((B, N, D)).astype(np.float32) for _ in range(2))
    dy, lens = r(B * T, D), ragged(B, T) if rag else None
    y, h, dev = g.ssm_scan(**i, batch=B, h0=h0, lens=lens, groups=G)
    ry, rh = so.ssm(**v, B=B, h0=h0, lens=lens, G=G)
    y2, h2, none = g.ssm_scan(**i, batch=B, h0=h0, lens=lens, groups=G, keep=False)
    assert none is None
    np.testing.assert_array_equal(y2, y)
    np.testing.assert_array_equal(h2, h)
    got = g.ssm_scan_bwd(dev, dy, dh)
    again = g.ssm_scan_bwd(dev, dy, dh)
    ref = so.ssm_bwd(**v, dy=r.val(dy), B=B, h0=h0, lens=lens, G=G, dh_out=dh)
    dev.free()
    rows = ("dx", "ddt", "dB", "dC")
    check("ssm", [("y", r.val(y), ry, r.tol(FWD)), ("h", h, rh, FWD)] +
          [(k, r.val(got[k]), ref[k], r.tol(GRAD) if k in rows else GRAD) for k in ref])
    for k in got:
        np.testing.assert_array_equal(got[k], again[k])


def test_ssm_without_softplus_bias_skip_and_states(g):
    rng = np.random.default_rng(5)
    B, T, D, N = 2, 37, 40, 16
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    i = dict(x=f(B * T, D), dt=rng.uniform(0.01, 0.3, (B * T, D)).astype(np.float32), A=-rng.uniform(0.5, 8, (N, D)).astype(np.float32),
             Bm=f(B * T, N), Cm=f(B * T, N))
    dy = f(B * T, D)
    y, h, dev = g.ssm_scan(**i, batch=B, softplus=False)
    ry, rh = so.ssm(**i, B=B, softplus=False)
    got, ref = g.ssm_scan_bwd(dev, dy), so.ssm_bwd(**i, dy=dy, B=B, softplus=False)
    check("ssm plain", [("y", y, ry, FWD), ("h", h, rh, FWD)] + [(k, got[k], ref[k], GRAD) for k in ref])


@pytest.mark.parametrize("T,D,N,e", [(400, 64, 16, 1.5), (400, 64, 16, 9.0), (1700, 64, 16, 1.5), (1700, 40, 5, 1.5), (300, 64, 40, 9.0), (200, 64, 40, 9.0), (300, 64, 20, 9.0)])
def test_ssm_growth_past_the_range_of_f32_over_rows_without_a_state(g, T, D, N, e):
    """States that grow by e a row in the exponent: many rows' growth (a tile's at 9) is far
    past f32's range, but nothing is there to grow before the last rows, and there is no
    gradient after the first."""
    rng = np.random.default_rng(14)
    last = int(60 / e)   # rows from the last x (to the first dy) on
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    i = dict(x=f(T, D), dt=np.full((T, D), e, np.float32), A=np.ones((N, D), np.float32), Bm=f(T, N), Cm=f(T, N))
    dy = f(T, D)
    i["x"][:-last] = 0
    dy[last:] = 0
    y, h, dev = g.ssm_scan(**i, batch=1, softplus=False)
    ry, rh = so.ssm(**i, B=1, softplus=False)
    got, ref = g.ssm_scan_bwd(dev, dy), so.ssm_bwd(**i, dy=dy, B=1, softplus=False)
    dev.free()
    check("growth", [("y", y, ry, FWD), ("h", h, rh, FWD)] + [(k, got[k], ref[k], GRAD) for k in ref])


# every instance of the split forward, rows one after another, and rows cut into chunks
GROWTH = [(1, 34, 16, 4), (1, 34, 16, 16), (1, 520, 16, 16), (1, 34, 1100, 16), (1, 130, 1100, 16), (1, 34, 16, 20), (1, 130, 16, 20),
          (1, 34, 16, 40), (8, 34, 2048, 16), (1, 1700, 24, 16), (1, 1700, 24, 20)]


@pytest.mark.parametrize("small,e", [(1e-10, 6.0), (1e-35, 10.0)])
@pytest.mark.parametrize("B,T,D,N", GROWTH)
def test_ssm_growth_of_small_states_past_the_range_of_f32(g, B, T, D, N, small, e):
    """The first K rows' growth, exp(K e), is past f32's range and the states that it meets
    are small: they stay finite until the last K rows take it back.  The gradients pass
    through the same factors from the other end.  A growth of G in the exponent takes the
    roundings of A and of each e A with it, 2 G 2^-24; twice that is allowed."""
    K = 16 if N <= 16 else 8
    e = e * 16 / K
    rng = np.random.default_rng(15)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    step = np.zeros((B, T, D), np.float32)
    step[:, :K], step[:, -K:] = e, -e
    i = dict(x=f(B * T, D) * np.float32(small), dt=step.reshape(B * T, D), A=np.ones((N, D), np.float32), Bm=f(B * T, N), Cm=f(B * T, N))
    h0, dh, dy = f(B, N, D) * np.float32(small), f(B, N, D) * np.float32(1e10), f(B * T, D) * np.float32(small)
    h0[:, ::3] = 0
    y, h, dev = g.ssm_scan(**i, batch=B, h0=h0, softplus=False)
    ry, rh = so.ssm(**i, B=B, h0=h0, softplus=False)
    got, ref = g.ssm_scan_bwd(dev, dy, dh), so.ssm_bwd(**i, dy=dy, B=B, h0=h0, softplus=False, dh_out=dh)
    dev.free()
    more = 4 * K * e * 2.0 ** -24
    if small * small < 1e-45:   # dy x has no f32
        assert not got.pop("dDk").any() and np.abs(ref.pop("dDk")).max() < 1e-45
    check("small growth", [("y", y, ry, FWD + more), ("h", h, rh, FWD + more)] + [(k, got[k], ref[k], GRAD + more) for k in ref])


def test_ssm_cut_in_two_is_the_sequence(g):
    rng = np.random.default_rng(6)
    r = Rows(rng, False)
    T, D, N, k = 50, 20, 16, 19
    i = ssm_inputs(r, rng, 1, T, D, N, 1)
    cut = lambda s: {n: a[s] if n in ("x", "dt", "Bm", "Cm") else a for n, a in i.items()}  # noqa: E731
    y, h, _ = g.ssm_scan(**i, batch=1, keep=False)
    y1, h1, _ = g.ssm_scan(**cut(slice(0, k)), batch=1, keep=False)
    y2, h2, _ = g.ssm_scan(**cut(slice(k, T)), batch=1, h0=h1, keep=False)
    check("cut", [("y", np.concatenate([y1, y2]), y, FWD), ("h", h2, h, FWD)])


@pytest.mark.parametrize("v", [-90.0, -20.0, -5.0, 0.0, 5.0, 25.0, 90.0])
def test_ssm_softplus_over_its_range(g, v):
    # one row, one state, B = C = 1: y = e x, whatever the size of e
    one = np.ones((1, 1), np.float32)
    y, _, _ = g.ssm_scan(one, one * np.float32(v), -one, one, one, batch=1, keep=False)
    e = np.logaddexp(np.float64(v), 0)
    assert abs(y[0, 0] - e) <= 2e-6 * e + 1e-38


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,D,N,G", [(1, 1, 1, 1), (1, 512, 16, 1), (5, 100, 12, 2), (70, 256, 16, 1), (3, 36, 64, 3), (9, 130, 33, 1)])
def test_ssm_step_goes_on_from_a_prompt(g, n, D, N, G, bf16):
    from asca_amd.gpu import DevBuf

    rng = np.random.default_rng(n + D + N)
    r = Rows(rng, bf16)
    T = 5
    i = ssm_inputs(r, rng, n, T, D, N, G)
    ry, rh = so.ssm(**{k: r.val(a) for k, a in i.items()}, B=n, G=G)
    cut = lambda a, t: np.ascontiguousarray(a.reshape(n, T, -1)[:, t])  # noqa: E731
    h = DevBuf.from_host(np.zeros((n, N, D), np.float32))
    for t in range(T):
        y = g.ssm_step(h, **{k: cut(i[k], t) for k in ("x", "dt", "Bm", "Cm")}, A=i["A"], dt_bias=i["dt_bias"], Dk=i["Dk"], groups=G)
        check(f"ssm step {t}", [("y", r.val(y), ry.reshape(n, T, D)[:, t], r.tol(FWD))])
    check("ssm step", [("h", h.to_host((n, N, D)), rh, FWD)])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,D,N,G", [(300, 2048, 12, 2), (260, 2050, 16, 1), (600, 1000, 33, 1), (530, 990, 8, 3), (524288, 1, 20, 1)])
def test_ssm_step_of_many_sequences(g, n, D, N, G, bf16):
    """From 2^19 channels on (of all sequences) a channel's states are loaded 8 at a time."""
    from asca_amd.gpu import DevBuf

    print(f"[ssm step] n={n} D={D} N={N} G={G} bf16={bf16}", flush=True)
    rng = np.random.default_rng(n + D + N)
    r = Rows(rng, bf16)
    i = ssm_inputs(r, rng, n, 1, D, N, G)
    h0 = rng.standard_normal((n, N, D), dtype=np.float32)
    v = {k: r.val(a).astype(np.float64) for k, a in i.items()}
    e = np.logaddexp(v["dt"] + v["dt_bias"], 0)
    wide = lambda m: np.repeat(m.reshape(n, G, N).transpose(0, 2, 1), D // G, axis=2)  # noqa: E731
    rh = np.exp(e[:, None] * v["A"]) * h0 + (e * v["x"])[:, None] * wide(v["Bm"])
    ry = (rh * wide(v["Cm"])).sum(1) + v["Dk"] * v["x"]
    h = DevBuf.from_host(h0)
    y = g.ssm_step(h, i["x"], i["dt"], i["A"], i["Bm"], i["Cm"], dt_bias=i["dt_bias"], Dk=i["Dk"], groups=G)
    check("ssm step", [("y", r.val(y), ry, r.tol(FWD)), ("h", h.to_host((n, N, D)), rh, FWD)])


@pytest.mark.parametrize("v", [-85.0, -60.0, -40.0])
def test_ssm_softplus_of_small_steps(g, v):
    """As above down to the smallest normal e, by itself: exp2 of v log2(e), whose argument
    is rounded twice (of at most 123, to 2^-17 together, or 2^-17 ln 2 of e)."""
    one = np.ones((1, 1), np.float32)
    y, _, _ = g.ssm_scan(one, one * np.float32(v), -one, one, one, batch=1, keep=False)
    e = np.logaddexp(np.float64(v), 0)
    assert abs(y[0, 0] - e) <= 2.0 ** -17 * e


# -------------------------------------------------------------- block norm


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (9, 256), (130, 260), (33, 512), (7, 1000), (5, 1024), (6, 1025), (3, 2048),
                                       (2, 4099), (2, 8192), (1, 16383), (3, 20001), (1030, 36)])
def test_block_norm(g, rows, cols, bf16):
    print(f"[norm] rows={rows} cols={cols} bf16={bf16}", flush=True)
    rng = np.random.default_rng(rows + cols)
    r = Rows(rng, bf16)
    x, y, z, dr, dn = (r(rows, cols) for _ in range(5))
    p = {k: (rng.standard_normal(cols) * 0.3 + 1).astype(np.float32) for k in ("w_post", "scale", "w_pre")}
    v = r.val
    got = g.block_norm(x, y, z, **p)
    ref = so.block_norm(v(x), v(y), v(z), **p)
    gb, rb = g.block_norm_bwd(x, y, z, dr, dn, **p), so.block_norm_bwd(v(x), v(y), v(z), v(dr), v(dn), **p)
    check("norm", [("r", v(got[0]), ref[0], r.tol(FWD)), ("n", v(got[1]), ref[1], r.tol(FWD))] +
          [(k, v(gb[k]), rb[k], r.tol(GRAD) if k in ("dx", "dy", "dz") else GRAD) for k in gb])


@pytest.mark.parametrize("have", ["x y z", "x y", "y z", "y", "x"])
@pytest.mark.parametrize("gains", [True, False])
@pytest.mark.parametrize("grads", ["dr dn", "dr", "dn"])
def test_block_norm_parts(g, have, gains, grads):
    rng = np.random.default_rng(len(have))
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    a = {k: f(10, 48) if k in have.split() else None for k in "xyz"}
    d = {k: f(10, 48) if k in grads.split() else None for k in ("dr", "dn")}
    p = {k: f(48) for k in (("w_post", "scale", "w_pre") if "y" in have else ("w_pre",))} if gains else {}
    got, ref = g.block_norm(*a.values(), **p), so.block_norm(*a.values(), **p)
    gb, rb = g.block_norm_bwd(*a.values(), *d.values(), **p), so.block_norm_bwd(*a.values(), *d.values(), **p)
    check(f"norm {have}", [("r", got[0], ref[0], FWD), ("n", got[1], ref[1], FWD)] + [(k, gb[k], rb[k], GRAD) for k in gb])


def test_block_norm_of_zero_rows_is_zero(g):
    z = np.zeros((3, 40), np.float32)
    r, n = g.block_norm(z, z, z)
    assert not r.any() and not n.any()
    o = g.block_norm_bwd(z, z, z, z + 1, None)
    assert np.isfinite(o["dy"]).all() and (o["dx"] == 1).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(2300, 132), (2101, 301), (2050, 500), (1100, 700), (1030, 1024), (600, 2048), (530, 1500), (520, 2052), (515, 2053),
                                       (3, 2049), (3, 3000), (2, 4096), (2, 4095)])
def test_block_norm_of_many_rows_and_of_wide_ones(g, rows, cols, bf16):
    """Backwards whose blocks go over several rows (the next row's loads, the parameters'
    sums over rows, wide rows' sums in memory), forwards of 2049 to 4096 columns."""
    print(f"[norm] rows={rows} cols={cols} bf16={bf16}", flush=True)
    rng = np.random.default_rng(rows + cols)
    r = Rows(rng, bf16)
    x, y, z, dr, dn = (r(rows, cols) for _ in range(5))
    p = {k: (rng.standard_normal(cols) * 0.3 + 1).astype(np.float32) for k in ("w_post", "scale", "w_pre")}
    v = r.val
    got, ref = g.block_norm(x, y, z, **p), so.block_norm(v(x), v(y), v(z), **p)
    gb, rb = g.block_norm_bwd(x, y, z, dr, dn, **p), so.block_norm_bwd(v(x), v(y), v(z), v(dr), v(dn), **p)
    check("norm", [("r", v(got[0]), ref[0], r.tol(FWD)), ("n", v(got[1]), ref[1], r.tol(FWD))] +
          [(k, v(gb[k]), rb[k], r.tol(GRAD) if k in ("dx", "dy", "dz") else GRAD) for k in gb])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(2300, 132), (1100, 700), (600, 1501), (520, 2052), (3, 4100), (2, 4099)])
def test_block_norm_in_place(g, rows, cols, bf16):
    """r over x, and dx over dr, give the bits of the calls beside them."""
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(rows + cols)
    r = Rows(rng, bf16)
    ty = int(bf16)
    x, y, z, dr, dn = (r(rows, cols) for _ in range(5))
    b = {k: gpu.DevBuf.from_array(a) for k, a in dict(x=x, y=y, z=z, dr=dr, dn=dn).items()}
    o = {k: gpu.DevBuf(x.nbytes) for k in ("r", "n", "n2", "dx", "dy", "dy2", "dz", "dz2")}
    w = {k: gpu.DevBuf.from_host((rng.standard_normal(cols) * 0.3 + 1).astype(np.float32)) for k in ("w1", "s", "w2")}
    dw = {k: gpu.DevBuf(cols * 4) for k in ("w1", "s", "w2", "w1_", "s_", "w2_")}
    ins = lambda: (_p(b["x"]), cols, _p(b["y"]), cols, _p(b["z"]), cols, _p(w["w1"]), _p(w["s"]), _p(w["w2"]))  # noqa: E731
    bwd = lambda dx, dy, dz, e: _lib.call("asca_block_norm_bwd", *ins(), _p(b["dr"]), cols, _p(b["dn"]), cols, _p(dx), cols, _p(o[dy]), cols,  # noqa: E731
                                          _p(o[dz]), cols, _p(dw["w1" + e]), _p(dw["s" + e]), _p(dw["w2" + e]), rows, cols, 1e-6, ty, None)
    fwd = lambda res, n: _lib.call("asca_block_norm_fwd", *ins(), _p(res), cols, _p(o[n]), cols, rows, cols, 1e-6, ty, None)  # noqa: E731
    bwd(o["dx"], "dy", "dz", "")
    bwd(b["dr"], "dy2", "dz2", "_")
    fwd(o["r"], "n")
    fwd(b["x"], "n2")
    _lib.call("asca_sync")
    get = lambda q, like: q.to_host(like.shape, like.dtype)  # noqa: E731
    for a, c in ((o["dx"], b["dr"]), (o["dy"], o["dy2"]), (o["dz"], o["dz2"]), (o["r"], b["x"]), (o["n"], o["n2"])):
        np.testing.assert_array_equal(get(a, x), get(c, x))
    for k in ("w1", "s", "w2"):
        np.testing.assert_array_equal(dw[k].to_host((cols,)), dw[k + "_"].to_host((cols,)))


@pytest.mark.parametrize("rows,cols", [(7, 1), (9, 48), (3, 700), (5, 2048), (2, 2050), (3, 4099)])
def test_block_norm_without_eps(g, rows, cols):
    """eps = 0 is defined wherever a row is not all zeros, also where there is no y."""
    rng = np.random.default_rng(cols)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, y, dr, dn, w = f(rows, cols) + 3, f(rows, cols) + 3, f(rows, cols), f(rows, cols), f(cols)
    for y_, p in ((None, dict(w_pre=w)), (y, dict(w_pre=w, scale=f(cols)))):
        got, ref = g.block_norm(x, y_, **p, eps=0.0), so.block_norm(x, y_, **p, eps=0.0)
        gb, rb = g.block_norm_bwd(x, y_, None, dr, dn, **p, eps=0.0), so.block_norm_bwd(x, y_, None, dr, dn, **p, eps=0.0)
        # a row of one column has no gradient: what is left is rounding of its terms, next to dr
        size = lambda k: np.abs(dr).max() if cols == 1 and k in ("dx", "dy") else 0.0  # noqa: E731
        check("norm eps=0", [("r", got[0], ref[0], FWD), ("n", got[1], ref[1], FWD)] +
              [(k, np.append(gb[k], size(k)), np.append(rb[k], size(k)), GRAD) for k in gb if cols > 1 or k in ("dx", "dw_pre")])


def test_block_norm_refuses_an_eps_below_zero(g):
    from asca_amd import _lib, gpu

    f = C.c_void_p(1 << 12)   # never dereferenced
    gpu.reset_stats()
    for eps in (-1e-6, float("-inf"), float("nan")):
        for call in (("asca_block_norm_fwd", f, 8, f, 8, None, 0, None, None, None, f, 8, None, 0, 4, 8, eps, 0, None),
                     ("asca_block_norm_bwd", f, 8, f, 8, None, 0, None, None, None, f, 8, None, 0, f, 8, None, 0, None, 0, None, None, None, 4, 8,
                      eps, 0, None)):
            with pytest.raises(_lib.AscaError) as ei:
                _lib.call(*call)
            assert ei.value.code == 1, str(ei.value)
    assert gpu.stats()[2] == 0


# ---------------------------------------------------------------- clipping


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [4096, 4097, 1, 12289], [7] * 300, [100003], []])
@pytest.mark.parametrize("place", ["in", "out"])
def test_grads_clip(g, sizes, bf16, place):
    from asca_amd import gpu

    rng = np.random.default_rng(sum(sizes) + len(sizes))
    r = Rows(rng, bf16)
    host = [r(k, scale=0.1 * (1 + i % 5)) for i, k in enumerate(sizes)]
    vals = [r.val(h) for h in host]
    for max_norm in (0.5, 1e6):
        src = [gpu.DevBuf.from_array(h) for h in host]
        dst = [gpu.DevBuf(h.nbytes) for h in host] if place == "out" else None
        gl = gpu.GradList(list(zip(src, sizes)), dst, dtype=gpu.BF16 if bf16 else gpu.F32)
        want, c, clipped = so.clip(vals, max_norm)
        assert abs(gl.norm() - want) <= 1e-6 * want
        norm, coef = gl.clip(max_norm)
        assert abs(norm - want) <= 1e-6 * want and abs(coef - c) <= 1e-6 * c
        for h, s, d, e in zip(host, src, dst or src, clipped):
            if h.size:
                got = d.to_host(h.shape, h.dtype)
                assert err(r.val(got), e) <= r.tol(FWD)
                if place == "out":
                    np.testing.assert_array_equal(s.to_host(h.shape, h.dtype), h)
        gl.close()


@pytest.mark.parametrize("bf16", [False, True])
def test_grads_clip_of_a_list_larger_than_the_cache(g, bf16):
    from asca_amd import gpu

    sizes = [67_108_864 << bf16, 5_000_003, 1]
    rng = np.random.default_rng(3)
    r = Rows(rng, bf16)
    block = r(1 << 20)
    host = [np.resize(block, k) for k in sizes]
    src = [gpu.DevBuf.from_array(h) for h in host]
    gl = gpu.GradList(list(zip(src, sizes)), dtype=gpu.BF16 if bf16 else gpu.F32)
    want = np.sqrt(sum(float(np.square(r.val(h[i:i + (1 << 22)]).astype(np.float64)).sum()) for h in host for i in range(0, h.size, 1 << 22)))
    norm, coef = gl.clip(100.0)
    assert abs(norm - want) <= 1e-6 * want and abs(coef - 100.0 / (want + 1e-6)) <= 1e-6 * coef
    for h, b in zip(host, src):
        got = b.to_host(h.shape, h.dtype)
        for i in range(0, h.size, 1 << 22):
            assert err(r.val(got[i:i + (1 << 22)]), r.val(h[i:i + (1 << 22)]).astype(np.float64) * 100.0 / (want + 1e-6)) <= r.tol(FWD)
    gl.close()
    for b in src:
        b.free()


def test_grads_norm_of_large_small_and_infinite_values(g):
    from asca_amd import gpu

    for val, n in ((1e30, 1000), (1e-30, 1000), (np.inf, 3), (np.nan, 3)):
        a = np.full(n, val, np.float32)
        gl = gpu.GradList([(gpu.DevBuf.from_host(a), n)])
        want = float(np.float32(np.sqrt((a.astype(np.float64) ** 2).sum())))
        norm, coef = gl.clip(1.0)
        assert norm == pytest.approx(want, rel=1e-6, nan_ok=True)
        assert (np.isnan(coef) if np.isnan(val) else coef == 0.0 if np.isinf(val) else coef == pytest.approx(min(1.0, 1 / want), rel=1e-6))
        gl.close()


def test_grads_clip_repeats_bit_for_bit(g):
    from asca_amd import gpu

    a = np.random.default_rng(2).standard_normal(1 << 20).astype(np.float32)
    d, o = gpu.DevBuf.from_host(a), gpu.DevBuf(a.nbytes)
    gl = gpu.GradList([(d, a.size)], [o])
    first = gl.clip(1.0)
    want = o.to_host(a.shape)
    for _ in range(5):
        assert gl.clip(1.0) == first
        np.testing.assert_array_equal(o.to_host(a.shape), want)
    gl.close()


# ------------------------------------- strides, streams, offsets, refusals


def _p(buf, off=0):
    return C.c_void_p(buf.ptr + off)


@pytest.mark.parametrize("bf16", [False, True])
def test_columns_of_wider_matrices_and_rows_past_a_length(g, bf16):
    """Every operand a range of columns of a wider matrix that is NaN elsewhere and past
    each length, at odd offsets; outputs land in theirs and leave the rest alone."""
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(8)
    r = Rows(rng, bf16)
    B, T, D, N, G, ld, at = 3, 37, 66, 12, 2, 131, 13
    size, ty = (2, 1) if bf16 else (4, 0)
    lens = np.array([37, 5, 0], np.int32)
    i = ssm_inputs(r, rng, B, T, D, N, G)
    dy = r(B * T, D)
    past = (np.arange(T)[None] >= lens[:, None]).reshape(-1)

    def wide(a):
        w = r.dev(np.full((B * T, ld), np.nan, np.float32))
        w[:, at:at + a.shape[1]] = a
        w[past] = r.dev(np.full(1, np.nan, np.float32))
        return gpu.DevBuf.from_array(w)

    ins = {k: wide(i[k]) for k in ("x", "dt", "Bm", "Cm")}
    bdy, blen = wide(dy), gpu.DevBuf.from_array(lens)
    par = {k: gpu.DevBuf.from_host(i[k]) for k in ("A", "dt_bias", "Dk")}
    mark = r.dev(np.full((B * T, ld), 7.0, np.float32))
    out = {k: gpu.DevBuf.from_array(mark) for k in ("y", "dx", "ddt", "dB", "dC")}
    f = {k: gpu.DevBuf(n * 4) for k, n in (("h", B * N * D), ("dbias", D), ("dA", N * D), ("dD", D), ("dh0", B * N * D))}
    n = C.c_size_t()
    _lib.call("asca_ssm_ws_bytes", B, T, D, N, C.byref(n))
    ws = gpu.DevBuf(n.value)
    a = at * size
    st = C.c_void_p()
    _lib.call("asca_stream_create", C.byref(st))
    head = (_p(ins["x"], a), ld, _p(ins["dt"], a), ld, _p(par["dt_bias"]), _p(par["A"]), _p(ins["Bm"], a), ld, _p(ins["Cm"], a), ld,
            _p(par["Dk"]))
    _lib.call("asca_ssm_fwd", *head, None, _p(blen), _p(out["y"], a), ld, _p(f["h"]), _p(ws), B, T, D, N, G, 1, ty, st)
    _lib.call("asca_ssm_bwd", *head, _p(blen), _p(bdy, a), ld, None, _p(ws), _p(out["dx"], a), ld, _p(out["ddt"], a), ld,
              _p(f["dbias"]), _p(f["dA"]), _p(out["dB"], a), ld, _p(out["dC"], a), ld, _p(f["dD"]), _p(f["dh0"]), B, T, D, N, G, 1,
              ty, st)
    w, cb = rng.standard_normal((4, D)).astype(np.float32), gpu.DevBuf.from_array(mark)
    bw = gpu.DevBuf.from_host(w)
    _lib.call("asca_conv_fwd", _p(ins["x"], a), ld, _p(bw), None, None, _p(blen), _p(cb, a), ld, None, B, T, D, 4, 1, ty, st)
    _lib.call("asca_stream_sync", st)
    _lib.call("asca_stream_destroy", st)
    v = {k: r.val(m) for k, m in i.items()}
    ry, rh = so.ssm(**v, B=B, lens=lens, G=G)
    ref = so.ssm_bwd(**v, dy=r.val(dy), B=B, lens=lens, G=G)
    ref.update(y=ry, conv=so.conv(v["x"], w, None, B, None, lens)[0])
    pairs = []
    for k, b in {**out, "conv": cb}.items():
        m = b.to_host((B * T, ld), mark.dtype)
        c = ref[k].shape[1]
        pairs.append((k, r.val(np.ascontiguousarray(m[:, at:at + c])), ref[k], r.tol(FWD if k in ("y", "conv") else GRAD)))
        assert (m[:, :at] == mark[0, 0]).all() and (m[:, at + c:] == mark[0, 0]).all(), k
        assert not r.val(np.ascontiguousarray(m[past, at:at + c])).any(), k
    pairs += [("h", f["h"].to_host((B, N, D)), rh, FWD), ("dA", f["dA"].to_host((N, D)), ref["dA"], GRAD),
              ("dD", f["dD"].to_host((D,)), ref["dDk"], GRAD), ("dbias", f["dbias"].to_host((D,)), ref["ddt_bias"], GRAD),
              ("dh0", f["dh0"].to_host((B, N, D)), ref["dh0"], GRAD)]
    check("wide", pairs)


def test_offsets_past_32_bits(g):
    """Rows 2^30 elements apart: the last of five begins at element 2^32."""
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(9)
    r = Rows(rng, True)
    T, D, N, ld = 5, 64, 16, 1 << 30
    i = ssm_inputs(r, rng, 1, T, D, N, 1)
    v = {k: r.val(m) for k, m in i.items()}
    big = gpu.DevBuf((4 * ld + 4 * 64) * 2)    # x, dt, y and conv's y side by side
    small = {k: gpu.DevBuf.from_array(i[k]) for k in ("Bm", "Cm", "A", "dt_bias", "Dk")}
    put = lambda k, c, t: _lib.call("asca_h2d", _p(big, (t * ld + c) * 2), np.ascontiguousarray(i[k][t]).ctypes.data_as(C.c_void_p), D * 2)  # noqa: E731
    for t in range(T):
        put("x", 0, t)
        put("dt", 64, t)
    w = rng.standard_normal((4, D)).astype(np.float32)
    bw = gpu.DevBuf.from_host(w)
    _lib.call("asca_ssm_fwd", _p(big), ld, _p(big, 128), ld, _p(small["dt_bias"]), _p(small["A"]), _p(small["Bm"]), N, _p(small["Cm"]),
              N, _p(small["Dk"]), None, None, _p(big, 256), ld, None, None, 1, T, D, N, 1, 1, 1, None)
    _lib.call("asca_conv_fwd", _p(big), ld, _p(bw), None, None, None, _p(big, 384), ld, None, 1, T, D, 4, 1, 1, None)
    _lib.call("asca_sync")

    def get(c):
        rows = np.empty((T, D), np.uint16)
        for t in range(T):
            _lib.call("asca_d2h", rows[t].ctypes.data_as(C.c_void_p), _p(big, (t * ld + c) * 2), D * 2)
        return r.val(rows)

    y, c = get(128), get(192)
    _lib.call("asca_block_norm_fwd", _p(big), ld, _p(big, 128), ld, None, 0, None, None, None, _p(big, 256), ld, None, 0, T, D, 1e-6, 1, None)
    _lib.call("asca_sync")
    n = get(128)
    big.free()
    _lib.call("asca_pool_release")
    check("far", [("y", y, so.ssm(**v, B=1)[0], BF), ("conv", c, so.conv(v["x"], w, None, 1)[0], BF),
                  ("norm", n, so.block_norm(v["x"], v["dt"])[0], BF)])


def test_calls_on_two_streams_at_once(g):
    """Scans, their backwards and the sums that use a stream's scratch, alternating over
    two streams without a wait between, against the same calls alone."""
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(10)
    r = Rows(rng, False)
    B, T, D, N = 2, 200, 96, 16
    st = [C.c_void_p() for _ in range(2)]
    for s in st:
        _lib.call("asca_stream_create", C.byref(s))
    cases = []
    for _ in range(2):
        i, dy = ssm_inputs(r, rng, B, T, D, N, 1), r(B * T, D)
        y, h, dev = g.ssm_scan(**i, batch=B)
        want = g.ssm_scan_bwd(dev, dy)
        o = {k: gpu.DevBuf(a.nbytes) for k, a in want.items()}
        cases.append((dev, gpu.DevBuf.from_host(dy), want, o))
    for _ in range(4):
        for (dev, bdy, _, o), s in zip(cases, st):
            q = dev.ins
            _lib.call("asca_ssm_bwd", _p(q["x"]), D, _p(q["dt"]), D, _p(q["bias"]), _p(q["A"]), _p(q["Bm"]), N, _p(q["Cm"]), N,
                      _p(q["Dk"]), None, _p(bdy), D, None, _p(q["ws"]), _p(o["dx"]), D, _p(o["ddt"]), D, _p(o["ddt_bias"]),
                      _p(o["dA"]), _p(o["dB"]), N, _p(o["dC"]), N, _p(o["dDk"]), _p(o["dh0"]), B, T, D, N, 1, 1, 0, s)
    for s in st:
        _lib.call("asca_stream_sync", s)
        _lib.call("asca_stream_destroy", s)
    for dev, _, want, o in cases:
        for k in want:
            np.testing.assert_array_equal(o[k].to_host(want[k].shape), want[k])


def test_empty_calls(g):
    z = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    w = z(4, 3) + 1
    y, s = g.conv(z(0, 3), w, batch=2, state=z(2, 3, 3) + 5)    # no rows: the state goes through
    assert y.shape == (0, 3) and (s == 5).all()
    dx, dw, db, ds = g.conv_bwd(z(0, 3), w, z(3), z(0, 3), batch=2, dstate_out=z(2, 3, 3) + 2)
    assert not dw.any() and not db.any() and (ds == 2).all()
    y, h, dev = g.ssm_scan(z(0, 3), z(0, 3), z(4, 3) - 1, z(0, 4), z(0, 4), batch=2, h0=z(2, 4, 3) + 5)
    assert (h == 5).all()
    o = g.ssm_scan_bwd(dev, z(0, 3), z(2, 4, 3) + 2)
    assert (o["dh0"] == 2).all() and not o["dA"].any() and not o["ddt_bias"].any()


def test_refusals(g):
    """Bad arguments come back as errors that name the call, and nothing is launched."""
    from asca_amd import _lib, gpu

    f = C.c_void_p(1 << 12)   # never dereferenced: every call is refused before a launch
    out = C.c_size_t()
    conv = lambda D=8, ld=8, W=4, ty=0, x=f, w=f, B=1, so_=None: ("asca_conv_fwd", x, ld, w, None, None, None, f, ld, so_, B, 4, D, W, 1, ty, None)  # noqa: E731
    ssm = lambda D=8, ld=8, N=4, G=1, ty=0, x=f, A=f, h0=None, ho=None: (  # noqa: E731
        "asca_ssm_fwd", x, ld, f, 8, None, A, f, 64, f, 64, None, h0, None, f, 8, ho, None, 1, 4, D, N, G, 1, ty, None)
    norm = lambda cols=8, ld=8, ty=0, x=f, y=f, z=f, r=f, w=None: (  # noqa: E731
        "asca_block_norm_fwd", x, ld, y, 1 << 15, z, 1 << 15, w, None, None, r, 1 << 15, None, 0, 4, cols, 1e-6, ty, None)
    h = C.c_void_p()
    one = (C.c_void_p * 1)(None)
    bad = [(conv(W=1), 3), (conv(W=9), 3), (conv(ty=2), 3), (conv(ld=7), 1), (conv(x=None), 1), (conv(w=None), 1), (conv(B=-1), 1),
           (("asca_conv_fwd", f, 8, f, None, f, None, f, 8, f, 1, 4, 8, 4, 1, 0, None), 1),
           (ssm(N=0), 3), (ssm(N=65), 3), (ssm(G=3), 1), (ssm(G=0), 1), (ssm(ty=-1), 3), (ssm(ld=7), 1), (ssm(x=None), 1), (ssm(A=None), 1),
           (ssm(h0=f, ho=f), 1), (("asca_ssm_ws_bytes", 1, -1, 8, 4, C.byref(out)), 1), (("asca_ssm_ws_bytes", 1, 1, 8, 4, None), 1),
           (("asca_ssm_ws_bytes", 1, (1 << 30) + 1, 8, 4, C.byref(out)), 3),
           (("asca_conv_fwd", f, 8, f, None, None, None, f, 8, None, 1, (1 << 30) + 1, 8, 4, 1, 0, None), 3),
           (norm(ld=7), 1), (norm(y=None), 1), (norm(r=None), 1), (norm(ty=7), 3),
           (norm(x=None, y=None, z=None), 1),
           (("asca_grads_create", one, None, (C.c_uint64 * 1)(4), 1, 0, C.byref(h)), 1),
           (("asca_grads_create", None, None, None, -1, 0, C.byref(h)), 1), (("asca_grads_create", None, None, None, 0, 5, C.byref(h)), 3),
           (("asca_grads_norm", None, f, None), 1), (("asca_grads_clip", None, 1.0, f, None), 1)]
    gpu.reset_stats()
    for (name, *args), code in bad:
        with pytest.raises(_lib.AscaError) as ei:
            _lib.call(name, *args)
        assert ei.value.code == code, (name, args, str(ei.value))
    gl = gpu.GradList([])
    for m in (-1.0, float("nan")):
        with pytest.raises(_lib.AscaError):
            gl.clip(m)
    assert gpu.stats()[2] == 0
    x = np.zeros((4, 8), np.float32)
    with pytest.raises(ValueError):
        g.ssm_scan(x, x[:3], np.zeros((4, 8)), x[:, :4], x[:, :4], batch=1)
    with pytest.raises(ValueError):
        g.conv(x.astype(np.float64), np.zeros((4, 8)), batch=1)
    with pytest.raises(ValueError):
        g.block_norm(None)


def test_calls_of_more_threads_than_a_launch_takes_are_refused(g):
    """HIP takes fewer than 2^32 threads in a launch; nothing is launched of a larger call."""
    from asca_amd import _lib, gpu

    f, k = C.c_void_p(1 << 12), 1 << 24   # the pointer is never dereferenced
    bad = [("asca_conv_fwd", f, 4096, f, None, None, None, f, 4096, None, 1, 1 << 30, 4096, 4, 1, 0, None),
           ("asca_conv_bwd", f, 4096, f, None, None, None, f, 4096, None, f, 4096, f, None, None, 1, 1 << 30, 4096, 4, 1, 0, None),
           ("asca_conv_step", f, f, 256, f, None, f, 256, k, 256, 4, 1, 0, None),
           ("asca_ssm_fwd", f, 128, f, 128, None, f, f, 8, f, 8, None, None, None, f, 128, None, None, k, 1, 128, 8, 1, 1, 0, None),
           ("asca_ssm_bwd", f, 128, f, 128, None, f, f, 8, f, 8, None, None, f, 128, None, f, f, 128, f, 128, None, f, f, 8, f, 8, None, None,
            k, 1, 128, 8, 1, 1, 0, None),
           ("asca_ssm_step", f, f, 256, f, 256, None, f, f, 8, f, 8, None, f, 256, k, 256, 8, 1, 1, 0, None)]
    bad += [("asca_block_norm_fwd", f, c, None, 0, None, 0, None, None, None, None, 0, f, c, rows, c, 1e-6, 0, None)
            for c, rows in ((8, 4 * k), (520, 2 * k), (1030, k), (5000, k // 2))]
    gpu.reset_stats()
    for name, *args in bad:
        with pytest.raises(_lib.AscaError) as ei:
            _lib.call(name, *args)
        assert ei.value.code == 3, (name, str(ei.value))
    assert gpu.stats()[2] == 0


@pytest.mark.parametrize("nth", [0, 1, 2])
def test_an_injected_failure_is_an_error_and_the_next_call_works(g, nth):
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(11)
    r = Rows(rng, False)
    i, dy = ssm_inputs(r, rng, 1, 20, 8, 4, 1), r(20, 8)
    _, _, dev = g.ssm_scan(**i, batch=1)
    want = g.ssm_scan_bwd(dev, dy)
    gpu.fail_after(nth)
    try:
        with pytest.raises(_lib.AscaError) as ei:
            g.ssm_scan_bwd(dev, dy)
        assert ei.value.code == 5
    finally:
        gpu.fail_after(-1)
    got = g.ssm_scan_bwd(dev, dy)
    for k in want:
        np.testing.assert_array_equal(got[k], want[k])


def _ssm_call(g, i, B, T, D, N, dy, G=1, lens=None):
    """Device buffers of a scan and its backward, and the two calls on a stream."""
    from asca_amd import _lib, gpu

    b = {k: gpu.DevBuf.from_array(a) for k, a in dict(i, dy=dy).items()}
    o = {k: gpu.DevBuf(n * 4) for k, n in (("y", B * T * D), ("h", B * N * D), ("dx", B * T * D), ("ddt", B * T * D), ("db", D), ("dA", N * D),
                                           ("dB", B * T * G * N), ("dC", B * T * G * N), ("dD", D), ("dh0", B * N * D))}
    n = C.c_size_t()
    _lib.call("asca_ssm_ws_bytes", B, T, D, N, C.byref(n))
    ws = gpu.DevBuf(n.value)
    head = (_p(b["x"]), D, _p(b["dt"]), D, _p(b["dt_bias"]), _p(b["A"]), _p(b["Bm"]), G * N, _p(b["Cm"]), G * N, _p(b["Dk"]))

    def run(st):
        _lib.call("asca_ssm_fwd", *head, None, None, _p(o["y"]), D, _p(o["h"]), _p(ws), B, T, D, N, G, 1, 0, st)
        _lib.call("asca_ssm_bwd", *head, None, _p(b["dy"]), D, None, _p(ws), _p(o["dx"]), D, _p(o["ddt"]), D, _p(o["db"]), _p(o["dA"]),
                  _p(o["dB"]), G * N, _p(o["dC"]), G * N, _p(o["dD"]), _p(o["dh0"]), B, T, D, N, G, 1, 0, st)

    return run, o, (b, ws)


def test_captured_calls_replay_the_eager_results(g):
    """A scan cut into chunks, a convolution, norms and clipping with their backwards,
    captured into a graph: each replay gives the eager bits, with the program's own
    calls between the replays."""
    from asca_amd import _lib, gpu

    hip = C.CDLL("libamdhip64.so.7")

    def ok(rc):
        assert rc == 0, rc

    rng = np.random.default_rng(12)
    r = Rows(rng, False)
    B, T, D, N = 1, 300, 64, 16
    i, dy = ssm_inputs(r, rng, B, T, D, N, 1), r(B * T, D)
    run, o, keep = _ssm_call(g, i, B, T, D, N, dy)
    w = gpu.DevBuf.from_host(rng.standard_normal((4, D)).astype(np.float32))
    bias = gpu.DevBuf.from_host(rng.standard_normal(D).astype(np.float32))
    x, bdy = keep[0]["x"], keep[0]["dy"]
    o.update({k: gpu.DevBuf(n * 4) for k, n in (("c", T * D), ("dc", T * D), ("dw", 4 * D), ("dcb", D), ("r", T * D), ("n", T * D),
                                                ("nx", T * D), ("ny", T * D), ("dwp", D), ("clip", D), ("stat", 2))})
    gl = C.c_void_p()
    one = lambda b: (C.c_void_p * 1)(b.ptr)  # noqa: E731
    _lib.call("asca_grads_create", one(o["dwp"]), one(o["clip"]), (C.c_uint64 * 1)(D), 1, 0, C.byref(gl))

    def everything(st):
        run(st)
        _lib.call("asca_conv_fwd", _p(x), D, _p(w), _p(bias), None, None, _p(o["c"]), D, None, B, T, D, 4, 1, 0, st)
        _lib.call("asca_conv_bwd", _p(x), D, _p(w), _p(bias), None, None, _p(bdy), D, None, _p(o["dc"]), D, _p(o["dw"]), _p(o["dcb"]),
                  None, B, T, D, 4, 1, 0, st)
        _lib.call("asca_block_norm_fwd", _p(x), D, _p(bdy), D, None, 0, _p(bias), None, None, _p(o["r"]), D, _p(o["n"]), D, T, D, 1e-6, 0, st)
        _lib.call("asca_block_norm_bwd", _p(x), D, _p(bdy), D, None, 0, _p(bias), None, None, _p(x), D, _p(bdy), D, _p(o["nx"]), D,
                  _p(o["ny"]), D, None, 0, _p(o["dwp"]), None, None, T, D, 1e-6, 0, st)
        _lib.call("asca_grads_clip", gl, 0.5, _p(o["stat"]), st)

    get = lambda: {k: b.to_host((b.nbytes // 4,)) for k, b in o.items()}  # noqa: E731
    everything(None)
    _lib.call("asca_sync")
    want = get()
    sp, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    _lib.call("asca_stream_create", C.byref(sp))
    ok(hip.hipStreamBeginCapture(sp, 0))
    everything(sp)
    ok(hip.hipStreamEndCapture(sp, C.byref(graph)))
    ok(hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)))
    for k in range(4):
        for b in o.values():
            _lib.call("asca_memset32", _p(b), 0, b.nbytes // 4, None)
        _lib.call("asca_sync")
        ok(hip.hipGraphLaunch(exe, sp))
        _lib.call("asca_stream_sync", sp)
        got = get()
        for name in want:
            np.testing.assert_array_equal(got[name], want[name], err_msg=f"replay {k}: {name}")
        g.conv(i["x"], rng.standard_normal((4, D)).astype(np.float32), batch=1)   # the program's own work between
    ok(hip.hipGraphExecDestroy(exe))
    ok(hip.hipGraphDestroy(graph))
    _lib.call("asca_stream_destroy", sp)
    _lib.call("asca_grads_destroy", gl)


@pytest.mark.parametrize("T,D,N", [(1700, 24, 16), (1700, 24, 20), (4096, 8, 40)])
def test_a_captured_scan_in_chunks_replays_the_eager_results(g, T, D, N):
    """Both passes of a forward that is cut into chunks, with the scratch between them, and
    its backward."""
    from asca_amd import _lib

    hip = C.CDLL("libamdhip64.so.7")

    def ok(rc):
        assert rc == 0, rc

    rng = np.random.default_rng(16)
    r = Rows(rng, False)
    i, dy = ssm_inputs(r, rng, 1, T, D, N, 1), r(T, D)
    run, o, keep = _ssm_call(g, i, 1, T, D, N, dy)
    get = lambda: {k: b.to_host((b.nbytes // 4,)) for k, b in o.items()}  # noqa: E731
    run(None)
    _lib.call("asca_sync")
    want = get()
    sp, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    _lib.call("asca_stream_create", C.byref(sp))
    ok(hip.hipStreamBeginCapture(sp, 0))
    run(sp)
    ok(hip.hipStreamEndCapture(sp, C.byref(graph)))
    ok(hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)))
    for k in range(4):
        for b in o.values():
            _lib.call("asca_memset32", _p(b), 0, b.nbytes // 4, None)
        _lib.call("asca_sync")
        ok(hip.hipGraphLaunch(exe, sp))
        _lib.call("asca_stream_sync", sp)
        got = get()
        for name in want:
            np.testing.assert_array_equal(got[name], want[name], err_msg=f"replay {k}: {name}")
        g.ssm_scan(**i, batch=1, keep=False)   # the program's own work between
    ok(hip.hipGraphExecDestroy(exe))
    ok(hip.hipGraphDestroy(graph))
    _lib.call("asca_stream_destroy", sp)


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("B,T,D,N", [(1, 70, 40, 16), (1, 70, 40, 6), (8, 40, 2048, 16), (1, 1100, 512, 12), (1, 1700, 24, 12), (5, 80, 512, 16)])
def test_an_infinity_or_nan_stays_with_what_it_reaches(g, bad, B, T, D, N):
    """One bad x: its channel from its row on, and the sums over channels of those rows;
    one bad dy: its channel up to its row, and those rows' sums.  Everything else keeps
    its bits."""
    rng = np.random.default_rng(13)
    r = Rows(rng, False)
    i, dy = ssm_inputs(r, rng, B, T, D, N, 1), r(B * T, D)
    row, ch = 21, 3

    def run(i, dy):
        y, h, dev = g.ssm_scan(**i, batch=B)
        o = g.ssm_scan_bwd(dev, dy)
        dev.free()
        return dict(o, y=y, h=h)

    want = run(i, dy)
    rows = np.arange(B * T)
    later, first = (rows >= row) & (rows < T), rows < T
    x2, dy2 = i["x"].copy(), dy.copy()
    x2[row, ch], dy2[row, ch] = bad, bad
    got = run({**i, "x": x2}, dy)
    assert not np.isfinite(got["y"][row, ch])
    clean = np.ones((B * T, D), bool)
    clean[later, ch] = False
    np.testing.assert_array_equal(got["y"][clean], want["y"][clean])
    np.testing.assert_array_equal(got["dC"][~later], want["dC"][~later])
    np.testing.assert_array_equal(got["dB"][rows != row], want["dB"][rows != row])
    assert not np.isfinite(got["dB"][row]).any()
    other = np.arange(D) != ch
    for k in ("dA", "dDk", "ddt_bias"):
        np.testing.assert_array_equal(got[k][..., other], want[k][..., other])
    for k in ("dx", "ddt"):
        np.testing.assert_array_equal(got[k][:, other], want[k][:, other])
    got = run(i, dy2)
    np.testing.assert_array_equal(got["y"], want["y"])
    up = first & (rows <= row)
    clean = np.ones((B * T, D), bool)
    clean[up, ch] = False
    assert not np.isfinite(got["dx"][row, ch])
    for k in ("dx", "ddt"):
        np.testing.assert_array_equal(got[k][clean], want[k][clean])
    np.testing.assert_array_equal(got["dC"][rows != row], want["dC"][rows != row])
    np.testing.assert_array_equal(got["dB"][~up], want["dB"][~up])
