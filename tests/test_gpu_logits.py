"""GPU parity of the operators behind a model's logits (largest logits, distillation,
beam search) against the float64 oracle, through the operator API and the C ABI.

Bounds.  u = 2^-24 is half a step of f32.  A sum of exponentials of V terms, each of an
argument rounded a few times, is off by at most u (V/64 + 48 + 4 log V + 4 x) of itself:
no lane of a wave adds more than V/64 terms one after another, the rest is added by
halves; the arguments' roundings weigh by their terms and that mean is at most log V, or
at most the range x of the arguments for a term alone.  A loss or a gradient is a sum of
terms whose sizes the oracle gives, each off by so much of itself, and is rounded once:
by u of itself in f32, 2^-8 in bf16.  Ids, parents and moved states are exact."""
import ctypes as C

import numpy as np
import pytest

from oracle import logits_oracle as lo

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def delta(z, tau=1.0):
    f = z[np.isfinite(z)]
    x = (f.max() - f.min()) / min(tau, 1.0) if f.size else 0.0
    return U * (z.shape[1] / 64 + 48 + 4 * np.log(z.shape[1]) + 4 * x)


def to_dev(a, bf16):
    """(what the device gets, its float64 values)"""
    from asca_amd import gpu

    a = np.asarray(a, np.float32)
    if not bf16:
        return a, a.astype(np.float64)
    b = gpu.to_bf16(a)
    return b, gpu.from_bf16(b).astype(np.float64)


def value(a):
    from asca_amd import gpu

    return (gpu.from_bf16(a) if a.dtype == np.uint16 else a).astype(np.float64)


def logits(rng, rows, V, bf16, spread=1.5):
    z = rng.standard_normal((rows, V)) * spread
    for r in range(rows):
        for c in rng.integers(0, V, min(6, V)):
            z[r, c] += 3 + 2 * rng.standard_normal()
    return to_dev(z, bf16)


class Strided:
    """A device matrix of wider rows that begins some elements into its buffer."""

    def __init__(self, a, pad=0, off=0, fill=None):
        from asca_amd import gpu

        self.shape, self.ld, self.off = a.shape, a.shape[1] + pad, off
        host = np.full(off + a.shape[0] * self.ld + 8, 0x7f7f if a.dtype == np.uint16 else 1e30, a.dtype)
        self.view(host)[:] = a if fill is None else fill
        self.before, self.buf, self.size = host, gpu.DevBuf.from_array(host), a.itemsize
        self.ptr = C.c_void_p(self.buf.ptr + off * a.itemsize)

    def view(self, host):
        rows, cols = self.shape
        return host[self.off:self.off + rows * self.ld].reshape(rows, self.ld)[:, :cols]

    def get(self):
        """The matrix; nothing beside it has changed."""
        host = self.buf.to_host(self.before.shape, self.before.dtype)
        out = self.view(host).copy()
        self.view(host)[:] = 0
        rest = self.before.copy()
        self.view(rest)[:] = 0
        np.testing.assert_array_equal(host, rest)
        return out


def _p(b):
    return C.c_void_p(None if b is None else b.ptr)


def up(a, dtype=None):
    from asca_amd import gpu

    return None if a is None else gpu.DevBuf.from_array(np.asarray(a, dtype or np.asarray(a).dtype))


# ---------------------------------------------------------- largest logits

TOP = [(1, 1, 1), (3, 1, 4), (2, 5, 8), (5, 63, 64), (1, 64, 64), (7, 256, 16), (4, 257, 5), (70, 255, 1), (3, 1000, 64),
       (9, 513, 20), (2, 2049, 64), (5, 4096, 7), (2, 4097, 33), (1, 32768, 8), (3, 8193, 64), (2, 50001, 64), (3, 131072, 64),
       (1, 200003, 10), (300, 300, 3), (600, 5000, 40)]


def check_top(got, z, K, tau=1.0):
    v, i, s = got
    rv, ri, rs = lo.top(z, K, tau)
    np.testing.assert_array_equal(i, ri)
    np.testing.assert_array_equal(np.asarray(v, np.float64), rv)
    bad = ~np.isfinite(rs)
    assert not np.isfinite(s[bad]).any()
    d = np.abs(s[~bad] - rs[~bad])
    assert (d <= U * np.abs(rs[~bad]) + delta(z, tau)).all(), d.max()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,V,K", TOP)
def test_top(g, rows, V, K, bf16):
    print(f"[top] rows={rows} V={V} K={K} bf16={bf16}", flush=True)
    z, val = logits(np.random.default_rng(rows + V + K), rows, V, bf16)
    for tau in (1.0, 3.0):
        check_top(g.top_logits(z, K, tau), val, K, tau)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pad,off", [(0, 0), (1, 0), (3, 1), (8, 5), (5, 7)])
@pytest.mark.parametrize("rows,V,K", [(5, 33, 9), (9, 250, 16), (4, 3001, 30), (3, 20001, 64)])
def test_top_of_strided_rows(g, rows, V, K, pad, off, bf16):
    from asca_amd import _lib, gpu

    z, val = logits(np.random.default_rng(V + pad), rows, V, bf16)
    m = Strided(z, pad, off)
    v, i, s = gpu.DevBuf(rows * K * 4), gpu.DevBuf(rows * K * 4), gpu.DevBuf(rows * 4)
    for lse in (s, None):
        _lib.call("asca_top_logits", m.ptr, m.ld, rows, V, K, 1.0, _p(v), _p(i), _p(lse), int(bf16), None)
    _lib.call("asca_sync")
    check_top((v.to_host((rows, K)), i.to_host((rows, K), np.int32), s.to_host((rows,))), val, K)
    m.get()


# as many rows as fill the device: a wave's rows of each number of pieces, whole rows and slices of a block
MANY = [(1100, 100, 64), (1030, 256, 31), (1030, 300, 16), (1100, 700, 64), (1030, 1900, 20), (1025, 3900, 33), (1040, 9000, 64),
        (1050, 20011, 5), (1030, 33001, 17)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,V,K", MANY)
def test_top_of_many_rows(g, rows, V, K, bf16):
    from asca_amd import _lib, gpu

    print(f"[top] rows={rows} V={V} K={K} bf16={bf16}", flush=True)
    rng = np.random.default_rng(rows + V)
    z, val = to_dev(rng.standard_normal((rows, V)), bf16)
    m = Strided(z, 1, 1)
    v, i, s = gpu.DevBuf(rows * K * 4), gpu.DevBuf(rows * K * 4), gpu.DevBuf(rows * 4)
    _lib.call("asca_top_logits", m.ptr, m.ld, rows, V, K, 0.7, _p(v), _p(i), _p(s), int(bf16), None)
    _lib.call("asca_sync")
    check_top((v.to_host((rows, K)), i.to_host((rows, K), np.int32), s.to_host((rows,))), val, K, 0.7)


@pytest.mark.parametrize("V", [90, 1000, 30000])
def test_top_of_large_logits(g, V):
    """Logits whose scaled size is past what one step of the exponent's argument keeps."""
    rng = np.random.default_rng(V)
    z = (rng.standard_normal((4, V)) + np.array([[1e5], [-1e5], [3e6], [-1e30]])).astype(np.float32)
    for tau in (1.0, 0.01):
        v, i, s = g.top_logits(z, 7, tau)
        rv, ri, rs = lo.top(z, 7, tau)
        np.testing.assert_array_equal(i, ri)
        np.testing.assert_array_equal(v, rv)
        assert (np.abs(s - rs) <= U * np.abs(rs) + delta(z[:1], tau)).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,V,K", [(1, 1 << 20, 64), (2, (1 << 21) + 3, 17)])
def test_top_of_the_longest_rows(g, rows, V, K, bf16):
    """A thread adds at most 16 pieces of 8, a lane then a few slices' sums: 136 terms."""
    z, val = logits(np.random.default_rng(V), rows, V, bf16)
    got = g.top_logits(z, K)
    check_top(got, val, K)
    rs = lo.top(val, K)[2]
    assert (np.abs(got[2] - rs) <= U * np.abs(rs) + U * (136 + 48 + 4 * np.log(V) + 4 * np.ptp(val))).all()


def orders(V):
    """Rows in which the largest lie where a selection by parts goes wrong."""
    up_ = np.arange(V) / 64.0
    few = np.full(V, -np.inf)
    few[[V - 1, V // 2]] = [1.0, 2.0]
    step = -np.abs(np.random.default_rng(0).standard_normal(V))
    step[::256] = 5 + np.arange(len(step[::256])) / 128
    wide = -np.abs(np.random.default_rng(1).standard_normal(V))
    wide[::1024] = 5 + np.arange(len(wide[::1024])) / 128
    return dict(up=up_, down=up_[::-1], equal=np.full(V, 0.5), two=np.arange(V) % 2 * 1.0, few=few, none=np.full(V, -np.inf),
                step=step, wide=wide, zeros=np.where(np.arange(V) % 3 == 0, -0.0, 0.0), low=np.full(V, -3e38),
                runs=np.repeat(np.arange(-(-V // 100)), 100)[:V] / 8.0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V,K", [(40, 64), (700, 64), (5000, 64), (5000, 3), (70000, 64)])
def test_top_of_ordered_equal_and_masked_rows(g, V, K, bf16):
    rows = orders(V)
    z, val = to_dev(np.stack(list(rows.values())), bf16)
    got = g.top_logits(z, K)
    for r, name in enumerate(rows):
        print(f"[top] {name} V={V} K={K}", flush=True)
        check_top([a[r:r + 1] for a in got], val[r:r + 1], K)


def test_top_of_infinities_and_nan(g):
    z = np.random.default_rng(5).standard_normal((6, 3000)).astype(np.float32)
    z[0, 7] = np.nan
    z[1, 8] = np.inf
    z[2, [9, 2999]] = [np.inf, np.nan]
    z[3] = np.nan
    z[4, 100:] = -np.inf
    check_top(g.top_logits(z, 5), z.astype(np.float64), 5)


# -------------------------------------------------------------- distillation

DISTILL = [(1, 1, 1), (2, 5, 8), (3, 64, 1), (5, 100, 64), (9, 256, 16), (4, 257, 5), (2, 1001, 20), (3, 2048, 33), (2, 5003, 64),
           (2, 16385, 7), (2, 33000, 64), (1, 70001, 40), (1, 131072, 64), (1, 300001, 3), (130, 600, 9), (700, 40, 4)]


def teacher(rng, val, K, tau, ragged=False):
    T, V = val.shape
    t = val + rng.standard_normal((T, V))
    k = min(K, V)
    ids = np.argsort(-t, axis=1, kind="stable")[:, :k]
    tv = np.take_along_axis(t, ids, 1).astype(np.float32)
    tl = np.array([lo.lse(r / tau) for r in t], np.float32)
    if k < K:
        ids, tv = np.pad(ids, ((0, 0), (0, K - k)), constant_values=-1), np.pad(tv, ((0, 0), (0, K - k)))
    if ragged:
        n = rng.integers(0, K + 1, T)
        ids = np.where(np.arange(K) < n[:, None], ids, rng.choice([-1, V, -7], (T, K)))
    return tv, ids.astype(np.int32), tl


def check_distill(got, val, tv, ids, bf16, **kw):
    L, dz, (tl, tg) = lo.distill(val, tv, ids, **kw)
    d = delta(val, kw.get("temperature", 1.0))
    e = np.abs(got[0] - L)
    assert (e <= U * np.abs(L) + d * tl).all(), (e.max(), tl[e.argmax()])
    if got[1] is not None:
        e = np.abs(value(got[1]) - dz)
        lim = (2.0 ** -8 if bf16 else U) * np.abs(dz) + d * tg + 1e-37
        assert (e <= lim).all(), (e.max(), np.unravel_index((e - lim).argmax(), e.shape))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V,K", DISTILL)
def test_distill(g, T, V, K, bf16):
    rng = np.random.default_rng(T + V + K)
    z, val = logits(rng, T, V, bf16)
    w = np.where(np.arange(T) % 3 == 1, 0.0, rng.uniform(0.5, 2, T)).astype(np.float32)
    tg = rng.integers(0, V + 1, T)   # V: none
    for rest, alpha, tau, ragged in ((True, 0.5, 2.0, False), (False, 1.0, 1.0, False), (True, 1.0, 1.0, True), (False, 0.3, 1.0, True),
                                     (True, 0.0, 1.0, False), (False, 0.9, 4.0, True), (True, 0.7, 0.5, False)):
        print(f"[distill] T={T} V={V} K={K} bf16={bf16} rest={rest} alpha={alpha} tau={tau} ragged={ragged}", flush=True)
        tv, ids, tl = teacher(rng, val, K, tau, ragged)
        kw = dict(tlse=tl if rest else None, targets=tg if alpha < 1 else None, weights=w if ragged else None, temperature=tau,
                  alpha=alpha, scale=0.37)
        check_distill(g.distill(z, tv, ids, **kw), val, tv, ids, bf16, **kw)
    L = g.distill(z, tv, ids, **kw)[0]
    L2, none = g.distill(z, tv, ids, grad=False, **kw)
    assert none is None
    np.testing.assert_array_equal(L, L2)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V", [(1, 1 << 20), (2, 600001), (2, (1 << 20) - 3), (3, 524293)])
def test_distill_of_the_longest_rows(g, T, V, bf16):
    """The largest bitmap, and rows of more slices than a split has; entries and targets in the last
    columns.  A thread adds up to 4 pieces of 8, then up to 64 such sums one after another: 96 terms."""
    print(f"[distill] T={T} V={V} bf16={bf16}", flush=True)
    rng = np.random.default_rng(V)
    z, val = logits(rng, T, V, bf16)
    K = 7
    tv, ids, tl = teacher(rng, val, K, 2.0)
    ids[:, 0], ids[:, 1], ids[:, 2] = V - 1, V - 2, 0
    tg = np.array([V - 1, V - 3, V - 9])[:T]
    d = delta(val[:, :64 * 96]) + U * 4 * (np.ptp(val) + np.log(V))
    for rest, alpha in ((True, 0.5), (False, 1.0)):
        kw = dict(tlse=tl + np.float32(0.5) if rest else None, targets=tg if alpha < 1 else None, temperature=2.0, alpha=alpha)
        got = g.distill(z, tv, ids, **kw)
        L, dz, (sl, sg) = lo.distill(val, tv, ids, **kw)
        assert (np.abs(got[0] - L) <= U * np.abs(L) + d * sl).all()
        assert (np.abs(value(got[1]) - dz) <= (2.0 ** -8 if bf16 else U) * np.abs(dz) + d * sg + 1e-37).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("pad,off,gpad,goff", [(0, 0, 0, 0), (1, 0, 1, 0), (3, 1, 3, 1), (8, 5, 0, 0), (5, 7, 2, 3)])
@pytest.mark.parametrize("T,V,K", [(5, 33, 9), (9, 250, 16), (3, 3001, 30), (2, 40001, 64)])
def test_distill_of_strided_rows(g, T, V, K, pad, off, gpad, goff, inplace, bf16):
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(V + pad)
    z, val = logits(rng, T, V, bf16)
    tv, ids, tl = teacher(rng, val, K, 2.0)
    tg = rng.integers(0, V, T)
    m = Strided(z, pad, off)
    out = m if inplace else Strided(z, gpad, goff, fill=0)
    ls, bt, bi, bl, btg = gpu.DevBuf(T * 4), up(tv), up(ids), up(tl), up(tg, np.uint32)
    _lib.call("asca_distill", m.ptr, m.ld, _p(bt), _p(bi), _p(bl), K, _p(btg), None, 2.0, 0.5, 1.0, _p(ls), out.ptr, out.ld, T, V,
              int(bf16), None)
    _lib.call("asca_sync")
    check_distill((ls.to_host((T,)), out.get()), val, tv, ids, bf16, tlse=tl, targets=tg, temperature=2.0, alpha=0.5)
    if not inplace:
        np.testing.assert_array_equal(m.get(), z)


# rows that are not few for their length, in each number of waves and pieces
ROWS = [(1030, 5, 3), (1030, 130, 9), (1030, 300, 16), (1030, 700, 33), (1030, 1500, 5), (1030, 3500, 64), (40, 1003, 20), (40, 3001, 7),
        (40, 5003, 64), (40, 9001, 11), (40, 17001, 30), (36, 30001, 64), (130, 40001, 5), (130, 70003, 64), (129, 140001, 3)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("T,V,K", ROWS)
def test_distill_of_many_rows(g, T, V, K, inplace, bf16):
    from asca_amd import _lib, gpu

    print(f"[distill] T={T} V={V} K={K} bf16={bf16} inplace={inplace}", flush=True)
    rng = np.random.default_rng(T + V)
    z, val = to_dev(rng.standard_normal((T, V)) * 2, bf16)
    ids = rng.integers(-1, V, (T, K)).astype(np.int32)   # some twice
    tv = (rng.standard_normal((T, K)) + 3).astype(np.float32)
    tl = np.array([lo.lse(r.astype(np.float64) / 2) for r in tv], np.float32) + 0.3
    tg, w = rng.integers(0, V + 2, T), np.where(np.arange(T) % 5 == 2, 0, rng.uniform(0.5, 2, T)).astype(np.float32)
    m = Strided(z, 1, 1)
    out = m if inplace else Strided(z, 1, 1, fill=0)
    ls, bt, bi, bl, btg, bw = gpu.DevBuf(T * 4), up(tv), up(ids), up(tl), up(tg, np.uint32), up(w)
    rest = not inplace
    _lib.call("asca_distill", m.ptr, m.ld, _p(bt), _p(bi), _p(bl if rest else None), K, _p(btg), _p(bw), 2.0, 0.5, 1.0, _p(ls), out.ptr,
              out.ld, T, V, int(bf16), None)
    _lib.call("asca_sync")
    check_distill((ls.to_host((T,)), out.get()), val, tv, ids, bf16, tlse=tl if rest else None, targets=tg, weights=w, temperature=2.0,
                  alpha=0.5)


@pytest.mark.parametrize("T,V", [(3, 60), (3, 900), (40, 9001), (2, 40000), (130, 70003)])
def test_distill_of_large_logits(g, T, V):
    """Logits whose scaled size is past what one step of the exponent's argument keeps: the same
    losses and gradients as without what all of a row have in common."""
    rng = np.random.default_rng(V)
    z = np.round(rng.standard_normal((T, V)) * 64) / 64
    ids = np.stack([rng.permutation(V)[:6] for _ in range(T)]).astype(np.int32)
    tv = rng.standard_normal((T, 6)).astype(np.float32)
    tl = np.array([lo.lse(r.astype(np.float64) / 2) for r in tv], np.float32) + 0.2
    kw = dict(tlse=tl, targets=ids[:, 1], temperature=2.0, alpha=0.5)
    for add in (0.0, 1e5, -1e5, 2.0 ** 17):   # exact sums in f32
        x = (z + add).astype(np.float32)
        got = g.distill(x, tv, ids, **kw)
        L, dz, (tl_, tg_) = lo.distill(z, tv, ids, **kw)
        d = delta(z)
        assert (np.abs(got[0] - L) <= U * np.abs(L) + d * tl_).all() and (np.abs(got[1] - dz) <= U * np.abs(dz) + d * tg_ + 1e-37).all()


@pytest.mark.parametrize("V", [50, 700, 9000, 40000, 140000])
def test_distill_entries_of_one_id(g, V):
    """Entries of one id are one with the sum of their p, whatever their order."""
    rng = np.random.default_rng(V)
    z, val = logits(rng, 4, V, False)
    tv, ids, tl = teacher(rng, val, 12, 1.0)
    ids[0, :] = ids[0, 0]
    ids[1, [3, 7, 11]] = ids[1, 3]
    ids[2, 6:] = ids[2, :6]
    for tlse in (tl + 3, None):
        kw = dict(tlse=tlse, targets=ids[:, 0], temperature=1.0, alpha=0.8)
        check_distill(g.distill(z, tv, ids, **kw), val, tv, ids, False, **kw)


@pytest.mark.parametrize("V", [50, 700, 9000, 40000, 140000])
def test_distill_of_a_student_sure_of_its_list(g, V):
    """The other ids' sum is 1e-20 and less of the whole, and their gradient still the rest's
    share among them; and the other way round."""
    rng = np.random.default_rng(V)
    z = rng.standard_normal((3, V)).astype(np.float32)
    ids = np.stack([rng.permutation(V)[:6] for _ in range(3)]).astype(np.int32)
    tv = rng.standard_normal((3, 6)).astype(np.float32)
    tl = np.array([lo.lse(r.astype(np.float64)) for r in tv], np.float32) + 0.2
    for lift in (60.0, 150.0, -60.0, -150.0):
        x = z.copy()
        for r in range(3):
            x[r, ids[r]] += lift
        for kw in (dict(tlse=tl, alpha=1.0), dict(tlse=tl, alpha=0.5, targets=ids[:, 1]), dict(alpha=0.5, targets=(ids[:, 1] + 1) % V)):
            check_distill(g.distill(x, tv, ids, **kw), x.astype(np.float64), tv, ids, False, **kw)


@pytest.mark.parametrize("V", [60, 900, 9000, 140000])
def test_distill_of_masked_logits(g, V):
    """-inf logits: no gradient there; a rest that no other id can give is left out."""
    rng = np.random.default_rng(V)
    z = rng.standard_normal((4, V)).astype(np.float32)
    ids = np.stack([rng.permutation(V)[:6] for _ in range(4)]).astype(np.int32)
    tv = rng.standard_normal((4, 6)).astype(np.float32)
    tl = np.array([lo.lse(r.astype(np.float64)) for r in tv], np.float32) + 0.2
    for r in range(3):   # rows 0 and 1 only the list, row 2 the list and one more
        keep = np.append(ids[r], [(set(range(V)) - set(ids[r])).pop()] if r == 2 else []).astype(int)
        m = np.full(V, -np.inf, np.float32)
        m[keep] = z[r, keep]
        z[r] = m
    tv[1, 3] = -np.inf   # p = 0 where the student has its own mask
    z[1, ids[1, 3]] = -np.inf
    for kw in (dict(tlse=tl), dict(), dict(tlse=tl, alpha=0.4, targets=ids[:, 0], temperature=2.0)):
        got = g.distill(z, tv, ids, **kw)
        check_distill(got, z.astype(np.float64), tv, ids, False, **kw)
        assert (got[1][0][np.isinf(z[0])] == 0).all()
    tv[1, 3] = 0.0       # the teacher gives what the student cannot: an infinite loss, a finite gradient
    L, dz = g.distill(z, tv, ids)
    assert L[1] == np.inf and np.isfinite(dz).all() and np.isfinite(L[[0, 2, 3]]).all()


@pytest.mark.parametrize("V", [60, 900, 9000, 140000])
def test_distill_rows_without_weight_or_entries(g, V):
    rng = np.random.default_rng(V)
    z, val = logits(rng, 6, V, False)
    tv, ids, tl = teacher(rng, val, 5, 1.0)
    z[1], z[4, 3] = np.nan, np.inf
    w = np.array([1, 0, 1, 1, 0, 1], np.float32)
    ids[2], tv[3] = -1, -np.inf
    for tlse in (tl, None):
        L, dz = g.distill(z, tv, ids, tlse=tlse, weights=w)
        assert np.isfinite(L).all() and np.isfinite(dz).all()
        assert L[1] == L[4] == 0 and not dz[[1, 4]].any()
        assert L[2] == 0 and np.abs(dz[2]).max() <= 2 * delta(val)   # one class alone: nothing to learn
        ok = [0, 2, 5]
        t = None if tlse is None else tlse[ok]
        check_distill((L[ok], dz[ok]), val[ok], tv[ok], ids[ok], False, tlse=t)
    assert L[3] == 0 and not dz[3].any() and not dz[2].any()         # an empty softmax
    # a NaN reaches its own row alone
    L, dz = g.distill(z, tv, ids)
    assert np.isnan(L[1]) and np.isnan(dz[1]).all() and np.isfinite(dz[[0, 2, 3, 5]]).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_distill_gradient_against_differences(g, bf16):
    """The loss along a direction, by the library's own losses."""
    rng = np.random.default_rng(9)
    T, V, K, tau = 6, 500, 10, 2.0
    z, val = logits(rng, T, V, False)
    tv, ids, tl = teacher(rng, val, K, tau)
    kw = dict(tlse=tl, targets=rng.integers(0, V, T), temperature=tau, alpha=0.6)
    if bf16:
        z, val = to_dev(z, True)
        z = value(z).astype(np.float32)
    dz = g.distill(z, tv, ids, **kw)[1].astype(np.float64)
    h = 2.0 ** -4
    step = (dz / np.linalg.norm(dz, axis=1, keepdims=True)).astype(np.float32)
    up_, dn = (lo.distill(z.astype(np.float64) + s * h * step, tv, ids, **kw)[0] for s in (1, -1))
    lib_up, lib_dn = (g.distill((z + np.float32(s * h) * step).astype(np.float32), tv, ids, grad=False, **kw)[0] for s in (1, -1))
    got = (lib_up.astype(np.float64) - lib_dn) / (2 * h)
    want = (dz * step).sum(1)
    third = np.abs((up_ - dn) / (2 * h) - want) + 1e-12   # of the differences themselves
    sizes = lo.distill(z.astype(np.float64), tv, ids, **kw)[2][0]
    assert (np.abs(got - want) <= 2 * third + 2 * (delta(val, tau) * sizes + U * 20) / h).all()


def test_rows_past_32_bits(g):
    """2.2e9 logits: the last rows' offsets pass 32 bits, in elements and in bytes."""
    from asca_amd import _lib, gpu

    rows, V, K = 33000, 65537, 5
    z = gpu.DevBuf(rows * V * 2)
    _lib.call("asca_memset32", _p(z), 0x3f803f80, rows * V // 2, None)   # ones
    rng = np.random.default_rng(2)
    last, val = logits(rng, 3, V, True)
    _lib.call("asca_sync")
    _lib.call("asca_h2d", C.c_void_p(z.ptr + (rows - 3) * V * 2), last.ctypes.data_as(C.c_void_p), C.c_size_t(last.nbytes))
    v, i, s, ls = (gpu.DevBuf(rows * k * 4) for k in (K, K, 1, 1))
    _lib.call("asca_top_logits", _p(z), V, rows, V, K, 1.0, _p(v), _p(i), _p(s), 1, None)
    _lib.call("asca_sync")
    hv, hi, hs = v.to_host((rows, K)), i.to_host((rows, K), np.int32), s.to_host((rows,))
    check_top((hv[-3:], hi[-3:], hs[-3:]), val, K)
    assert (hi[:-3] == np.arange(K)).all() and (hv[:-3] == 1).all()
    _lib.call("asca_distill", _p(z), V, _p(v), _p(i), None, K, None, None, 1.0, 1.0, 1.0, _p(ls), _p(z), V, rows, V, 1, None)
    _lib.call("asca_sync")
    out = np.empty((3, V), np.uint16)
    _lib.call("asca_d2h", out.ctypes.data_as(C.c_void_p), C.c_void_p(z.ptr + (rows - 3) * V * 2), C.c_size_t(out.nbytes))
    check_distill((ls.to_host((rows,))[-3:], out), val, hv[-3:], hi[-3:], True)
    for b in (z, v, i, s, ls):
        b.free()
    _lib.call("asca_pool_release")


# --------------------------------------------------------------- beam search

BEAM = [(1, 1, 1), (1, 4, 2), (3, 5, 7), (1, 4, 256), (7, 4, 256), (2, 8, 1000), (5, 3, 4099), (1, 32, 300), (2, 16, 9001), (1, 5, 70000),
        (3, 2, 33000), (40, 4, 600), (2, 32, 20000), (300, 2, 50)]


def check_step(got, val, scores, K, ended=None, eos=-1, stay=False):
    s, tok, par, end = lo.beam_step(val, scores, K, ended, eos, stay)
    assert (par == got[2]).all() and (tok == got[1]).all(), (tok, got[1], par, got[2])
    fin = np.isfinite(s)
    np.testing.assert_array_equal(got[0][~fin], s[~fin])
    assert (np.abs(got[0][fin] - s[fin]) <= U * np.abs(s[fin]) + delta(val)).all()
    if ended is not None:
        np.testing.assert_array_equal(got[3], end)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("G,K,V", BEAM)
def test_beam_step(g, G, K, V, bf16):
    rng = np.random.default_rng(G * 100 + K + V)
    z, val = logits(rng, G * K, V, bf16)
    sc = (-5 - 3 * rng.random(G * K)).astype(np.float32)
    for stay in (False, True):
        print(f"[beam] G={G} K={K} V={V} bf16={bf16} stay={stay}", flush=True)
        check_step(g.beam_step(z, sc, k=K, stay=stay), val, sc, K, stay=stay)
        end = (rng.random(G * K) < 0.3).astype(np.int32) * rng.integers(1, 9, G * K).astype(np.int32)
        dead = np.where(rng.random(G * K) < 0.3, -np.inf, sc).astype(np.float32)
        eos = int(rng.integers(0, V))
        z2 = z.copy()
        z2[end != 0] = to_dev(np.full(1, np.nan), bf16)[0][0]   # an ended beam's logits are not read
        check_step(g.beam_step(z2, dead, k=K, ended=end, eos=eos, stay=stay), value(z2), dead, K, end, eos, stay)


@pytest.mark.parametrize("stay", [False, True])
def test_beam_first_step(g, stay):
    """One beam counts: its K best tokens in order."""
    rng = np.random.default_rng(4)
    z, val = logits(rng, 12, 500, False)
    sc = np.where(np.arange(12) % 6 == 0, 0.0, -np.inf).astype(np.float32)
    check_step(g.beam_step(z, sc, k=6, stay=stay), val, sc, 6, stay=stay)


@pytest.mark.parametrize("V", [30000, 70000])
def test_beam_first_step_of_many_beams(g, V):
    """A single beam of 32 counts, whose slices' first keys are fewer than the beams."""
    rng = np.random.default_rng(V)
    z, val = to_dev(rng.standard_normal((64, V)), False)
    sc = np.where(np.arange(64) % 32 == 5, -1.0, -np.inf).astype(np.float32)
    for stay in (False, True):
        check_step(g.beam_step(z, sc, k=32, stay=stay), val, sc, 32, stay=stay)


@pytest.mark.parametrize("G,K,V", [(600, 9, 256), (300, 4, 2100), (300, 16, 700), (260, 4, 9001)])
def test_beam_step_of_many_groups(g, G, K, V):
    rng = np.random.default_rng(G)
    z, val = to_dev(rng.standard_normal((G * K, V)) * 2, True)
    sc = (-5 - 3 * rng.random(G * K)).astype(np.float32)
    end = (rng.random(G * K) < 0.2).astype(np.int32)
    check_step(g.beam_step(z, sc, k=K, ended=end, eos=3, stay=True), val, sc, K, end, 3, True)


@pytest.mark.parametrize("V", [3, 50, 3000, 70000])
@pytest.mark.parametrize("stay", [False, True])
def test_beam_ties_go_to_the_lowest_place(g, V, stay):
    """Equal logits everywhere, and equal scores: beams before tokens."""
    for K in (2, 5, 32):
        z = np.zeros((2 * K, V), np.float32)
        sc = np.full(2 * K, -1.0, np.float32)
        got = g.beam_step(z, sc, k=K, stay=stay)
        check_step(got, z.astype(np.float64), sc, K, stay=stay)
        z[:, V // 2:] = 1.0   # runs of equals
        check_step(g.beam_step(z, sc, k=K, stay=stay), z.astype(np.float64), sc, K, stay=stay)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pad,off", [(0, 0), (4, 0), (0, 3)])
@pytest.mark.parametrize("G,K,V", [(9, 3, 37), (9, 4, 257), (3, 16, 257), (9, 4, 2001), (2, 5, 9001), (2, 3, 50001), (300, 4, 2501)])
def test_beams_of_the_same_logits_tie(g, G, K, V, pad, off, bf16):
    """A group's beams have one row's logits and one score, at addresses that differ by elements:
    each token ties over the beams, and the ties go to the lowest one."""
    from asca_amd import _lib, gpu

    z, val = to_dev(np.repeat(np.random.default_rng(G + V + off).standard_normal((G, V)) * 2, K, 0), bf16)
    n, sc = G * K, np.repeat(-np.random.default_rng(V).random(G), K).astype(np.float32)
    m, bs, out, tok, par = Strided(z, pad, off), up(sc), gpu.DevBuf(n * 4), gpu.DevBuf(n * 4), gpu.DevBuf(n * 4)
    for stay in (False, True):
        _lib.call("asca_beam_step", m.ptr, m.ld, _p(bs), None, -1, int(stay), _p(out), None, _p(tok), _p(par), G, K, V, int(bf16), None)
        _lib.call("asca_sync")
        check_step((out.to_host((n,)), tok.to_host((n,), np.uint32), par.to_host((n,), np.int32)), val, sc, K, stay=stay)


@pytest.mark.parametrize("V", [40, 300, 3000, 40000])
@pytest.mark.parametrize("stay", [False, True])
def test_beam_logits_below_a_score_s_rounding(g, V, stay):
    """Logits too small to change a beam's sum in 64 bits: its tokens come in the logits' order
    whatever the number of beams, after an equal beam's before them."""
    tiny = np.float32(1e-20)
    first = None
    for K in (32, 8, 3, 1):
        z = np.zeros((K, V), np.float32)
        z[:, 1::2] = -1.0
        order = np.random.default_rng(V).permutation(np.arange(0, V, 2))[:12]
        z[:, order] = tiny * np.arange(12, 0, -1, dtype=np.float32)   # the largest first
        sc = np.where(np.arange(K) < 2, -1.0, -np.inf).astype(np.float32)
        got = g.beam_step(z, sc, k=K)
        picks = list(zip(got[2].tolist(), got[1].tolist()))
        want = [(b, int(t)) for b in range(2) for t in [*order, *np.setdiff1d(np.arange(0, V, 2), order)]][:K]
        assert picks == want
        first = first or picks
        assert picks == first[:K]
        check_step(g.beam_step(z, sc, k=K, stay=stay), z.astype(np.float64), sc, K, stay=stay)


@pytest.mark.parametrize("V", [9, 300, 40000])
@pytest.mark.parametrize("stay", [False, True])
def test_beam_masks_leave_few_or_no_candidates(g, V, stay):
    rng = np.random.default_rng(V)
    K = 6
    z = rng.standard_normal((4 * K, V)).astype(np.float32)
    sc = -rng.random(4 * K).astype(np.float32)
    z[:K] = -np.inf                   # group 0: nothing
    z[K:2 * K] = -np.inf              # group 1: three candidates in two beams
    z[K + 1, [2, V - 1]], z[K + 4, 5] = [0.5, 0.25], 1.0
    z[2 * K, 3], z[2 * K + 1, 4] = np.nan, np.inf       # group 2: beams whose sums are not finite
    sc[2 * K + 2] = np.nan
    sc[3 * K:] = -np.inf              # group 3: every beam dead
    val = z.astype(np.float64)
    val[2 * K + 1, 4] = np.inf
    check_step(g.beam_step(z, sc, k=K, stay=stay), val, sc, K, stay=stay)
    end = np.zeros(4 * K, np.int32)
    end[[0, K]] = 1
    check_step(g.beam_step(z, sc, k=K, ended=end, eos=1, stay=stay), val, sc, K, end, 1, stay)


def test_beam_step_over_its_inputs(g):
    """new_scores and new_ended may be scores and ended; strided logits."""
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(8)
    G, K, V = 3, 4, 1003
    z, val = logits(rng, G * K, V, True)
    sc, end = -rng.random(G * K).astype(np.float32), (np.arange(G * K) % 5 == 0).astype(np.int32)
    m, bs, be, tok, par = Strided(z, 3, 1), up(sc), up(end), gpu.DevBuf(G * K * 4), gpu.DevBuf(G * K * 4)
    _lib.call("asca_beam_step", m.ptr, m.ld, _p(bs), _p(be), 7, 1, _p(bs), _p(be), _p(tok), _p(par), G, K, V, 1, None)
    _lib.call("asca_sync")
    n = G * K
    check_step((bs.to_host((n,)), tok.to_host((n,), np.uint32), par.to_host((n,), np.int32), be.to_host((n,), np.int32)), val, sc, K, end,
               7, True)
    m.get()


STATES = [(1, 1, 1, 4), (2, 3, 4, 100), (3, 5, 8, 4096), (1, 7, 32, 48), (8, 2, 4, 16384), (2, 33, 5, 3996), (1, 2, 3, 1), (2, 3, 5, 17),
          (1, 130, 2, 8200)]


@pytest.mark.parametrize("outer,G,K,nbytes", STATES)
def test_beam_states(g, outer, G, K, nbytes):
    from asca_amd import gpu

    rng = np.random.default_rng(nbytes + K)
    a = rng.integers(0, 256, (outer, G * K, nbytes)).astype(np.uint8)
    for kind in ("any", "same", "self", "stay", "outside"):
        print(f"[states] outer={outer} G={G} K={K} bytes={nbytes} {kind}", flush=True)
        par = rng.integers(0, K, G * K)
        if kind == "same":
            par[:] = K - 1
        if kind == "self":
            par = np.tile(np.arange(K), G)
        if kind == "stay":
            par = np.where(rng.random(G * K) < 0.5, np.tile(np.arange(K), G), 0)
        if kind == "outside":
            par = np.where(rng.random(G * K) < 0.4, rng.choice([-1, K, 1 << 30, -(1 << 31)], G * K), par)
        par = par.astype(np.int32)
        buf = gpu.DevBuf.from_array(a)
        g.beam_states([(buf, None, outer, nbytes)], par, groups=G, k=K)
        np.testing.assert_array_equal(buf.to_host(a.shape, np.uint8), lo.beam_states(a, a, par, G, K, K))
        buf.upload(a)
        dst0 = np.full_like(a, 9)
        dst = gpu.DevBuf.from_array(dst0)
        g.beam_states([(buf, dst, outer, nbytes)], gpu.DevBuf.from_array(par), groups=G, k=K)
        np.testing.assert_array_equal(dst.to_host(a.shape, np.uint8), lo.beam_states(a, dst0, par, G, K, K))
        np.testing.assert_array_equal(buf.to_host(a.shape, np.uint8), a)


@pytest.mark.parametrize("ks,kd", [(1, 4), (1, 32), (5, 1), (3, 8), (32, 2)])
def test_beam_states_fork_and_pick(g, ks, kd):
    from asca_amd import gpu

    rng = np.random.default_rng(ks + kd)
    outer, G = 2, 3
    shapes = [(outer, G, 400), (1, G, 52), (3, G, 7)]
    src = [rng.integers(0, 256, (o, n * ks, b)).astype(np.uint8) for o, n, b in shapes]
    dst = [np.full((o, n * kd, b), 7, np.uint8) for o, n, b in shapes]
    for par in (None, rng.integers(0, ks, G * kd).astype(np.int32)):
        bs, bd = [gpu.DevBuf.from_array(a) for a in src], [gpu.DevBuf.from_array(a) for a in dst]
        g.beam_states([(x, y, o, b) for x, y, (o, _, b) in zip(bs, bd, shapes)], par, groups=G, k=kd, k_src=ks)
        for x, a, y in zip(src, dst, bd):
            np.testing.assert_array_equal(y.to_host(a.shape, np.uint8), lo.beam_states(x, a, par, G, ks, kd))


def test_beam_states_of_many_buffers_at_odd_addresses(g):
    """Eight buffers, in place and not, none of them aligned for the widest words."""
    from asca_amd import _lib, gpu

    rng = np.random.default_rng(6)
    G, K = 3, 4
    par = rng.integers(0, K, G * K).astype(np.int32)
    bpar = gpu.DevBuf.from_array(par)
    host = [rng.integers(0, 256, (i % 3 + 1, G * K, 5 + 31 * i)).astype(np.uint8) for i in range(8)]
    bufs = [gpu.DevBuf.from_array(np.concatenate([np.zeros(i + 1, np.uint8), a.reshape(-1)])) for i, a in enumerate(host)]
    dsts = [gpu.DevBuf(b.nbytes) if i % 2 else None for i, b in enumerate(bufs)]
    n = len(bufs)
    vp = C.c_void_p * n
    num = C.c_uint64 * n
    _lib.call("asca_beam_states", vp(*[b.ptr + i + 1 for i, b in enumerate(bufs)]), vp(*[None if d is None else d.ptr for d in dsts]),
              num(*[a.shape[0] for a in host]), num(*[a.shape[2] for a in host]), n, _p(bpar), G, K, K, None)
    _lib.call("asca_sync")
    for i, a in enumerate(host):
        if dsts[i] is None:
            got = bufs[i].to_host((a.size + i + 1,), np.uint8)
            assert not got[:i + 1].any()
            got = got[i + 1:].reshape(a.shape)
        else:
            got = dsts[i].to_host(a.shape, np.uint8)
        np.testing.assert_array_equal(got, lo.beam_states(a, a, par, G, K, K))


# ------------------------------------------------------------------- together


def _decode_calls(g, rng, G=5, K=4, V=3001, T=9):
    """A teacher's list, a distilled row set, a choice and its states; `run(stream)` makes the calls."""
    from asca_amd import _lib, gpu

    n = G * K
    z, val = logits(rng, n, V, False)
    bz, sc = up(z), up(-rng.random(n).astype(np.float32))
    st0 = rng.standard_normal((2, n, 300)).astype(np.float32)
    o = {k: gpu.DevBuf(4 * s) for k, s in (("v", n * 8), ("i", n * 8), ("s", n), ("loss", n), ("dz", n * V), ("ns", n), ("tok", n), ("par", n),
                                           ("st", st0.size), ("few", 16), ("few_i", 16))}
    src = up(st0)
    one = lambda b: (C.c_void_p * 1)(b.ptr)  # noqa: E731
    keep = [bz, sc, src]

    def run(stream):
        _lib.call("asca_top_logits", _p(bz), V, n, V, 8, 2.0, _p(o["v"]), _p(o["i"]), _p(o["s"]), 0, stream)
        _lib.call("asca_top_logits", _p(bz), V, 2, V, 8, 2.0, _p(o["few"]), _p(o["few_i"]), None, 0, stream)
        _lib.call("asca_distill", _p(bz), V, _p(o["v"]), _p(o["i"]), _p(o["s"]), 8, None, None, 2.0, 1.0, 1.0, _p(o["loss"]), _p(o["dz"]), V,
                  n, V, 0, stream)
        _lib.call("asca_beam_step", _p(bz), V, _p(sc), None, -1, 0, _p(o["ns"]), None, _p(o["tok"]), _p(o["par"]), G, K, V, 0, stream)
        _lib.call("asca_beam_states", one(src), one(o["st"]), (C.c_uint64 * 1)(2), (C.c_uint64 * 1)(1200), 1, _p(o["par"]), G, K, K, stream)

    get = lambda: {k: b.to_host((b.nbytes // 4,)).view(np.uint32) for k, b in o.items()}  # noqa: E731
    return run, get, o, keep, (val, st0, G, K)


def test_a_run_of_them_together(g):
    """What a teacher leaves is what distillation takes: a student of the same logits loses
    nothing; states follow the choice that was made beside it."""
    from asca_amd import _lib

    run, get, o, keep, (val, st0, G, K) = _decode_calls(g, np.random.default_rng(1))
    run(None)
    _lib.call("asca_sync")
    n, V = val.shape
    check_top((o["v"].to_host((n, 8)), o["i"].to_host((n, 8), np.int32), o["s"].to_host((n,))), val, 8, 2.0)
    d = delta(val, 2.0) + 2 * U * 12   # the list's sum is rounded once more
    assert np.abs(o["loss"].to_host((n,))).max() <= 4 * 16 * d
    assert np.abs(o["dz"].to_host((n, V))).max() <= 2 * 4 * d
    par = o["par"].to_host((n,), np.int32)
    np.testing.assert_array_equal(o["st"].to_host(st0.shape), lo.beam_states(st0, st0, par, G, K, K))


def test_on_two_streams_at_once(g):
    from asca_amd import _lib

    sets = [_decode_calls(g, np.random.default_rng(s), G=3 + s) for s in range(2)]
    want = []
    for run, get, *_ in sets:
        run(None)
        _lib.call("asca_sync")
        want.append(get())
    sts = [C.c_void_p() for _ in sets]
    for s in sts:
        _lib.call("asca_stream_create", C.byref(s))
    for _ in range(20):
        for (run, *_), s in zip(sets, sts):
            run(s)
    for s in sts:
        _lib.call("asca_stream_sync", s)
    for (run, get, *_), w in zip(sets, want):
        for k, a in get().items():
            np.testing.assert_array_equal(a, w[k], err_msg=k)
    for s in sts:
        _lib.call("asca_stream_destroy", s)


def test_from_several_host_threads(g):
    import threading

    from asca_amd import _lib

    sets = [_decode_calls(g, np.random.default_rng(50 + s), G=2 + s, V=3001 + 9000 * s) for s in range(4)]
    want = []
    for run, get, *_ in sets:
        run(None)
        _lib.call("asca_sync")
        want.append(get())
    errs = []

    def work(i):
        try:
            s = C.c_void_p()
            _lib.call("asca_stream_create", C.byref(s))
            for _ in range(30):
                sets[i][0](s)
            _lib.call("asca_stream_sync", s)
            _lib.call("asca_stream_destroy", s)
        except BaseException as e:  # noqa: BLE001 (reported below)
            errs.append(repr(e))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
    assert not errs and not any(t.is_alive() for t in ts)
    for (run, get, *_), w in zip(sets, want):
        for k, a in get().items():
            np.testing.assert_array_equal(a, w[k], err_msg=k)


def test_captured_calls_replay_the_eager_results(g):
    """Two graphs on one stream, replayed in turn, with eager calls on it between."""
    from asca_amd import _lib

    hip = C.CDLL("libamdhip64.so.7")

    def ok(rc):
        assert rc == 0, rc

    sets = [_decode_calls(g, np.random.default_rng(20 + s), G=2 + 3 * s, V=3001 + 30000 * s) for s in range(2)]
    want = []
    for run, get, *_ in sets:
        run(None)
        _lib.call("asca_sync")
        want.append(get())
    sp, exes, graphs = C.c_void_p(), [], []
    _lib.call("asca_stream_create", C.byref(sp))
    for run, *_ in sets:
        graph, exe = C.c_void_p(), C.c_void_p()
        ok(hip.hipStreamBeginCapture(sp, 0))
        run(sp)
        ok(hip.hipStreamEndCapture(sp, C.byref(graph)))
        ok(hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)))
        exes.append(exe), graphs.append(graph)
    for k in range(4):
        for i in (0, 1):
            run, get, o, *_ = sets[i]
            for b in o.values():
                _lib.call("asca_memset32", _p(b), 0, b.nbytes // 4, None)
            _lib.call("asca_sync")
            ok(hip.hipGraphLaunch(exes[i], sp))
            _lib.call("asca_stream_sync", sp)
            for name, a in get().items():
                np.testing.assert_array_equal(a, want[i][name], err_msg=f"replay {k} of {i}: {name}")
            sets[1 - i][0](sp)   # the other set eagerly
            _lib.call("asca_stream_sync", sp)
    for exe, graph in zip(exes, graphs):
        ok(hip.hipGraphExecDestroy(exe))
        ok(hip.hipGraphDestroy(graph))
    _lib.call("asca_stream_destroy", sp)


def test_results_do_not_change_from_call_to_call(g):
    from asca_amd import _lib

    run, get, *_ = _decode_calls(g, np.random.default_rng(3), G=40, V=9001)
    run(None)
    _lib.call("asca_sync")
    want = get()
    for _ in range(5):
        run(None)
        _lib.call("asca_sync")
        for k, a in get().items():
            np.testing.assert_array_equal(a, want[k], err_msg=k)
