"""The models' use of the operators behind the logits: distilled training steps against
differences and against the cross-entropy that they are made of, beam searches against the
same search on the host over the models' own logits, and the example."""
import sys

import numpy as np
import pytest

from conftest import ROOT
from oracle import logits_oracle as lo
from test_gpu_ssm_model import GRAD, model, oracle_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rest,alpha", [(True, 0.6), (False, 1.0)])
def test_distilled_gradients_against_differences(g, rest, alpha):
    m, p = model()
    big, bp = model(vocab=17, d=32, n_layers=1, n_state=3)
    rng = np.random.default_rng(5)
    B, T, K, tau = 3, 21, 6, 2.0
    ids, tgt = rng.integers(0, 17, B * T), rng.integers(0, 17, B * T)
    w = rng.uniform(0.5, 1.5, B * T).astype(np.float32)
    t = big.teacher(ids, B, K, tau, rest)
    tv, ti, tl = t.to_host()
    tz = oracle_logits(big, bp, ids, B)
    want = lo.top(tz, K, tau)
    assert np.abs(tv - want[0]).max() <= 2e-5 * np.abs(tz).max()   # the teacher is f32
    np.testing.assert_array_equal(ti, want[1])
    assert (tl is None) != rest

    def loss_of(q):
        return lo.distill(oracle_logits(m, q, ids, B), tv, ti, tlse=tl, targets=tgt, weights=w, temperature=tau, alpha=alpha)[0].mean()

    loss = m.forward_backward(ids, tgt if alpha < 1 else None, B, t, alpha=alpha, weights=w)
    assert abs(loss - loss_of(p)) <= 1e-4 * abs(loss)
    gr, h = m.grads(), 1e-5
    for k, a in p.items():
        if k == "embed":
            continue
        u = gr[k].astype(np.float64)
        u /= np.linalg.norm(u)
        up, dn = (loss_of({**p, k: a.astype(np.float64) + s * h * u}) for s in (1, -1))
        want, got = (up - dn) / (2 * h), float((gr[k] * u).sum())
        assert abs(got - want) <= GRAD * abs(want) + 1e-9, k
    t.free()
    m.close()
    big.close()


def test_a_teacher_sure_of_one_id_is_a_target(g):
    """Distillation from a list of one id at temperature 1 is the cross-entropy of that id, and
    a mixture's gradients are the mixture's, in both models."""
    from asca_amd.gpu import Teacher
    from asca_amd.model import DeviceModel

    rng = np.random.default_rng(8)
    d = DeviceModel(32, 32, 2, 2, 2, 48)
    d.set_params([(0.1 * rng.standard_normal(a.shape)).astype(np.float32) for a in d.params()])
    s, _ = model(vocab=32)
    n = 48
    ids, one, two = (rng.integers(0, 32, n) for _ in range(3))
    t = Teacher.upload(rng.standard_normal((n, 1)), one[:, None])

    def grads(m):
        gr = m.grads()
        return list(gr.values()) if isinstance(gr, dict) else gr

    for m in (d, s):
        distill = m.distill if m is d else lambda i, g_, b, t_, **k: s.forward_backward(i, g_, b, t_, **k)
        l1 = m.forward_backward(ids, one, 2)
        g1 = grads(m)
        l2 = m.forward_backward(ids, two, 2)
        g2 = grads(m)
        got = distill(ids, None, 2, t, alpha=1.0)
        ga = grads(m)
        mix = distill(ids, two, 2, t, alpha=0.25)
        gm = grads(m)
        hard = distill(ids, two, 2, t, alpha=0.0)
        gh = grads(m)
        assert abs(got - l1) <= 1e-5 * l1 and abs(mix - (0.25 * l1 + 0.75 * l2)) <= 1e-5 * l1 and abs(hard - l2) <= 1e-5 * l2
        for a, b, c, x, y in zip(g1, g2, ga, gm, gh):
            big = max(np.abs(a).max(), np.abs(b).max())
            assert np.abs(c - a).max() <= GRAD * big and np.abs(y - b).max() <= GRAD * big
            assert np.abs(x - (0.25 * a + 0.75 * b)).max() <= GRAD * big
    w = np.where(np.arange(n) < n // 2, 2.0, 0.0)   # the first sequence alone
    full = d.distill(ids, two, 2, t, alpha=0.25, weights=w)
    half = d.distill(ids[:n // 2], two[:n // 2], 1, Teacher.upload(np.zeros((n // 2, 1)), one[:n // 2, None]), alpha=0.25)
    assert abs(full - half) <= 1e-5 * half
    d.close()
    s.close()


def host_search(step, logits, beams, steps, eos, pick):
    """The same search on the host: `step(tokens)` gives the beams' next logits, `pick(parents)`
    moves their states."""
    n, V = logits.shape
    sc = np.where(np.arange(n * beams) % beams == 0, 0.0, -np.inf)
    z, end = np.repeat(logits, beams, 0), np.zeros(n * beams, np.int32)
    seqs = [[] for _ in range(n * beams)]
    for t in range(steps):
        sc, tok, par, new = lo.beam_step(z, sc, beams, end if eos is not None else None, -1 if eos is None else eos)
        sc = sc.astype(np.float32)
        rows = np.arange(n * beams) // beams * beams + par
        seqs = [seqs[r] + [int(x)] for r, x in zip(rows, tok)]
        if eos is not None:
            end = new
        if t + 1 < steps:
            pick(rows)
            z = step(tok)
    cut = lambda s: s[:s.index(eos) + 1] if eos in s else s  # noqa: E731
    return [[cut(s) for s in seqs[g * beams:(g + 1) * beams]] for g in range(n)], sc.reshape(n, beams)


@pytest.mark.parametrize("eos", [None, 3])
@pytest.mark.parametrize("beams,steps", [(1, 5), (3, 7), (5, 20), (17, 3)])
def test_searches_against_the_host(g, beams, steps, eos):
    """Sequences and scores of both models, prompts of different lengths where they can be."""
    from asca_amd.model import DeviceModel

    rng = np.random.default_rng(beams)
    n = 3
    ids = rng.integers(0, 17, (n, 9))
    m, p = model()
    lens = np.array([9, 1, 4])
    got, sc = m.beam_search(ids, beams, steps, lens, eos)
    hist = [[list(ids[b, :lens[b]]) for b in range(n)]]
    first = np.stack([oracle_logits(m, p, np.array(s), 1)[-1] for s in hist[0]])
    hist[0] = [list(s) for s in hist[0] for _ in range(beams)]

    def pick(rows):
        hist[0] = [list(hist[0][r]) for r in rows]

    def step(tok):
        for s, x in zip(hist[0], tok):
            s.append(int(x))
        return np.stack([oracle_logits(m, p, np.array(s), 1)[-1] for s in hist[0]])

    want, ws = host_search(step, first, beams, steps, eos, pick)
    fin = np.isfinite(ws)
    np.testing.assert_array_equal(fin, np.isfinite(sc))
    assert np.abs(sc[fin] - ws[fin]).max() <= 1e-4 * np.abs(ws[fin]).max()
    for a, b, ok in zip(got, want, fin):
        for x, y, f in zip(a, b, ok):
            assert not f or list(x) == y
    m.close()

    d = DeviceModel(17, 32, 2, 2, 2, 48)
    d.set_params([(0.3 * rng.standard_normal(a.shape)).astype(np.float32) for a in d.params()])
    got, sc = d.beam_search(ids, beams, steps, eos)
    one = d.new_decode_state(n)
    for t in range(9):
        first = d.step(ids[:, t], one)
    shape = (2, n, d.decode_state_floats() // 2)
    st = [np.repeat(one.to_host(shape), beams, 1)]
    buf = d.new_decode_state(n * beams)

    def dpick(rows):
        st[0] = st[0][:, rows]

    def dstep(tok):
        buf.upload(st[0])
        z = d.step(tok, buf)
        st[0] = buf.to_host(st[0].shape)
        return z

    want, ws = host_search(dstep, first, beams, steps, eos, dpick)
    fin = np.isfinite(ws)
    assert np.abs(sc[fin] - ws[fin]).max() <= 1e-5 * np.abs(ws[fin]).max()
    for a, b, ok in zip(got, want, fin):
        for x, y, f in zip(a, b, ok):
            assert not f or list(x) == y
    one.free()
    buf.free()
    d.close()


def test_a_search_in_which_every_beam_ends(g):
    """The search stops where all have ended; a beam that has is not touched again."""
    m, p = model()
    p = dict(p)
    p["head"] = p["head"].copy()
    p["head"][:, 3] *= 30          # eos stands out, whichever way the row points
    m.set_params(p)
    got, sc = m.beam_search(np.random.default_rng(0).integers(0, 17, (4, 6)), 2, 60, eos=3)
    for rows, s in zip(got, sc):
        for r, x in zip(rows, s):
            assert 3 not in r[:-1]
    m.close()


def test_a_search_stops_where_every_beam_has_ended(g, monkeypatch):
    """eos is the likeliest token of every row (channel 0, which every embedding has most of, gives it
    alone): all beams end, each counted step after that is left out, and tokens and scores are the
    host's and those of a longer search."""
    m, p = model()
    p = {k: a.copy() for k, a in p.items()}
    p["embed"][:, 0] = 8.0
    p["head"][0] = 0.0
    p["head"][0, 3] = 0.7
    m.set_params(p)
    rng = np.random.default_rng(6)
    n, beams, steps = 4, 3, 30
    ids = rng.integers(0, 17, (n, 5))
    calls = []
    step_dev = m._step_dev
    monkeypatch.setattr(m, "_step_dev", lambda *a: calls.append(1) or step_dev(*a))
    got, sc = m.beam_search(ids, beams, steps, eos=3)
    hist = [[list(s) for s in ids for _ in range(beams)]]

    def pick(rows):
        hist[0] = [list(hist[0][r]) for r in rows]

    def step(tok):
        for s, x in zip(hist[0], tok):
            s.append(int(x))
        return np.stack([oracle_logits(m, p, np.array(s), 1)[-1] for s in hist[0]])

    first = np.stack([oracle_logits(m, p, np.array(s), 1)[-1] for s in ids])
    assert (first.argmax(1) == 3).all()
    want, ws = host_search(step, first, beams, steps, 3, pick)
    assert all(r[-1] == 3 and 3 not in r[:-1] for rows in want for r in rows)
    ended = max(len(r) for rows in want for r in rows)     # steps after which all have
    assert 1 < ended <= 16
    assert len(calls) == (7 if ended <= 8 else 15)         # looked at every 8 steps
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert list(x) == y
    assert np.abs(sc - ws).max() <= 1e-4 * np.abs(ws).max()
    more, msc = m.beam_search(ids, beams, 2 * steps, eos=3)
    np.testing.assert_array_equal(sc, msc)
    assert all(list(x) == list(y) for a, b in zip(got, more) for x, y in zip(a, b))
    m.close()


def test_the_example_runs(g):
    sys.path.insert(0, str(ROOT))
    try:
        from examples import distill_bytes
    finally:
        sys.path.pop(0)
    losses, out = distill_bytes.main(steps=20)
    assert len(losses) == 20 and np.isfinite(losses).all() and len(out) == 2
