"""The state space byte model (asca_amd/ssm.py) on the GPU: its gradients against
central differences of a float64 forward, its prompts and single rows against its
full-length forward, and the example that trains and decodes with it."""
import sys

import numpy as np
import pytest

from conftest import ROOT
from oracle import ssm_oracle as so

pytestmark = pytest.mark.gpu

FWD, GRAD = 2e-5, 1e-4


def oracle_logits(m, p, ids, batch):
    """The model's logits in float64, from the parameters' values."""
    p = {k: np.asarray(v, np.float64) for k, v in p.items()}
    x = p["embed"][ids]
    x, n = so.block_norm(x, w_pre=p["w_pre.0"][0])
    for i in range(m.L):
        w = lambda k: p[f"{k}.{i}"]  # noqa: E731
        uz = n @ w("w_in")
        c, _ = so.conv(uz[:, :m.d], w("conv_w"), w("conv_b")[0], batch)
        rbc = c @ w("w_x")
        y, _ = so.ssm(c, rbc[:, :m.R] @ w("w_dt"), w("A"), rbc[:, m.R:m.R + m.N], rbc[:, m.R + m.N:], batch, w("dt_bias")[0], w("Dk")[0])
        x, n = so.block_norm(x, y @ w("w_o"), uz[:, m.d:], w("w_post")[0], w("scale")[0], p[f"w_pre.{i + 1}"][0])
    return n @ p["head"]


def oracle_loss(m, p, ids, tgt, batch):
    z = oracle_logits(m, p, ids, batch)
    z = z - z.max(1, keepdims=True)
    return float((np.log(np.exp(z).sum(1)) - z[np.arange(len(tgt)), tgt]).mean())


def model(vocab=17, d=24, n_layers=2, n_state=5, conv_width=4):
    from asca_amd.ssm import SsmModel

    m = SsmModel(vocab, d, n_layers, n_state, conv_width)
    p = m.init(3)
    rng = np.random.default_rng(4)
    for k, a in p.items():   # no parameter at a value that hides its gradient
        p[k] = (a + 0.1 * np.abs(a).mean() * rng.standard_normal(a.shape) + (0.05 if k.startswith("conv_b") else 0)).astype(np.float32)
    m.set_params(p)
    return m, p


def test_gradients_against_differences(g):
    m, p = model()
    rng = np.random.default_rng(5)
    B, T = 3, 21
    ids, tgt = rng.integers(0, 17, B * T), rng.integers(0, 17, B * T)
    loss = m.forward_backward(ids, tgt, B)
    assert abs(loss - oracle_loss(m, p, ids, tgt, B)) <= FWD * loss
    gr = m.grads()
    h = 1e-5
    for k, a in p.items():
        if k == "embed":
            continue
        # along the gradient itself: the difference is its squared norm
        u = gr[k].astype(np.float64)
        u /= np.linalg.norm(u)
        up, dn = (oracle_loss(m, {**p, k: a.astype(np.float64) + s * h * u}, ids, tgt, B) for s in (1, -1))
        want = (up - dn) / (2 * h)
        got = float((gr[k] * u).sum())
        v = rng.standard_normal(a.shape)
        v /= np.linalg.norm(v)
        up, dn = (oracle_loss(m, {**p, k: a.astype(np.float64) + s * h * v}, ids, tgt, B) for s in (1, -1))
        side = abs((up - dn) / (2 * h) - float((gr[k] * v).sum()))
        print(f"[ssm model] {k}: {got:.6e} against {want:.6e}, across {side:.1e}", flush=True)
        assert abs(got - want) <= GRAD * abs(want) + 1e-9
        assert side <= GRAD * abs(want) + 1e-9
    m.close()


def test_prompts_and_rows_give_the_forward(g):
    m, p = model()
    rng = np.random.default_rng(6)
    n, T, more = 4, 19, 5
    ids = rng.integers(0, 17, (n, T + more))
    lens = np.array([19, 1, 7, 18])
    st = m.new_state(n)
    got = m.prompt(ids[:, :T], st, lens)
    want = np.stack([oracle_logits(m, p, ids[b, :lens[b]], 1)[-1] for b in range(n)])
    assert np.abs(got - want).max() <= FWD * np.abs(want).max()
    seqs = [list(ids[b, :lens[b]]) for b in range(n)]
    for k in range(more):
        nxt = ids[:, T + k]
        got = m.step(nxt, st)
        for s, t in zip(seqs, nxt):
            s.append(t)
        want = np.stack([oracle_logits(m, p, np.array(s), 1)[-1] for s in seqs])
        assert np.abs(got - want).max() <= FWD * np.abs(want).max()
    # a second prompt goes on from the states that the rows left
    again = rng.integers(0, 17, (n, 6))
    got = m.prompt(again, st)
    want = np.stack([oracle_logits(m, p, np.concatenate([s, a]), 1)[-1] for s, a in zip(seqs, again)])
    assert np.abs(got - want).max() <= FWD * np.abs(want).max()
    m.close()


def test_clip_bounds_the_norm_of_every_gradient(g):
    m, _ = model()
    rng = np.random.default_rng(7)
    m.forward_backward(rng.integers(0, 17, 40), rng.integers(0, 17, 40), 2)
    before = m.grads()
    want = float(np.sqrt(sum((a.astype(np.float64) ** 2).sum() for k, a in before.items() if k != "embed")))
    norm, c = m.clip(0.5 * want)
    assert abs(norm - want) <= 1e-6 * want and abs(c - 0.5) <= 1e-5
    for k, a in m.grads().items():
        np.testing.assert_allclose(a, before[k] * c, rtol=1e-6, atol=0)
    m.close()


def test_clip_of_the_delta_model_between_backward_and_update(g):
    from asca_amd.model import DeviceModel

    m = DeviceModel(32, 32, 2, 2, 2, 48)
    rng = np.random.default_rng(8)
    p = [(0.1 * rng.standard_normal(a.shape)).astype(np.float32) for a in m.params()]
    m.set_params(p)
    ids, tgt = rng.integers(0, 32, 48), rng.integers(0, 32, 48)
    m.forward_backward(ids, tgt, 2)
    before = m.grads()
    want, c, clipped = so.clip(before, 0.1)
    norm, coef = m.clip_grads(0.1)
    assert c < 1 and abs(norm - want) <= 1e-6 * want and abs(coef - c) <= 1e-6 * c
    for a, b in zip(m.grads(), clipped):
        np.testing.assert_allclose(a, b, rtol=1e-6, atol=1e-30)
    m.adamw()
    assert all(np.isfinite(a).all() for a in m.params())
    m.close()


def test_the_example_learns_and_goes_on(g):
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import ssm_bytes
    finally:
        sys.path.pop(0)
    losses, out = ssm_bytes.main(steps=120)
    assert losses[0] > 4.0 and losses[-1] < 0.2
    whole = ssm_bytes.TEXT * 4
    for o in out:
        assert whole.startswith(o)
