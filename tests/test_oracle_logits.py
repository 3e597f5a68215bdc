"""The float64 definitions behind a model's logits against torch's derivatives, against
differences, and against every continuation counted out."""
import itertools

import numpy as np
import pytest
import torch

from oracle import logits_oracle as lo


def case(rng, T, V, K, rest):
    z = rng.standard_normal((T, V)) * 2
    t = z + rng.standard_normal((T, V))
    ids = np.argsort(-t, axis=1)[:, :K].astype(np.int32)
    return z, np.take_along_axis(t, ids, 1), ids, np.array([lo.lse(r / 2.0) for r in t]) if rest else None, rng.integers(0, V, T)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("alpha", [0.0, 0.3, 1.0])
def test_the_distillation_gradient_is_the_losses_derivative(rest, alpha):
    rng = np.random.default_rng(1)
    z, tv, ids, tl, tg = case(rng, 5, 19, 4, rest)
    ids[1, 2:] = -1          # a shorter list
    ids[2, 1] = ids[2, 0]    # one id twice
    ids[3] = -1              # none
    tg[4] = 19               # no target
    w = rng.uniform(0.5, 2, 5)
    kw = dict(tlse=tl, targets=tg, weights=w, temperature=2.0, alpha=alpha, scale=0.7)
    L, dz, _ = lo.distill(z, tv, ids, **kw)
    h = 1e-6
    for t, i in itertools.product(range(5), range(19)):
        up, dn = z.copy(), z.copy()
        up[t, i] += h
        dn[t, i] -= h
        want = (lo.distill(up, tv, ids, **kw)[0][t] - lo.distill(dn, tv, ids, **kw)[0][t]) / (2 * h) * 0.7
        assert abs(dz[t, i] - want) <= 1e-8 + 1e-6 * abs(want)


def test_against_torch():
    rng = np.random.default_rng(2)
    z, tv, ids, tl, tg = case(rng, 6, 30, 30, True)   # the whole vocabulary is listed: a plain divergence
    x = torch.tensor(z, requires_grad=True)
    t = torch.zeros(6, 30, dtype=torch.float64)
    t.scatter_(1, torch.tensor(ids).long(), torch.tensor(tv))
    F = torch.nn.functional
    kl = F.kl_div(F.log_softmax(x / 2.0, 1), F.softmax(t / 2.0, 1), reduction="none").sum(1)
    loss = 0.4 * F.cross_entropy(x, torch.tensor(tg), reduction="none") + 0.6 * 4.0 * kl
    loss.sum().backward()
    for lse in (None, tl):
        L, dz, _ = lo.distill(z, tv, ids, tlse=lse, targets=tg, temperature=2.0, alpha=0.6)
        np.testing.assert_allclose(L, loss.detach().numpy(), rtol=1e-12)
        np.testing.assert_allclose(dz, x.grad.numpy(), atol=1e-14)


def test_top_takes_the_lower_id_of_equals_and_no_nan():
    z = np.array([[1.0, 3.0, 3.0, -np.inf, 2.0], [np.nan, 0.0, -0.0, np.nan, -np.inf]])
    v, i, _ = lo.top(z, 4)
    np.testing.assert_array_equal(i, [[1, 2, 4, 0], [1, 2, -1, -1]])
    np.testing.assert_array_equal(v, [[3, 3, 2, 1], [0, 0, -np.inf, -np.inf]])


@pytest.mark.parametrize("stay", [False, True])
def test_beams_against_all_continuations(stay):
    """With as many beams as two steps' continuations nothing is lost: the scores are the best
    of all pairs of tokens'."""
    rng = np.random.default_rng(3)
    V, K = 5, 5
    first, second = rng.standard_normal((1, V)), rng.standard_normal((V, V))   # logits after each first token
    z = np.repeat(first, K, 0)
    s, tok, par, _ = lo.beam_step(z, [0.0] + [-np.inf] * (K - 1), K, stay=stay)
    assert sorted(tok) == list(range(V)) and (par == 0).all()
    s2, tok2, par2, _ = lo.beam_step(second[tok], s, K, stay=stay)
    lp = lambda r: r - lo.lse(r)  # noqa: E731
    every = sorted(((lp(first[0])[a] + lp(second[a])[b], a, b) for a in range(V) for b in range(V)), reverse=True)[:K]
    got = sorted(((x, int(tok[p]), int(t)) for x, t, p in zip(s2, tok2, par2)), reverse=True)
    for (x, a, b), (y, c, d) in zip(every, got):
        assert abs(x - y) < 1e-12 and (a, b) == (c, d)
    if stay:   # a beam that has a child keeps one in its slot
        for p in set(par2):
            assert par2[p] == p
    else:
        assert (np.diff(s2) <= 0).all()


def test_an_ended_beam_goes_on_as_itself():
    z = np.zeros((3, 4))
    s, tok, par, end = lo.beam_step(z, [-1.0, -0.5, -np.inf], 3, ended=[1, 0, 0], eos=2)
    assert (s[0], tok[0], par[0], end[0]) == (-1.0, 2, 0, 1)
    np.testing.assert_array_equal(tok[1:], [0, 1])
    np.testing.assert_array_equal(par[1:], [1, 1])
    np.testing.assert_array_equal(end[1:], [0, 0])
