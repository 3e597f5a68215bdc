"""Plain float64 definitions of the operators behind a model's logits (largest logits,
distillation from a teacher's largest, a beam search's choice and its states' move),
row after row.  Test infrastructure: nothing in asca_amd/ imports it.  Arguments as in
include/asca_hip.h.
"""
from __future__ import annotations

import numpy as np

f8 = np.float64


def lse(v):
    """log sum exp of a vector; -inf of none."""
    m = v.max(initial=-np.inf)
    return m if not np.isfinite(m) else m + np.log(np.exp(v - m).sum())


def top(logits, K, temperature=1.0):
    """(values, ids, lse)."""
    z = np.asarray(logits, f8)
    v, i = np.full((len(z), K), -np.inf), np.full((len(z), K), -1, np.int32)
    for r, row in enumerate(z):
        at = [c for c in np.lexsort((np.arange(len(row)), -row)) if row[c] > -np.inf][:K]   # NaN compares false
        i[r, :len(at)] = at
        v[r, :len(at)] = row[at]
    return v, i, np.array([lse(row / temperature) for row in z])


def distill(logits, tval=None, tids=None, tlse=None, targets=None, weights=None, temperature=1.0, alpha=1.0, scale=1.0):
    """(losses, dlogits, terms): terms are the sizes of what is added up in each loss and
    in each gradient, for a bound on rounding: (of the losses, of the gradients)."""
    z = np.asarray(logits, f8)
    T, V = z.shape
    L, dz, tl, tg = np.zeros(T), np.zeros((T, V)), np.zeros(T), np.zeros((T, V))
    for t in range(T):
        w = 1.0 if weights is None else float(weights[t])
        if w == 0:
            continue
        soft, g, sl, sg = 0.0, np.zeros(V), 0.0, np.zeros(V)
        if alpha > 0:
            p, lists = {}, [(int(i), float(v)) for i, v in zip(tids[t], tval[t]) if 0 <= i < V]
            at = np.array([v for _, v in lists]) / temperature
            norm = float(tlse[t]) if tlse is not None else lse(at)
            for (i, _), v in zip(lists, at):
                p[i] = p.get(i, 0.0) + (np.exp(v - norm) if norm > -np.inf else 0.0)
            lq = z[t] / temperature - lse(z[t] / temperature)
            q = np.exp(lq)
            mass = sum(p.values())
            for i, pi in p.items():
                if pi > 0:
                    soft += pi * (np.log(pi) - lq[i])
                    sl += pi * (1 + abs(np.log(pi)) + abs(lq[i]) + abs(z[t, i]) / temperature)
            inside = np.zeros(V, bool)
            inside[list(p)] = True
            rest = max(0.0, 1.0 - mass) if tlse is not None else 0.0
            lqr = lse(lq[~inside])
            meets = rest > 0 and lqr > -np.inf
            if meets:
                soft += rest * (np.log(rest) - lqr)
                sl += rest * (1 + abs(np.log(rest)) + abs(lqr)) + abs(np.log(rest) - lqr) + 1
                mass += rest
            g += mass * q
            for i, pi in p.items():
                g[i] -= pi
                sg[i] += pi
            if meets:
                share = np.where(inside, 0.0, np.exp(lq - lqr))
                g -= rest * share
                sg += (rest + 1) * share
            soft *= alpha * temperature ** 2
            g *= alpha * temperature
            sl *= alpha * temperature ** 2
            sg = (sg + (1 + mass) * q) * alpha * temperature
        if alpha < 1 and 0 <= int(targets[t]) < V:
            lp = z[t] - lse(z[t])
            soft += (1 - alpha) * -lp[int(targets[t])]
            h = np.exp(lp)
            sl += (1 - alpha) * (1 + abs(lse(z[t])) + abs(z[t, int(targets[t])]))
            sg += (1 - alpha) * h
            h[int(targets[t])] -= 1
            g += (1 - alpha) * h
            sg[int(targets[t])] += 1 - alpha
        L[t], dz[t], tl[t], tg[t] = w * soft, scale * w * g, abs(w) * sl, abs(scale * w) * sg
    return L, dz, (tl, tg)


def beam_step(logits, scores, K, ended=None, eos=-1, stay=False):
    """(scores, tokens, parents, ended or None) of groups of K beams.  Candidates of one score
    come by their beams, and of one beam by their logits, then by their ids."""
    z, s = np.asarray(logits, f8), np.asarray(scores, f8)
    n, V = z.shape
    ns, tok, par = np.full(n, -np.inf), np.full(n, max(eos, 0), np.uint32), np.zeros(n, np.int32)
    end = np.zeros(n, np.int32)
    for g in range(n // K):
        cand = []   # (-score, beam, -logit, id)
        for b in range(K):
            r = g * K + b
            if not np.isfinite(s[r]):
                continue
            if ended is not None and ended[r]:
                cand.append((-s[r], b, 0.0, eos))
                continue
            norm = lse(z[r]) if not np.isnan(z[r]).any() else np.nan
            if not np.isfinite(norm):
                continue
            x = s[r] + (z[r] - norm)
            keep = np.argsort(-z[r], kind="stable")[:K]   # no more of one beam can be chosen
            cand += [(-x[c], b, -z[r, c], int(c)) for c in keep if z[r, c] > -np.inf]
        cand = sorted(cand)[:K]
        picks = [(-x, b, c) for x, b, _, c in cand] + [None] * (K - len(cand))
        slots, left = {}, list(range(K))
        if stay:
            for r, c in enumerate(picks):
                if c is not None and c[1] in left:
                    slots[r] = c[1]
                    left.remove(c[1])
        for r in range(K):
            if r not in slots:
                slots[r] = left.pop(0)
        for r, c in enumerate(picks):
            j = g * K + slots[r]
            if c is None:
                par[j] = slots[r]
                continue
            ns[j], par[j], tok[j] = c
            end[j] = int(c[2] == eos or (ended is not None and ended[g * K + c[1]] != 0))
    return ns, tok, par, None if ended is None else end


def beam_states(src, dst, parents, groups, k_src, k_dst):
    """src (outer, groups*k_src, ...) into dst (outer, groups*k_dst, ...)."""
    out = dst.copy()
    for g in range(groups):
        for j in range(k_dst):
            q = 0 if parents is None else int(parents[g * k_dst + j])
            if 0 <= q < k_src:
                out[:, g * k_dst + j] = src[:, g * k_src + q]
    return out
