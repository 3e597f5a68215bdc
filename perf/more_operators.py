"""Cases of the operators behind a model's logits: the largest logits of rows, the
distillation of a teacher's largest logits with its gradient, and the steps of a beam
search with the reordering of the states that its sequences carry, each in its plain
form (elementary torch operations), through the library's entry points, and in 64 bits
from its definition.

Formulas (z a row of V logits, tau a temperature, w a row's weight):
  top      the K largest z, descending, ties to the lowest id; lse = log sum exp(z / tau)
  distill  p_k = exp(v_k / tau - tlse) of the listed ids (the rest 1 - sum p is one class
           more), or without tlse the softmax of v / tau over the list; q = softmax(z / tau)
           KL = sum p_k log(p_k / q_k) [+ p_r log(p_r / q_r)]
           loss = w ((1 - a) (log sum exp z - z_target) + a tau^2 KL), dlogits its gradient
           times a scale.  Ids below 0 are no entries.
  beam     the K best of s_b + z_bi - log sum exp z_b over a group's K beams and V tokens,
           ties to the lowest b V + i; an ended beam has one candidate, itself.  `stay`: the
           best child of a beam takes its slot, the others the slots that are left.
  states   slot <- the state of its parent's slot in the same group
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False


def listed():
    return [
        # What a teacher of the byte model's width leaves for one training batch.
        dict(name="top_t16384v256k16", op="top", rows=16384, V=256, K=16, tau=2.0, dtype="f32"),
        # A teacher of a large odd vocabulary: rows that begin at no multiple of 16 bytes.
        dict(name="top_t4096v50001k64", op="top", rows=4096, V=50001, K=64, tau=1.0, dtype="bf16"),
        # The largest logits of one token of one sequence, where latency counts.
        dict(name="top_n1v32768k8", op="top", rows=1, V=32768, K=8, tau=1.0, dtype="f32"),
        # A distilled training step of the byte model: targets and a teacher's top 16 with the rest as a class.
        dict(name="distill_t16384v256k16", op="distill", T=16384, V=256, K=16, tau=2.0, alpha=0.5, rest=True, ragged=False,
             dtype="f32"),
        # The same for a large vocabulary, the teacher's list taken as all there is; the largest case.
        dict(name="distill_t4096v131072k64", op="distill", T=4096, V=131072, K=64, tau=1.0, alpha=1.0, rest=False, ragged=False,
             dtype="bf16"),
        # Odd sizes, lists of different lengths, rows without weight (padding of a batch).
        dict(name="distill_ragged_t1000v32001k20", op="distill", T=1000, V=32001, K=20, tau=4.0, alpha=0.9, rest=True,
             ragged=True, dtype="f32"),
        # A few rows of a large vocabulary (a short sequence): rows alone do not fill the device.
        dict(name="distill_t8v131072k32", op="distill", T=8, V=131072, K=32, tau=1.0, alpha=0.5, rest=True, ragged=False,
             dtype="f32"),
        # A token of one sequence in 4 beams of the byte model, selection and states (8 layers of 8 64 x 64), where
        # latency counts.
        dict(name="search_g1k4v256", op="search", G=1, K=4, V=256, stay=True, ended=False, L=8, state=8 * 64 * 64, dtype="f32"),
        # Selection for 16 sequences in 8 beams of a large odd vocabulary, some of them ended.
        dict(name="beam_g16k8v50001", op="beam", G=16, K=8, V=50001, stay=False, ended=True, dtype="bf16"),
        # Selection for 64 sequences in 4 beams of a large vocabulary.
        dict(name="beam_g64k4v131072", op="beam", G=64, K=4, V=131072, stay=True, ended=False, dtype="f32"),
        # 512 sequences of 16 heads of 128 x 128 in 128 groups, in place: half of the beams survive.
        dict(name="states_g128k4", op="states", G=128, K=4, L=1, state=16 * 128 * 128, distinct=2, inplace=True),
        # States of a 2-layer scan model of odd width that move to other buffers in the beams' new order.
        dict(name="states_g33k5", op="states", G=33, K=5, L=2, state=16 * 999, distinct=3, inplace=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["top", "top", "distill", "distill", "distill", "beam", "beam", "search", "states", "states"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "top":
        while True:
            c = dict(rows=_log(rng, 1, 16384), V=_log(rng, 64, 131072), K=rng.randint(1, 64), tau=rng.choice([1.0, 1.0, 2.0, 4.0]))
            if c["rows"] * c["V"] <= 4096 * 50001:
                return dict(op=op, dtype=dtype, **c)
    if op == "distill":
        while True:
            c = dict(T=_log(rng, 1, 16384), V=_log(rng, 64, 131072), K=rng.randint(1, 64), tau=rng.choice([1.0, 1.0, 2.0, 4.0]),
                     alpha=rng.choice([1.0, 1.0, 0.5, 0.9]), rest=rng.choice([True, False]), ragged=rng.choice([True, False, False]))
            if c["T"] * c["V"] <= 4096 * 131072 // (2 if dtype == "f32" else 1):
                return dict(op=op, dtype=dtype, **c)
    if op in ("beam", "search"):
        while True:
            c = dict(G=_log(rng, 1, 128), K=rng.randint(1, 16), V=_log(rng, 64, 131072), stay=rng.choice([True, False]),
                     ended=rng.choice([True, False]))
            if op == "search":
                c.update(stay=True, L=rng.choice([1, 2, 8]), state=rng.choice([2, 8, 16]) * rng.choice([32, 64, 100, 128]) ** 2)
            if c["G"] * c["K"] * (c["V"] + 2 * c.get("L", 0) * c.get("state", 0)) <= 128 * 4 * 131072:
                return dict(op=op, dtype=dtype, **c)
    while True:
        c = dict(G=_log(rng, 1, 128), K=rng.randint(2, 16), L=rng.choice([1, 2, 8]), state=_log(rng, 1000, 300000))
        if c["G"] * c["K"] * c["L"] * c["state"] <= 128 * 4 * 16 * 128 * 128:
            return dict(op="states", distinct=rng.randint(1, c["K"]), inplace=rng.choice([True, False]), **c)


# ------------------------------------------------------------------- inputs


def _type(case):
    return torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(g, rows, V, ty):
    """Logits of a trained model: a bell around 0 and a few tokens a row that stand out, the
    further the fewer."""
    z = torch.randn(rows, V, generator=g, device="cuda") * 1.5
    few = min(8, V)
    at = torch.randint(0, V, (rows, few), generator=g, device="cuda")
    up = 4.0 + 2.0 * torch.randn(rows, few, generator=g, device="cuda")
    z.scatter_add_(1, at, up)
    return z.to(ty)


def prepare(case, seed):
    g, ty, op = _gen(seed), _type(case), case["op"]
    s = dict(case=case)
    if op == "top":
        s["z"] = _logits(g, case["rows"], case["V"], ty)
    elif op == "distill":
        T, V, K, tau = case["T"], case["V"], case["K"], case["tau"]
        z = s["z"] = _logits(g, T, V, ty)
        # the teacher: the student's logits moved about, its K largest and their whole sum
        tval, tids, tlse = [], [], []
        for a in range(0, T, 1024):
            t = z[a:a + 1024].float()
            t = t + torch.randn(t.shape, generator=g, device="cuda")
            v, i = torch.topk(t, K, 1)
            tval.append(v), tids.append(i.int()), tlse.append(torch.logsumexp(t.double() / tau, 1).float())
        s["tval"], s["tids"] = torch.cat(tval), torch.cat(tids)
        s["tlse"] = torch.cat(tlse) if case["rest"] else None
        s["targets"] = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
        near = torch.rand(T, generator=g, device="cuda") < 0.7   # most targets are what the teacher holds likely
        s["targets"] = torch.where(near, s["tids"][:, 0], s["targets"])
        s["weights"] = None
        if case["ragged"]:
            n = torch.randint(0, K + 1, (T, 1), generator=g, device="cuda")
            s["tids"] = torch.where(torch.arange(K, device="cuda") < n, s["tids"], -1)
            row = torch.arange(T, device="cuda")
            s["weights"] = torch.where(row % 8 == 7, 0.0, 0.5 + torch.rand(T, generator=g, device="cuda"))
            s["targets"] = torch.where(row % 16 == 0, V, s["targets"])   # positions without a target
        s["scale"] = 1.0 / T
    if op in ("beam", "search"):
        G, K, V = case["G"], case["K"], case["V"]
        s["z"] = _logits(g, G * K, V, ty)
        s["scores"] = -5.0 - 3.0 * torch.rand(G * K, generator=g, device="cuda")
        s["eos"] = 1 if case["ended"] else -1
        s["ended"] = (torch.arange(G * K, device="cuda", dtype=torch.int32) % 8 == 3).int() if case["ended"] else None
    if op in ("states", "search"):
        n = case["G"] * case["K"]
        s["state"] = torch.randn(case["L"], n, case["state"], generator=g, device="cuda")
    if op == "states":
        # `distinct` beams of a group survive in their slots, the others' slots take a copy of one of them
        G, K, D = case["G"], case["K"], case["distinct"]
        order = torch.argsort(torch.rand(G, K, generator=g, device="cuda"), 1)
        pick = torch.gather(order, 1, torch.randint(0, D, (G, K), generator=g, device="cuda"))
        par = torch.empty(G, K, dtype=torch.int64, device="cuda")
        keep = torch.arange(K, device="cuda") < D
        par.scatter_(1, order, torch.where(keep, order, pick))
        s["parents"] = par.int().view(-1)
        s["dst"] = None if case["inplace"] else torch.zeros_like(s["state"])
    return s


# ------------------------------------------------------------- plain forms


def _plain_top(s):
    c = s["case"]
    z = s["z"].float()
    v, i = torch.sort(z, dim=1, descending=True, stable=True)
    y = z / c["tau"]
    m = y.amax(1, keepdim=True)
    lse = m[:, 0] + torch.log(torch.exp(y - m).sum(1))
    return dict(values=v[:, :c["K"]].contiguous(), ids=i[:, :c["K"]].int().contiguous(), lse=lse)


def _softmax(y):
    """The softmax of rows, and the logarithm of their sum in 64 bits: a divergence of near
    distributions is a small difference of large logarithms."""
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    t = e.sum(1, keepdim=True, dtype=torch.float64)
    return e / t.float(), m.double() + torch.log(t)


def _plain_distill(s):
    c = s["case"]
    ty, tau, a, V = _type(c), c["tau"], c["alpha"], c["V"]
    z = s["z"].float()
    there = s["tids"] >= 0
    some = there.any(1, keepdim=True)
    ids = torch.where(there, s["tids"], 0).long()
    t = torch.where(there, s["tval"].double() / tau, -torch.inf)
    q, lse = _softmax(z / tau)
    lqk = torch.gather(z, 1, ids).double() / tau - lse
    if s["tlse"] is None:
        p = torch.exp(t - torch.where(some, t.amax(1, keepdim=True), 0.0))
        p = p / torch.where(some, p.sum(1, keepdim=True), 1.0)
    else:
        p = torch.exp(t - s["tlse"].double()[:, None])
    kl = torch.where(p > 0, p * (torch.log(p) - lqk), 0.0).sum(1)
    if s["tlse"] is not None:
        inside = torch.zeros_like(z, dtype=torch.bool)
        row, k = torch.nonzero(there, as_tuple=True)
        inside[row, ids[row, k]] = True
        pr = torch.clamp(1.0 - p.sum(1), min=0.0)
        qr = torch.where(inside, 0.0, q).sum(1, dtype=torch.float64)
        kl = kl + torch.where((pr > 0) & (qr > 0), pr * (torch.log(pr) - torch.log(qr)), 0.0)
        dz = torch.where(inside, q, q * (1.0 - pr / qr).float()[:, None])
    else:
        dz = torch.where(some, q, 0.0)
    del q
    dz.scatter_add_(1, ids, -p.float())
    loss, dz = a * tau * tau * kl, dz * (a * tau)
    if a < 1.0:
        hard, lse = _softmax(z)
        has = s["targets"] < V
        tg = torch.where(has, s["targets"], 0).long()[:, None]
        loss = loss + (1.0 - a) * torch.where(has, (lse - torch.gather(z, 1, tg))[:, 0], 0.0)
        hard.scatter_add_(1, tg, torch.full_like(tg, -1, dtype=torch.float32))
        dz = dz + (1.0 - a) * torch.where(has[:, None], hard, 0.0)
    if s["weights"] is not None:
        loss, dz = loss * s["weights"], dz * s["weights"][:, None]
    return dict(losses=loss.float(), dlogits=(dz * s["scale"]).to(ty))


def _plain_beam(s):
    """Scores in 64 bits: those of different beams can lie next to each other."""
    c = s["case"]
    G, K, V = c["G"], c["K"], c["V"]
    z, sc = s["z"].double(), s["scores"].double()
    m = z.amax(1, keepdim=True)
    cand = sc[:, None] + (z - (m + torch.log(torch.exp(z - m).sum(1, keepdim=True))))
    if s["ended"] is not None:
        e = s["ended"] > 0
        only = torch.full_like(cand, -torch.inf)
        only[:, s["eos"]] = sc
        cand = torch.where(e[:, None], only, cand)
    v, i = torch.sort(cand.view(G, K * V), dim=1, descending=True, stable=True)
    v, i = v[:, :K], i[:, :K]
    parent, token = i // V, i % V
    if c["stay"]:
        slot = torch.full((G, K), -1, dtype=torch.int64, device=z.device)
        taken = torch.zeros(G, K, dtype=torch.bool, device=z.device)
        for r in range(K):   # the best child of a beam stays in its slot
            p = parent[:, r:r + 1]
            free = ~torch.gather(taken, 1, p)
            slot[:, r] = torch.where(free, p, -1)[:, 0]
            taken.scatter_(1, p, True)
        for r in range(K):   # the others take the first that are left
            first = torch.argmax((~taken).int(), 1, keepdim=True)
            need = slot[:, r:r + 1] < 0
            slot[:, r] = torch.where(need, first, slot[:, r:r + 1])[:, 0]
            taken.scatter_(1, first, torch.gather(taken, 1, first) | need)
        back = torch.argsort(slot, 1)
        v, parent, token = (torch.gather(x, 1, back) for x in (v, parent, token))
    out = dict(scores=v.reshape(-1).float(), tokens=token.reshape(-1).int(), parents=parent.reshape(-1).int())
    if s["ended"] is not None:
        before = torch.gather(e.view(G, K), 1, parent).reshape(-1)
        out["ended"] = (before | (out["tokens"] == s["eos"])).int()
    return out


def _plain_states(s, parents, dst):
    c = s["case"]
    G, K = c["G"], c["K"]
    row = torch.arange(G, device=parents.device)[:, None] * K + parents.view(G, K)
    moved = torch.index_select(s["state"], 1, row.view(-1))
    dst.copy_(moved)
    return dst


# -------------------------------------------------------- the library's calls


def _ptr(t):
    return None if t is None else t.data_ptr()


def _calls(s):
    """The calls of one pass with their arguments and the outputs that they write, made on a
    state's first pass and kept with it, as a program keeps its buffers."""
    from asca_amd.gpu import gpu

    if gpu() is None:
        raise RuntimeError("no GPU backend")
    c, p = s["case"], _ptr
    op, ty = c["op"], 1 if c.get("dtype") == "bf16" else 0
    f32 = lambda *n: torch.empty(*n, device="cuda")  # noqa: E731
    i32 = lambda *n: torch.empty(*n, device="cuda", dtype=torch.int32)  # noqa: E731
    calls, out = [], {}
    if op == "top":
        rows, V, K = c["rows"], c["V"], c["K"]
        out.update(values=f32(rows, K), ids=i32(rows, K), lse=f32(rows))
        calls.append(("asca_top_logits", (p(s["z"]), V, rows, V, K, c["tau"], p(out["values"]), p(out["ids"]), p(out["lse"]), ty,
                                          None)))
    elif op == "distill":
        T, V, K = c["T"], c["V"], c["K"]
        out.update(losses=f32(T), dlogits=torch.empty_like(s["z"]))
        calls.append(("asca_distill", (p(s["z"]), V, p(s["tval"]), p(s["tids"]), p(s["tlse"]), K, p(s["targets"]),
                                       p(s["weights"]), c["tau"], c["alpha"], s["scale"], p(out["losses"]), p(out["dlogits"]), V, T,
                                       V, ty, None)))
    if op in ("beam", "search"):
        G, K, V = c["G"], c["K"], c["V"]
        out.update(scores=f32(G * K), tokens=i32(G * K), parents=i32(G * K))
        if s["ended"] is not None:
            out["ended"] = i32(G * K)
        calls.append(("asca_beam_step", (p(s["z"]), V, p(s["scores"]), p(s["ended"]), s["eos"], int(c["stay"]), p(out["scores"]),
                                         p(out.get("ended")), p(out["tokens"]), p(out["parents"]), G, K, V, ty, None)))
    if op in ("states", "search"):
        dst = s.get("dst")
        out["state"] = s["state"] if dst is None else dst
        one = lambda t: None if t is None else (ctypes.c_void_p * 1)(t.data_ptr())  # noqa: E731
        n64 = lambda n: (ctypes.c_uint64 * 1)(n)  # noqa: E731
        calls.append(("asca_beam_states", (one(s["state"]), one(dst), n64(c["L"]), n64(4 * c["state"]), 1,
                                           p(out["parents"] if op == "search" else s["parents"]), c["G"], c["K"], c["K"], None)))
    return calls, out


def run(state):
    if own:
        from asca_amd import _lib

        if "calls" not in state:
            state["calls"] = _calls(state)
        calls, out = state["calls"]
        for name, args in calls:
            _lib.call(name, *args)
        return dict(out)
    op = state["case"]["op"]
    if op == "top":
        return _plain_top(state)
    if op == "distill":
        return _plain_distill(state)
    if op == "states":
        dst = state["dst"] if state["dst"] is not None else state["state"]
        return dict(state=_plain_states(state, state["parents"], dst))
    out = _plain_beam(state)
    if op == "search":
        out["state"] = _plain_states(state, out["parents"], state["state"])
    return out


# ------------------------------------------------------------------- work


def _moved(K, distinct):
    """States read and written in a group whose survivors stay: a read of each that is copied, a write of each copy."""
    return min(distinct, K - distinct) + K - distinct


def work(case):
    op, e = case["op"], 2 if case.get("dtype") == "bf16" else 4
    if op == "top":
        n = case["rows"] * case["V"]
        return dict(bytes=e * n + case["rows"] * (8 * case["K"] + 4), flops=5 * n)
    if op == "distill":
        T, n, hard = case["T"], case["T"] * case["V"], case["alpha"] < 1.0
        read = T - T // 8 if case["ragged"] else T   # rows without weight are not read
        return dict(bytes=e * case["V"] * (read + T) + 8 * T * case["K"] + 4 * T * (1 + case["rest"] + hard + case["ragged"]),
                    flops=n * (12 if hard and case["tau"] != 1.0 else 7))
    if op == "states":
        G, K = case["G"], case["K"]
        if case["inplace"]:
            moved = _moved(K, case["distinct"])
        else:
            moved = case["distinct"] + K
        return dict(bytes=4 * case["L"] * case["state"] * G * moved, flops=0)
    G, K, V = case["G"], case["K"], case["V"]
    rows = G * K - ((G * K + 4) // 8 if case["ended"] else 0)   # an ended beam's logits are not read
    w = dict(bytes=e * rows * V + 24 * G * K, flops=4 * rows * V)
    if op == "search" and K > 1:
        # as many survivors as when the K best fell on the beams evenly
        distinct = max(1, int(K * (1.0 - (1.0 - 1.0 / K) ** K)))
        w["bytes"] += 4 * case["L"] * case["state"] * G * _moved(K, distinct)
    return w


# ------------------------------------------------------------ 64-bit values


def _largest(x, K):
    """The K largest of each row, one after another, the lowest place first among equals."""
    x, place = x.clone(), torch.arange(x.shape[1], device=x.device)
    v, i = [], []
    for _ in range(K):
        top = x.max(1, keepdim=True).values
        at = torch.where(x == top, place, x.shape[1]).min(1, keepdim=True).values
        v.append(top), i.append(at)
        x.scatter_(1, at, -torch.inf)
    return torch.cat(v, 1), torch.cat(i, 1)


def _exact_top(s):
    c = s["case"]
    v, i, lse = [], [], []
    for a in range(0, c["rows"], 512):
        z = s["z"][a:a + 512].double()
        x, y = _largest(z, c["K"])
        v.append(x), i.append(y), lse.append(torch.logsumexp(z / c["tau"], 1))
    return dict(values=torch.cat(v), ids=torch.cat(i).int(), lse=torch.cat(lse))


def _exact_distill(s):
    c = s["case"]
    T, V, K, tau, a = (c[k] for k in ("T", "V", "K", "tau", "alpha"))
    losses, grads = torch.zeros(T, dtype=torch.float64, device="cuda"), torch.empty(T, V, dtype=torch.float64, device="cuda")
    for r in range(0, T, 256):
        z = s["z"][r:r + 256].double()
        n = z.shape[0]
        ids, tv = s["tids"][r:r + 256].long(), s["tval"][r:r + 256].double() / tau
        # the teacher as a row over the vocabulary; column V takes what is no entry
        col = torch.where(ids < 0, V, ids)
        listed = torch.zeros(n, V + 1, dtype=torch.float64, device="cuda").scatter_(1, col, 1.0)[:, :V] > 0
        weight = torch.exp(tv - (tv.max(1, keepdim=True).values if s["tlse"] is None else s["tlse"][r:r + 256].double()[:, None]))
        p = torch.zeros(n, V + 1, dtype=torch.float64, device="cuda").scatter_add_(1, col, weight)[:, :V]
        some = listed.any(1)
        if s["tlse"] is None:
            p = p / torch.where(some, p.sum(1), 1.0)[:, None]
        lz = torch.logsumexp(z / tau, 1, keepdim=True)
        q = torch.exp(z / tau - lz)
        soft = torch.xlogy(p, p).sum(1) - torch.where(p > 0, p * (z / tau - lz), 0.0).sum(1)
        if s["tlse"] is not None:
            rest = torch.clamp(1.0 - p.sum(1), min=0.0)
            lqr = torch.logsumexp(torch.where(listed, -torch.inf, z / tau), 1) - lz[:, 0]
            live = (rest > 0) & torch.isfinite(lqr)
            soft = soft + torch.where(live, torch.xlogy(rest, rest) - rest * lqr, 0.0)
            mass = p.sum(1) + torch.where(live, rest, 0.0)   # d/dz of minus sum p log q, the rest's among them
            inner = torch.where(live, rest, 0.0) * torch.exp(-lqr)
            g = q * mass[:, None] - p - torch.where(listed, 0.0, q) * torch.where(live, inner, 0.0)[:, None]
        else:
            g = torch.where(some[:, None], q, 0.0) - p
        loss, g = a * tau ** 2 * soft, a * tau * g
        if a < 1.0:
            tg = s["targets"][r:r + 256].long()
            has = tg < V
            hot = torch.zeros(n, V + 1, dtype=torch.float64, device="cuda").scatter_(1, tg[:, None], 1.0)[:, :V]
            l1 = torch.logsumexp(z, 1, keepdim=True)
            loss = loss + (1 - a) * torch.where(has, l1[:, 0] - (z * hot).sum(1), 0.0)
            g = g + (1 - a) * torch.where(has[:, None], torch.exp(z - l1) - hot, 0.0)
        if s["weights"] is not None:
            w = s["weights"][r:r + 256].double()
            loss, g = loss * w, g * w[:, None]
        losses[r:r + 256], grads[r:r + 256] = loss, g * s["scale"]
    return dict(losses=losses, dlogits=grads)


def _exact_beam(s):
    c = s["case"]
    G, K, V = c["G"], c["K"], c["V"]
    out = dict(scores=torch.empty(G, K, dtype=torch.float64, device="cuda"))
    for k in ("tokens", "parents") + (("ended",) if s["ended"] is not None else ()):
        out[k] = torch.empty(G, K, dtype=torch.int32, device="cuda")
    done = torch.zeros(G, K, dtype=torch.bool, device="cuda") if s["ended"] is None else s["ended"].view(G, K) > 0
    for b in range(G):
        z = s["z"][b * K:(b + 1) * K].double()
        sc = s["scores"][b * K:(b + 1) * K].double()
        cand = sc[:, None] + z - torch.logsumexp(z, 1, keepdim=True)
        for k in torch.nonzero(done[b])[:, 0].tolist():
            cand[k] = -torch.inf
            cand[k, s["eos"]] = sc[k]
        v, i = _largest(cand.view(1, -1), K)
        par, tok = (i[0] // V).tolist(), (i[0] % V).tolist()
        if c["stay"]:
            where, left = {}, list(range(K))
            for r, q in enumerate(par):
                if q in left:
                    where[r] = q
                    left.remove(q)
            for r in range(K):
                if r not in where:
                    where[r] = left.pop(0)
        else:
            where = {r: r for r in range(K)}
        for r in range(K):
            j = where[r]
            out["scores"][b, j], out["tokens"][b, j], out["parents"][b, j] = v[0, r], tok[r], par[r]
            if s["ended"] is not None:
                out["ended"][b, j] = int(bool(done[b, par[r]]) or tok[r] == s["eos"])
    return {k: x.view(-1) for k, x in out.items()}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "top":
        return _exact_top(s)
    if op == "distill":
        return _exact_distill(s)
    out = _exact_beam(s) if op in ("beam", "search") else {}
    if op in ("states", "search"):
        par = (s["parents"] if op == "states" else out["parents"]).tolist()
        K = case["K"]
        old = s["state"].double()
        out["state"] = torch.stack([old[:, j // K * K + q] for j, q in enumerate(par)], 1)
    return out
