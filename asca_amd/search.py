"""Beam search over a model's decode steps, with the beams' states on the device
(asca_beam_step and asca_beam_states).

A model gives `_state_bufs(states, n)`: its state buffers as (DevBuf, outer, bytes a
sequence), and `_step_dev(tokens, n, states)`: the device logits (n, vocab) of one
token each, tokens a DevBuf of uint32.
"""
from __future__ import annotations

import numpy as np

from . import _lib
from .gpu import F32, DevBuf, _vp, gpu

MAX_BEAMS = 32   # asca_beam_step


def check(n: int, beams: int, steps: int, eos: int | None, vocab: int) -> None:
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"{beams} beams, 1 to {MAX_BEAMS}")
    if n < 1 or steps < 1:
        raise ValueError(f"{n} sequences, {steps} steps")
    if eos is not None and not 0 <= eos < vocab:
        raise ValueError(f"eos {eos} of {vocab} tokens")


def beam_search(model, logits: DevBuf, states, states_k, n: int, beams: int, steps: int, eos: int | None = None):
    """The `beams` best continuations of n sequences, up to `steps` tokens each, from the
    logits (n, vocab) of their last tokens and `states` of n sequences; `states_k` takes the
    beams' (n * beams sequences).  Returns (tokens, scores): for each sequence its beams best
    first, each an int array that ends with eos where it met it, and (n, beams) summed log
    probabilities (-inf where there were fewer continuations)."""
    V, nk, end = model.vocab, n * beams, -1 if eos is None else int(eos)
    check(n, beams, steps, eos, V)
    dev = gpu()
    bufs: list[DevBuf] = []

    def new(nbytes) -> DevBuf:
        bufs.append(DevBuf(nbytes))
        return bufs[-1]

    try:
        # the sequence's own state and logits for every beam, of which one counts at first
        wide, first = new(nk * V * 4), np.full((n, beams), -np.inf, np.float32)
        first[:, 0] = 0.0
        old, fresh = model._state_bufs(states, n), model._state_bufs(states_k, nk)
        dev.beam_states([(logits, wide, 1, V * 4)] + [(a, b, o, k) for (a, o, k), (b, _, _) in zip(old, fresh, strict=True)], None,
                        groups=n, k=beams, k_src=1, sync=False)
        scores, ended = new(nk * 4), new(nk * 4) if end >= 0 else None
        scores.upload(first.reshape(-1))
        if ended is not None:
            ended.upload(np.zeros(nk, np.int32))
        tokens, parents = new(steps * nk * 4), new(steps * nk * 4)
        row = lambda b, t: _vp(b.ptr + 4 * t * nk)  # noqa: E731
        z, done = wide, steps
        for t in range(steps):
            _lib.call("asca_beam_step", _vp(z), V, _vp(scores), _vp(ended), end, 1, _vp(scores), _vp(ended), row(tokens, t),
                      row(parents, t), n, beams, V, F32, None)
            if t + 1 == steps:
                break
            if ended is not None and t % 8 == 7:   # a look at the flags waits for the device
                _lib.call("asca_sync")
                alive = np.isfinite(scores.to_host((nk,))) & (ended.to_host((nk,), np.int32) == 0)
                if not alive.any():
                    done = t + 1
                    break
            dev.beam_states([(b, None, o, k) for b, o, k in fresh], _View(parents, 4 * t * nk, nk * 4), groups=n, k=beams,
                            sync=False)
            z = model._step_dev(_View(tokens, 4 * t * nk, nk * 4), nk, states_k)
        _lib.call("asca_sync")
        tok, par = tokens.to_host((steps, n, beams), np.uint32)[:done], parents.to_host((steps, n, beams), np.int32)[:done]
        sc = scores.to_host((n, beams))
    finally:
        for b in bufs:
            b.free()
    return _trace(tok, par, sc, end)


def _trace(tok, par, sc, end):
    """Beams best first and their tokens, from every step's tokens and parents."""
    steps, n, beams = tok.shape
    order = np.argsort(-sc, axis=1, kind="stable")
    out = []
    for g in range(n):
        rows = []
        for j in order[g]:
            seq, at = np.empty(steps, np.int64), int(j)
            for t in reversed(range(steps)):
                seq[t], at = tok[t, g, at], int(par[t, g, at])
            stop = np.flatnonzero(seq == end) if end >= 0 else np.empty(0, int)
            rows.append(seq[:stop[0] + 1] if stop.size else seq)
        out.append(rows)
    return out, np.take_along_axis(sc, order, 1)


class _View(DevBuf):
    """A part of another buffer, which owns the memory."""

    __slots__ = ("of",)

    def __init__(self, of: DevBuf, at: int, nbytes: int):
        if at + nbytes > of.nbytes:
            raise ValueError(f"{nbytes} bytes at {at} of {of.nbytes}")
        self.of, self.ptr, self.nbytes = of, of.ptr + at, nbytes

    def free(self) -> None:
        self.ptr = None
