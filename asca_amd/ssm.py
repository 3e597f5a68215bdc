"""A device-resident byte model of selective state space blocks, over the state
space block's entry points of include/asca_hip.h and asca_gemm.

A layer, with x the residual stream (rows of d) and nrm its normalised rows:
  u | z = nrm w_in;  c = conv(u);  r | B | C = c w_x;  dt = r w_dt
  o = scan(c, dt, A, B, C) w_o
  x' = x + scale o (rms(o o silu(z)) o w_post);  nrm' = rms(x') o w_pre'
The residual's update and both norms are one call (asca_block_norm_fwd); u, z and
r, B, C are columns of one product each.  Everything is f32, B and C are one group.
The embedding stays as it is set: no gradient of it is formed (unlike DeviceModel's).

It trains (forward_backward, clip, adamw), reads prompts of different lengths
(prompt) and decodes one row for many sequences on their states (step), like
DeviceModel does for the delta block.  It learns from a teacher's largest logits and
leaves its own for a student (forward_backward, teacher), and searches over beams
(beam_search).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib, search
from .gpu import F32, DevBuf, GradList, Teacher, _vp, describe, gpu

_f32 = np.float32
EPS = 1e-6


class SsmModel:
    def __init__(self, vocab: int, d: int, n_layers: int, n_state: int = 16, conv_width: int = 4, dt_rank: int | None = None):
        if gpu() is None:  # lazy device initialisation, as DeviceModel
            raise RuntimeError(describe())
        self.vocab, self.d, self.L, self.N, self.W = vocab, d, n_layers, n_state, conv_width
        self.R = dt_rank or -(-d // 16)
        self.X = self.R + 2 * n_state
        layer = [("w_in", d, 2 * d), ("conv_w", conv_width, d), ("conv_b", 1, d), ("w_x", d, self.X), ("w_dt", self.R, d),
                 ("dt_bias", 1, d), ("A", n_state, d), ("Dk", 1, d), ("w_o", d, d), ("w_post", 1, d), ("scale", 1, d)]
        shapes = [("embed", vocab, d), ("head", d, vocab)] + [(f"{k}.{i}", r, c) for i in range(n_layers) for k, r, c in layer]
        shapes += [(f"w_pre.{i}", 1, d) for i in range(n_layers + 1)]
        self.tensors, at = [], 0
        for name, r, c in shapes:
            self.tensors.append((name, at, r, c))
            at += -(-r * c // 4) * 4   # every tensor 16-byte aligned
        self._at = {name: off for name, off, _, _ in self.tensors}
        self.n_floats = at
        self._flat = {k: DevBuf(at * 4) for k in ("params", "grads", "m", "v")}
        for b in self._flat.values():
            _lib.call("asca_memset32", _vp(b), 0, at, None)
        # the embedding is a fixed table: its gradient is not formed
        self._clip = GradList([(self._flat["grads"].ptr + 4 * o, r * c) for n, o, r, c in self.tensors if n != "embed"], dtype=F32)
        self._step = 0
        self._bufs: dict = {}

    # -- parameters --------------------------------------------------------------
    def init(self, seed: int = 0) -> dict:
        """Initial parameters as {name: array}: steps of 0.001 to 0.1, A = -1 .. -N."""
        rng, p = np.random.default_rng(seed), {}
        for name, _, r, c in self.tensors:
            k = name.split(".")[0]
            if k in ("w_post", "w_pre", "Dk"):
                a = np.ones((r, c))
            elif k == "scale":
                a = np.full((r, c), 0.5)
            elif k == "A":
                a = -np.repeat(np.arange(1, r + 1.0)[:, None], c, 1)
            elif k == "dt_bias":
                a = np.log(np.expm1(np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), (r, c)))))
            elif k == "conv_b":
                a = np.zeros((r, c))
            else:
                a = rng.standard_normal((r, c)) / np.sqrt(1 if k == "embed" else r)
            p[name] = a.astype(_f32)
        return p

    def set_params(self, p: dict) -> None:
        flat = np.zeros(self.n_floats, _f32)
        for name, off, r, c in self.tensors:
            flat[off:off + r * c] = np.asarray(p[name], _f32).reshape(-1)
        _lib.call("asca_sync")
        self._flat["params"].upload(flat)

    def _get(self, which: str) -> dict:
        _lib.call("asca_sync")
        flat = self._flat[which].to_host((self.n_floats,))
        return {name: flat[off:off + r * c].reshape(r, c).copy() for name, off, r, c in self.tensors}

    def params(self) -> dict:
        return self._get("params")

    def grads(self) -> dict:
        return self._get("grads")

    # -- device buffers -----------------------------------------------------------
    def _p(self, name: str, which: str = "params"):
        return C.c_void_p(self._flat[which].ptr + 4 * self._at[name])

    def _g(self, name: str):
        return self._p(name, "grads")

    def _buf(self, key: str, nbytes: int) -> DevBuf:
        b = self._bufs.get(key)
        if b is None or b.nbytes < nbytes:
            b = self._bufs[key] = DevBuf(nbytes)
        return b

    def _rows(self, key: str, rows: int, cols: int) -> C.c_void_p:
        return _vp(self._buf(key, rows * cols * 4))

    def _up(self, key: str, a, dtype) -> C.c_void_p:
        a = np.ascontiguousarray(a, dtype)
        b = self._buf(key, a.nbytes)
        b.upload(a)
        return _vp(b)

    @staticmethod
    def _col(p: C.c_void_p, c: int) -> C.c_void_p:
        return C.c_void_p(p.value + 4 * c)

    @staticmethod
    def _gemm(ta, tb, m, n, k, a, lda, b, ldb, c, ldc, beta=0.0):
        _lib.call("asca_gemm", ta, tb, m, n, k, 1.0, a, lda, b, ldb, beta, c, ldc, None, None)

    def _ids(self, ids, used=None) -> np.ndarray:
        """Ids as int32; one outside the table is refused, or 0 where it is not `used`."""
        ids = np.asarray(ids).astype(np.int64)
        if used is not None:
            ids = np.where(used, ids, 0)
        if ids.size and not 0 <= int(ids.min()) <= int(ids.max()) < self.vocab:
            raise ValueError(f"ids from {ids.min()} to {ids.max()}, expected 0 .. {self.vocab - 1}")
        return ids.astype(np.int32)

    # -- forward --------------------------------------------------------------------
    def _forward(self, ids, batch: int, keep: bool, states=None, lens=None, one: bool = False) -> C.c_void_p:
        """Normalised rows after the last layer.  `keep`: layer by layer, for the
        backward; `states`: (conv, scan) states that the rows go on from and leave
        (`one`: a single row each, updated in place; ids may be on the device then)."""
        rows, d, N, W, R, X = batch if isinstance(ids, DevBuf) else len(ids), self.d, self.N, self.W, self.R, self.X
        T = rows // batch
        tag = (lambda k, i: f"{k}.{i}") if keep else (lambda k, i: f"{k}.{i % 2}")
        x, nrm = self._rows(tag("x", 0), rows, d), self._rows(tag("n", 0), rows, d)
        _lib.call("asca_gather_rows", self._p("embed"), _vp(ids) if isinstance(ids, DevBuf) else self._up("ids", ids, np.int32),
                  rows, d, x, None)
        _lib.call("asca_block_norm_fwd", x, d, None, 0, None, 0, None, None, self._p("w_pre.0"), None, 0, nrm, d, rows, d, EPS, F32, None)
        for i in range(self.L):
            uz, c, y = self._rows(tag("uz", i), rows, 2 * d), self._rows(tag("c", i), rows, d), self._rows(tag("y", i), rows, d)
            rbc, dt = self._rows(tag("rbc", i), rows, X), self._rows(tag("dt", i), rows, d)
            o = self._rows(tag("o", i), rows, d)
            w = lambda k: self._p(f"{k}.{i}")  # noqa: E731
            self._gemm(0, 0, rows, 2 * d, d, nrm, d, w("w_in"), 2 * d, uz, 2 * d)
            cs = hs = cn = hn = None
            if states is not None:
                cs, hs = self._col(states[0], i * batch * (W - 1) * d), self._col(states[1], i * batch * N * d)
            if states is not None and not one:   # a prompt's calls leave new states beside the old
                cn, hn = self._rows("conv_new", batch * (W - 1), d), self._rows("scan_new", batch * N, d)
            if one:
                _lib.call("asca_conv_step", cs, uz, 2 * d, w("conv_w"), w("conv_b"), c, d, batch, d, W, 1, F32, None)
            else:
                _lib.call("asca_conv_fwd", uz, 2 * d, w("conv_w"), w("conv_b"), cs, lens, c, d, cn, batch, T, d, W, 1, F32, None)
            self._gemm(0, 0, rows, X, d, c, d, w("w_x"), X, rbc, X)
            self._gemm(0, 0, rows, d, R, rbc, X, w("w_dt"), d, dt, d)
            ins = (c, d, dt, d, w("dt_bias"), w("A"), self._col(rbc, R), X, self._col(rbc, R + N), X, w("Dk"))
            if one:
                _lib.call("asca_ssm_step", hs, *ins, y, d, batch, d, N, 1, 1, F32, None)
            else:
                ws = None
                if keep:
                    n = C.c_size_t()
                    _lib.call("asca_ssm_ws_bytes", batch, T, d, N, C.byref(n))
                    ws = _vp(self._buf(f"ws.{i}", n.value))
                _lib.call("asca_ssm_fwd", *ins, hs, lens, y, d, hn, ws, batch, T, d, N, 1, 1, F32, None)
            if cn is not None:
                _lib.call("asca_d2d", cs, cn, batch * (W - 1) * d * 4, None)
                _lib.call("asca_d2d", hs, hn, batch * N * d * 4, None)
            self._gemm(0, 0, rows, d, d, y, d, w("w_o"), d, o, d)
            x2, n2 = self._rows(tag("x", i + 1), rows, d), self._rows(tag("n", i + 1), rows, d)
            _lib.call("asca_block_norm_fwd", x, d, o, d, self._col(uz, d), 2 * d, w("w_post"), w("scale"), self._p(f"w_pre.{i + 1}"),
                      x2, d, n2, d, rows, d, EPS, F32, None)
            x, nrm = x2, n2
        return nrm

    def _head(self, nrm: C.c_void_p, rows: int) -> C.c_void_p:
        logits = self._rows("logits", rows, self.vocab)
        self._gemm(0, 0, rows, self.vocab, self.d, nrm, self.d, self._p("head"), self.vocab, logits, self.vocab)
        return logits

    # -- training -------------------------------------------------------------------
    def forward_backward(self, ids, targets, batch: int, teacher: Teacher | None = None, alpha: float = 0.5,
                         weights=None) -> float:
        """Mean cross-entropy of batch sequences (rows b*T ..), its gradients in grads().  With
        a teacher's largest logits of the same rows the mean of asca_distill's loss, alpha of
        the teacher (targets may be None with alpha = 1), `weights` a weight a row."""
        rows, d, V, N, W, R, X, L = len(ids), self.d, self.vocab, self.N, self.W, self.R, self.X, self.L
        if batch < 1 or rows < 1 or rows % batch or np.shape(ids) != (rows,) or (
                np.shape(targets) != (rows,) and not (targets is None and teacher is not None and alpha == 1.0)):
            raise ValueError("ids/targets must hold batch * seq tokens each")
        if teacher is not None and teacher.rows != rows:
            raise ValueError(f"a teacher of {teacher.rows} rows for {rows}")
        if weights is not None and (teacher is None or np.shape(weights) != (rows,)):
            raise ValueError(f"weights of shape {np.shape(weights)}, expected {(rows,)} and a teacher")
        T = rows // batch
        nrm = self._forward(self._ids(ids), batch, True)
        logits = self._head(nrm, rows)
        dlog, losses = self._rows("dlog", rows, V), self._rows("losses", rows, 1)
        tgt = None if targets is None else self._up("tgt", targets, np.uint32)
        if teacher is None:
            _lib.call("asca_cross_entropy", logits, tgt, rows, V, dlog, losses, None)
        else:
            _lib.call("asca_distill", logits, V, _vp(teacher.values), _vp(teacher.ids), _vp(teacher.lse), teacher.k, tgt,
                      None if weights is None else self._up("weights", weights, _f32), teacher.temperature, alpha, 1.0 / rows, losses,
                      dlog, V, rows, V, F32, None)
        dn, dr, do, duz = (self._rows(k, rows, c) for k, c in (("dn", d), ("dr", d), ("do", d), ("duz", 2 * d)))
        dy, dc, ddt, drbc = (self._rows(k, rows, c) for k, c in (("dy", d), ("dc", d), ("ddt", d), ("drbc", X)))
        self._gemm(1, 0, d, V, rows, nrm, d, dlog, V, self._g("head"), V)
        self._gemm(0, 1, rows, d, V, dlog, V, self._p("head"), V, dn, d)
        first = None   # nothing but the norm reads the last layer's residual stream
        for i in reversed(range(L)):
            w, g = (lambda k: self._p(f"{k}.{i}")), (lambda k: self._g(f"{k}.{i}"))
            at = lambda k, j=i: _vp(self._bufs[f"{k}.{j}"])  # noqa: E731
            _lib.call("asca_block_norm_bwd", at("x"), d, at("o"), d, self._col(at("uz"), d), 2 * d, w("w_post"), w("scale"),
                      self._p(f"w_pre.{i + 1}"), first, d, dn, d, dr, d, do, d, self._col(duz, d), 2 * d, g("w_post"), g("scale"),
                      self._g(f"w_pre.{i + 1}"), rows, d, EPS, F32, None)
            first = dr
            self._gemm(1, 0, d, d, rows, at("y"), d, do, d, g("w_o"), d)
            self._gemm(0, 1, rows, d, d, do, d, w("w_o"), d, dy, d)
            rbc = at("rbc")
            _lib.call("asca_ssm_bwd", at("c"), d, at("dt"), d, w("dt_bias"), w("A"), self._col(rbc, R), X, self._col(rbc, R + N), X,
                      w("Dk"), None, dy, d, None, at("ws"), dc, d, ddt, d, g("dt_bias"), g("A"), self._col(drbc, R), X,
                      self._col(drbc, R + N), X, g("Dk"), None, batch, T, d, N, 1, 1, F32, None)
            self._gemm(1, 0, R, d, rows, rbc, X, ddt, d, g("w_dt"), d)
            self._gemm(0, 1, rows, R, d, ddt, d, w("w_dt"), d, drbc, X)
            self._gemm(1, 0, d, X, rows, at("c"), d, drbc, X, g("w_x"), X)
            self._gemm(0, 1, rows, d, X, drbc, X, w("w_x"), X, dc, d, 1.0)
            _lib.call("asca_conv_bwd", at("uz"), 2 * d, w("conv_w"), w("conv_b"), None, None, dc, d, None, duz, 2 * d, g("conv_w"),
                      g("conv_b"), None, batch, T, d, W, 1, F32, None)
            self._gemm(1, 0, d, 2 * d, rows, at("n"), d, duz, 2 * d, g("w_in"), 2 * d)
            self._gemm(0, 1, rows, d, 2 * d, duz, 2 * d, w("w_in"), 2 * d, dn, d)
        _lib.call("asca_block_norm_bwd", _vp(self._bufs["x.0"]), d, None, 0, None, 0, None, None, self._p("w_pre.0"), None, d, dn, d,
                  None, 0, None, 0, None, 0, None, None, self._g("w_pre.0"), rows, d, EPS, F32, None)
        _lib.call("asca_sync")
        return float(self._bufs["losses"].to_host((rows,)).mean(dtype=np.float64))

    def clip(self, max_norm: float) -> tuple[float, float]:
        """Scale the gradients to a global norm of at most max_norm: (norm, factor)."""
        return self._clip.clip(max_norm)

    def adamw(self, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, wd=0.01) -> None:
        """One AdamW step over every trained tensor."""
        self._step += 1
        s = gpu().adamw_scalars(lr, beta1, beta2, eps, wd, self._step)
        off = self._at["head"]   # all but the embedding, which comes first
        at = lambda k: C.c_void_p(self._flat[k].ptr + 4 * off)  # noqa: E731
        _lib.call("asca_adamw", at("params"), at("grads"), at("m"), at("v"), self.n_floats - off, s[0], beta1, beta2, s[1], s[2], None)

    def teacher(self, ids, batch: int, k: int, temperature: float = 1.0, rest: bool = True) -> Teacher:
        """The k largest logits of each row of batch sequences on the device, and with `rest`
        the whole sum's logarithm, for a student's forward_backward."""
        rows = len(ids)
        if batch < 1 or rows < 1 or rows % batch or np.shape(ids) != (rows,):
            raise ValueError("ids must hold batch * seq tokens")
        logits = self._head(self._forward(self._ids(ids), batch, False), rows)
        t = Teacher(DevBuf(rows * k * 4), DevBuf(rows * k * 4), DevBuf(rows * 4) if rest else None, rows, k, temperature)
        _lib.call("asca_top_logits", logits, self.vocab, rows, self.vocab, k, t.temperature, _vp(t.values), _vp(t.ids), _vp(t.lse),
                  F32, None)
        return t

    # -- serving ----------------------------------------------------------------------
    def new_state(self, n_seq: int) -> tuple[DevBuf, DevBuf]:
        """Zero (convolution, scan) states of n_seq sequences, all layers."""
        st = tuple(DevBuf(self.L * n_seq * k * self.d * 4) for k in (self.W - 1, self.N))
        for b in st:
            _lib.call("asca_memset32", _vp(b), 0, b.nbytes // 4, None)
        return st

    def _states(self, states, n: int) -> tuple:
        """The addresses of states that hold n sequences; a layer's begin at its index
        times n, so those of another number are refused."""
        for b, k in zip(states, (self.W - 1, self.N), strict=True):
            if b.nbytes != self.L * n * k * self.d * 4:
                raise ValueError(f"states of {b.nbytes} bytes for n={n} sequences ({self.L * n * k * self.d * 4})")
        return tuple(_vp(b) for b in states)

    def prompt(self, ids, states, lens=None) -> np.ndarray:
        """Rows of n_seq prompts, ids (n_seq, T) of which sequence b has lens[b], going on
        from `states` and leaving them after each one's last row; the (n_seq, V) logits of
        that row (of a prompt of length 0: of its first column's id, which it does not take).
        Ids past a length may be anything."""
        ids = np.atleast_2d(np.asarray(ids))
        n, T = ids.shape
        if n == 0 or T == 0:
            raise ValueError(f"ids of shape {ids.shape} have no row to give logits of")
        st = self._states(states, n)
        dl = None
        if lens is None:
            last = np.full(n, T - 1)
        else:
            lens = np.clip(np.asarray(lens, np.int32), 0, T)
            if lens.shape != (n,):
                raise ValueError(f"lens has shape {lens.shape}, expected {(n,)}")
            last = np.maximum(lens - 1, 0)
        ids = self._ids(ids, np.arange(T) <= last[:, None])
        if lens is not None:
            dl = self._up("lens", lens, np.int32)
        nrm = self._forward(ids.reshape(-1), n, False, st, dl)
        pick = self._rows("pick", n, self.d)
        _lib.call("asca_gather_rows", nrm, self._up("last", np.arange(n) * T + last, np.int32), n, self.d, pick, None)
        self._head(pick, n)
        _lib.call("asca_sync")
        return self._bufs["logits"].to_host((n, self.vocab))

    def step(self, ids, states) -> np.ndarray:
        """One row for each sequence on its states, in place; (n_seq, V) logits."""
        ids = self._ids(np.atleast_1d(ids))
        if ids.size == 0 or ids.size != len(ids):
            raise ValueError(f"ids of shape {ids.shape}, expected one for each sequence")
        nrm = self._forward(ids, len(ids), False, self._states(states, len(ids)), one=True)
        self._head(nrm, len(ids))
        _lib.call("asca_sync")
        return self._bufs["logits"].to_host((len(ids), self.vocab))

    def _step_dev(self, ids: DevBuf, n: int, states) -> DevBuf:
        """The device logits of one step on device ids."""
        self._head(self._forward(ids, n, False, self._states(states, n), one=True), n)
        return self._bufs["logits"]

    def _state_bufs(self, states, n: int) -> list:
        """The states' layout, (L, n) states of a layer each."""
        self._states(states, n)
        return [(b, self.L, k * self.d * 4) for b, k in zip(states, (self.W - 1, self.N), strict=True) if k]

    def beam_search(self, ids, beams: int, steps: int, lens=None, eos: int | None = None):
        """The `beams` best continuations, up to `steps` tokens, of n prompts, ids (n, T) of
        which sequence b has lens[b]: (tokens, scores) of search.beam_search."""
        ids = np.atleast_2d(np.asarray(ids))
        n = len(ids)
        search.check(n, beams, steps, eos, self.vocab)
        one, many = self.new_state(n), self.new_state(n * beams)
        try:
            self.prompt(ids, one, lens)
            return search.beam_search(self, self._bufs["logits"], one, many, n, beams, steps, eos)
        finally:
            for b in (*one, *many):
                b.free()

    def close(self) -> None:
        self._clip.close()
        for b in (*self._bufs.values(), *self._flat.values()):
            b.free()
        self._bufs, self._flat = {}, {}

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
