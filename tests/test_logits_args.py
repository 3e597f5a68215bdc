"""Refusals of the operators behind the logits, at the C entries and in Python, before any
device call.  CPU only."""
import ctypes as C

import numpy as np
import pytest

from asca_amd import _lib, gpu, model, search, ssm

P = C.c_void_p(0x1000)   # never followed: a refused call reads no device memory
INVALID, UNSUPPORTED = 1, 3
NAN, INF = float("nan"), float("inf")


def code(name, *args):
    return getattr(_lib.load(), name)(*args)


def top(**k):
    a = dict(z=P, ld=10, rows=2, V=10, K=3, tau=1.0, v=P, i=P, lse=None, ty=0)
    a.update(k)
    return code("asca_top_logits", *a.values(), None)


@pytest.mark.parametrize("bad,want", [
    (dict(ld=9), INVALID), (dict(rows=-1), INVALID), (dict(V=0), INVALID), (dict(V=-3), INVALID), (dict(K=0), UNSUPPORTED),
    (dict(K=65), UNSUPPORTED), (dict(K=-1), UNSUPPORTED), (dict(tau=0.0), INVALID), (dict(tau=-1.0), INVALID),
    (dict(tau=NAN), INVALID), (dict(tau=INF), INVALID), (dict(z=None), INVALID), (dict(v=None), INVALID), (dict(i=None), INVALID),
    (dict(ty=2), UNSUPPORTED), (dict(z=C.c_void_p(0x1002)), INVALID), (dict(z=C.c_void_p(0x1001), ty=1), INVALID),
    (dict(rows=1 << 40), UNSUPPORTED)])
def test_top_logits(bad, want):
    assert top(**bad) == want and _lib.load().asca_last_error()


def distill(**k):
    a = dict(z=P, ld=10, tval=P, tids=P, tlse=None, K=3, tg=P, w=None, tau=1.0, alpha=0.5, scale=1.0, loss=P, dz=P, lddl=10, T=2,
             V=10, ty=0)
    a.update(k)
    return code("asca_distill", *a.values(), None)


@pytest.mark.parametrize("bad,want", [
    (dict(ld=9), INVALID), (dict(dz=C.c_void_p(0x9000), lddl=9), INVALID), (dict(T=-1), INVALID), (dict(V=0), INVALID),
    (dict(K=0), UNSUPPORTED), (dict(K=65), UNSUPPORTED), (dict(tau=0.0), INVALID), (dict(tau=NAN), INVALID),
    (dict(alpha=-0.1), INVALID), (dict(alpha=1.5), INVALID), (dict(alpha=NAN), INVALID), (dict(scale=INF), INVALID),
    (dict(scale=NAN), INVALID), (dict(z=None), INVALID), (dict(loss=None), INVALID), (dict(tval=None), INVALID),
    (dict(tids=None), INVALID), (dict(tg=None), INVALID), (dict(alpha=0.0, tg=None), INVALID), (dict(lddl=11), INVALID),
    (dict(V=(1 << 20) + 1, ld=1 << 21, lddl=1 << 21), UNSUPPORTED), (dict(ty=7), UNSUPPORTED), (dict(z=C.c_void_p(0x1001)), INVALID),
    (dict(dz=C.c_void_p(0x9001), ty=1), INVALID), (dict(T=1 << 40), UNSUPPORTED)])
def test_distill(bad, want):
    assert distill(**bad) == want and _lib.load().asca_last_error()


def step(**k):
    a = dict(z=P, ld=10, s=P, e=None, eos=-1, stay=0, ns=P, ne=None, tok=P, par=P, groups=2, K=4, V=10, ty=0)
    a.update(k)
    return code("asca_beam_step", *a.values(), None)


@pytest.mark.parametrize("bad,want", [
    (dict(ld=9), INVALID), (dict(groups=-1), INVALID), (dict(K=0), UNSUPPORTED), (dict(K=33), UNSUPPORTED), (dict(V=0), INVALID),
    (dict(eos=10, e=P, ne=P), INVALID), (dict(eos=3), INVALID), (dict(eos=3, e=P), INVALID), (dict(eos=3, ne=P), INVALID),
    (dict(e=P), INVALID), (dict(ne=P), INVALID), (dict(z=None), INVALID), (dict(s=None), INVALID), (dict(ns=None), INVALID),
    (dict(tok=None), INVALID), (dict(par=None), INVALID), (dict(ty=-1), UNSUPPORTED), (dict(z=C.c_void_p(0x1003)), INVALID)])
def test_beam_step(bad, want):
    assert step(**bad) == want and _lib.load().asca_last_error()


def states(n=1, src=0x1000, dst=None, outer=2, nbytes=64, count=None, groups=3, ks=4, kd=4):
    s = (C.c_void_p * 9)(*[src + 0x100000 * i if src else None for i in range(9)])
    d = None if dst is None else (C.c_void_p * 9)(*[dst] * 9)
    return code("asca_beam_states", s, d, (C.c_uint64 * 9)(*[outer] * 9), (C.c_uint64 * 9)(*[nbytes] * 9),
                n if count is None else count, P, groups, ks, kd, None)


@pytest.mark.parametrize("bad,want", [
    (dict(count=9), INVALID), (dict(count=-1), INVALID), (dict(groups=-1), INVALID), (dict(ks=0), UNSUPPORTED),
    (dict(ks=33, kd=33), UNSUPPORTED), (dict(kd=33), UNSUPPORTED), (dict(kd=0), UNSUPPORTED), (dict(ks=1), INVALID),
    (dict(dst=0x1000, ks=1), INVALID), (dict(src=0), INVALID),
    (dict(dst=0x1010), INVALID), (dict(dst=0x1000 + 2 * 3 * 4 * 64 - 1), INVALID),   # the last byte of the source
    (dict(outer=1 << 41), INVALID), (dict(nbytes=1 << 41), INVALID), (dict(outer=1 << 30, nbytes=1 << 20), UNSUPPORTED)])
def test_beam_states(bad, want):
    assert states(**bad) == want and _lib.load().asca_last_error()


def test_more_blocks_than_a_launch_takes():
    """Rows that memory could hold, in blocks of more threads than 256."""
    assert distill(T=9 << 20, V=8200, ld=8200, lddl=8200, ty=1) == UNSUPPORTED
    assert top(rows=9 << 20, V=40000, ld=40000) == UNSUPPORTED


def test_more_groups_than_a_launch_takes():
    assert step(groups=1 << 24, K=1, V=1, ld=1) == step(groups=1 << 24, K=1, V=9000, ld=9000) == UNSUPPORTED


@pytest.mark.parametrize("ty", [0, 1])
@pytest.mark.parametrize("V", [(1 << 30) + 1, 0x7fffffff - 4, 0x7fffffff])
def test_vocabularies_past_the_end_of_a_row(V, ty):
    """Columns of a row are counted in 32 bits, and its slices' ends past the last of them."""
    assert top(rows=1, V=V, ld=1 << 31, ty=ty) == UNSUPPORTED
    assert step(groups=1, K=1, V=V, ld=1 << 31, ty=ty) == UNSUPPORTED


@pytest.mark.parametrize("tau", [1e-31, 1e-42])
def test_a_temperature_without_a_finite_inverse(tau):
    assert top(tau=tau) == distill(tau=tau) == INVALID


@pytest.mark.parametrize("bad", [
    dict(dz=C.c_void_p(0x1004)), dict(dz=C.c_void_p(0x1000 - 4)), dict(dz=C.c_void_p(0x1000 + 40)), dict(dz=C.c_void_p(0x1000 + 76)),
    dict(dz=C.c_void_p(0x1000 + 36), ld=20, lddl=20), dict(dz=C.c_void_p(0x1000 + 44), ld=20, lddl=20),
    dict(dz=C.c_void_p(0x1000 + 40), ld=10, lddl=20)])
def test_gradients_that_share_memory_with_the_logits(bad):
    assert distill(**bad) == INVALID and _lib.load().asca_last_error()


def test_gradients_beside_the_logits():
    n = C.c_int(0)
    if _lib.load().asca_device_count(C.byref(n)) == 0 and n.value > 0:
        pytest.skip("a GPU is present; this checks the no-device path")
    assert distill(dz=C.c_void_p(0x1000 + 80)) == distill(dz=C.c_void_p(0x1000 + 40), ld=20, lddl=20) == 4
    assert distill(dz=C.c_void_p(0x1000 - 80)) == distill() == 4


def pairs(src, dst, k_src=4, outer=2, nbytes=64):
    n = len(src)
    arr = lambda t, a: (t * n)(*a)  # noqa: E731
    return code("asca_beam_states", arr(C.c_void_p, src), arr(C.c_void_p, dst), arr(C.c_uint64, [outer] * n),
                arr(C.c_uint64, [nbytes] * n), n, P, 3, k_src, 4, None)


SIZE = 2 * 3 * 4 * 64   # bytes of a buffer of four beams


@pytest.mark.parametrize("src,dst", [
    ([0x10000, 0x10000], [None, None]),                       # the same buffer twice, in place
    ([0x10000, 0x10000 + SIZE - 1], [None, None]),
    ([0x10000, 0x20000], [0x30000, 0x30000]),                 # one destination for two
    ([0x10000, 0x20000], [0x30000, 0x30000 + SIZE - 16]),
    ([0x10000, 0x20000], [0x20000, 0x30000]),                 # a destination that is another's source
    ([0x10000, 0x20000], [None, 0x10000]),
    ([0x10000, 0x20000], [0x20000 + SIZE - 1, None])])
def test_beam_states_that_share_memory(src, dst):
    assert pairs(src, dst) == INVALID and _lib.load().asca_last_error()


def test_beam_states_of_one_source():
    """Two destinations may take from one source, and lie side by side."""
    n = C.c_int(0)
    if _lib.load().asca_device_count(C.byref(n)) == 0 and n.value > 0:
        pytest.skip("a GPU is present; this checks the no-device path")
    assert pairs([0x10000, 0x10000], [0x30000, 0x30000 + SIZE]) == pairs([0x10000, 0x10000 + SIZE], [None, None]) == 4


def test_right_calls_get_as_far_as_the_device():
    lib = _lib.load()
    n = C.c_int(0)
    if lib.asca_device_count(C.byref(n)) == 0 and n.value > 0:
        pytest.skip("a GPU is present; this checks the no-device path")
    assert top() == top(V=70000, ld=70000) == distill() == distill(V=70000, ld=70000, lddl=70000) == 4
    assert step() == step(V=70000, ld=70000) == states() == states(dst=0x9000000, ks=1) == 4


def test_ids_that_are_none():
    np.testing.assert_array_equal(gpu._entry_ids([[3, -1, 1 << 31, (1 << 32) + 2, 0x7fffffff]]), [[3, -1, -1, -1, 0x7fffffff]])


def test_pointers_may_be_null_where_nothing_is_there():
    lib = _lib.load()
    assert lib.asca_beam_states(None, None, None, None, 0, None, 3, 1, 4, None) == 0
    assert top(rows=0, z=None, v=None, i=None) == 0
    assert distill(T=0, z=None, loss=None, tval=None, tids=None, tg=None, dz=None) == 0
    assert step(groups=0, z=None, s=None, ns=None, tok=None, par=None) == 0


# ------------------------------------------------------------------ Python


class Buf(gpu.DevBuf):
    __slots__ = ()

    def __init__(self, nbytes):
        self.nbytes, self.ptr = int(nbytes), 1 << 20

    def upload(self, a):
        pass

    def free(self):
        pass

    def to_host(self, shape, dtype=np.float32):
        return np.zeros(shape, dtype)


@pytest.fixture
def log(monkeypatch):
    calls: list = []
    for m in (gpu, model, ssm, search):
        monkeypatch.setattr(m, "DevBuf", Buf)
    monkeypatch.setattr(gpu._lib, "call", lambda name, *a: calls.append(name))
    return calls


def launched(log):
    return [c for c in log if c not in ("asca_sync", "asca_stream_sync")]


def refused(log, f, *a, **k):
    del log[:]
    with pytest.raises(ValueError):
        f(*a, **k)
    assert not launched(log)


def test_shapes_of_host_arrays(log):
    g = gpu.Gpu("", 1)
    z = np.zeros((4, 7), np.float32)
    v, i = np.zeros((4, 2), np.float32), np.zeros((4, 2), np.int32)
    refused(log, g.top_logits, z.astype(np.float64), 2)
    refused(log, g.distill, z, v[:3], i[:3], alpha=1.0)
    refused(log, g.distill, z, v, i[:, :1])
    refused(log, g.distill, z, v, i, tlse=np.zeros(3))
    refused(log, g.distill, z, v, i, targets=np.zeros(5, int), alpha=0.5)
    refused(log, g.distill, z, v, i, weights=np.zeros((4, 1)))
    refused(log, g.beam_step, z, np.zeros(4), k=3)
    refused(log, g.beam_step, z, np.zeros(4), k=0)
    refused(log, g.beam_step, z, np.zeros(3), k=2)
    refused(log, g.beam_step, z, np.zeros(4), k=2, ended=np.zeros(2), eos=1)
    g.distill(z, v, i)
    g.beam_step(z, np.zeros(4), k=2)
    assert launched(log) == ["asca_distill", "asca_beam_step"]


def test_buffers_smaller_than_their_states(log):
    g = gpu.Gpu("", 1)
    refused(log, g.beam_states, [(Buf(2 * 3 * 4 * 8 - 1), None, 2, 8)], [0] * 12, groups=3, k=4)
    refused(log, g.beam_states, [(Buf(2 * 3 * 8), Buf(2 * 3 * 4 * 8 - 1), 2, 8)], None, groups=3, k=4, k_src=1)
    refused(log, g.beam_states, [(Buf(2 * 3 * 4 * 8), None, 2, 8)], [0] * 11, groups=3, k=4)
    refused(log, g.beam_states, [(Buf(2 * 3 * 4 * 8), None, 2, 8)], Buf(11 * 4), groups=3, k=4)
    g.beam_states([(Buf(2 * 3 * 8), Buf(2 * 3 * 4 * 8), 2, 8)], None, groups=3, k=4, k_src=1)
    assert launched(log) == ["asca_beam_states"]


def test_teachers(log, monkeypatch):
    for bad in (dict(ids=np.zeros((4, 3))), dict(ids=np.zeros(4)), dict(lse=np.zeros(5))):
        a = dict(values=np.zeros((4, 2)), ids=np.zeros((4, 2)), lse=None)
        a.update(bad)
        refused(log, gpu.Teacher.upload, **a)
    t = gpu.Teacher.upload(np.zeros((6, 2)), np.zeros((6, 2)))
    monkeypatch.setattr(ssm, "gpu", lambda: True)
    monkeypatch.setattr(ssm, "GradList", lambda *a, **k: None)
    m = ssm.SsmModel(17, 8, 1)
    ids = np.zeros(6, int)
    refused(log, m.forward_backward, np.zeros(4, int), np.zeros(4, int), 2, t)       # another number of rows
    refused(log, m.forward_backward, ids, None, 2, t, alpha=0.5)                      # alpha of the targets
    refused(log, m.forward_backward, ids, None, 2)
    refused(log, m.forward_backward, ids, ids, 2, t, weights=np.zeros(5))
    refused(log, m.forward_backward, ids, ids, 2, weights=np.zeros(6))                # weights without a teacher
    refused(log, m.teacher, np.zeros((2, 3), int), 2, 4)
    refused(log, m.teacher, ids, 4, 2)
    refused(log, m.teacher, ids + 17, 2, 4)
    m.forward_backward(ids, None, 2, t, alpha=1.0)
    assert "asca_distill" in log
    d = model.DeviceModel.__new__(model.DeviceModel)
    d._h, d._grad_list, d._bufs, d.vocab = 1, None, {}, 17
    refused(log, d.distill, np.zeros(4, int), np.zeros(4, int), 2, t)
    refused(log, d.distill, ids, np.zeros(5, int), 2, t)
    refused(log, d.distill, ids, ids, 4, t)
    refused(log, d.distill, ids, ids, 0, t)
    refused(log, d.distill, ids, ids, 2, t, weights=np.zeros(3))
    d.distill(ids, None, 2, t, alpha=1.0, sync=False)
    assert launched(log) == ["asca_model_distill"]
    d._h = None


@pytest.mark.parametrize("bad", [dict(beams=0), dict(beams=33), dict(steps=0), dict(eos=17), dict(eos=-1)])
def test_searches(log, monkeypatch, bad):
    monkeypatch.setattr(ssm, "gpu", lambda: True)
    monkeypatch.setattr(ssm, "GradList", lambda *a, **k: None)
    m = ssm.SsmModel(17, 8, 1)
    a = dict(beams=2, steps=3, eos=None)
    a.update(bad)
    refused(log, m.beam_search, np.zeros((2, 3), int), **a)
    d = model.DeviceModel.__new__(model.DeviceModel)
    d._h, d._grad_list, d._bufs, d.vocab = None, None, {}, 17
    refused(log, d.beam_search, np.zeros((2, 3), int), **a)
    refused(log, d.beam_search, np.zeros((2, 0), int), 2, 3)


def test_a_search_is_traced_back():
    tok = np.array([[[5, 6, 7]], [[1, 2, 3]], [[4, 9, 8]]])      # steps, sequences, beams
    par = np.array([[[0, 0, 0]], [[2, 0, 0]], [[1, 1, 0]]])
    seqs, sc = search._trace(tok, par, np.array([[-3.0, -1.0, -2.0]]), 9)
    assert [list(s) for s in seqs[0]] == [[5, 2, 9], [7, 1, 8], [5, 2, 4]]
    np.testing.assert_array_equal(sc, [[-1.0, -2.0, -3.0]])
