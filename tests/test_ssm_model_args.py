"""The state space byte model's checks of its arguments: what would read or write
outside a buffer is refused before anything is uploaded or launched.  CPU only: the
library's calls and device buffers are replaced by recorders."""
import numpy as np
import pytest

from asca_amd import ssm


class Buf:
    """A device buffer's size; what is uploaded into it."""

    log: list = []

    def __init__(self, nbytes):
        self.nbytes, self.ptr = int(nbytes), 1 << 20

    def upload(self, a):
        assert a.nbytes <= self.nbytes
        self.log.append(("upload", np.array(a)))

    def to_host(self, shape, dtype=np.float32):
        return np.zeros(shape, dtype)

    def free(self):
        pass


@pytest.fixture
def model(monkeypatch):
    """(model, log of calls and uploads) with V = 17, d = 8, two layers."""
    log = Buf.log = []

    def call(name, *args):
        log.append((name, args))

    class List:
        def __init__(self, *a, **k):
            pass

        def close(self):
            pass

    monkeypatch.setattr(ssm, "gpu", lambda: True)
    monkeypatch.setattr(ssm, "DevBuf", Buf)
    monkeypatch.setattr(ssm, "GradList", List)
    monkeypatch.setattr(ssm, "_vp", lambda b: ssm.C.c_void_p(b.ptr))
    monkeypatch.setattr(ssm._lib, "call", call)
    m = ssm.SsmModel(17, 8, 2, n_state=5, conv_width=3)
    return m, log


def refused(log, f, *args):
    del log[:]
    with pytest.raises(ValueError):
        f(*args)
    assert not log, log[0][0]


def names(log):
    return [n for n, _ in log]


def test_states_of_another_number_of_sequences(model):
    m, log = model
    for n in (1, 2, 4, 6):   # layer i's states begin at i times the number of sequences: fewer would move others'
        st = m.new_state(n)
        refused(log, m.step, np.zeros(3, int), st)
        refused(log, m.prompt, np.zeros((3, 5), int), st)
    st = m.new_state(3)
    refused(log, m.step, np.zeros(3, int), st[::-1])
    refused(log, m.step, np.zeros(3, int), (st[0], Buf(4)))
    m.step(np.zeros(3, int), st)
    m.prompt(np.zeros((3, 5), int), st)
    assert "asca_ssm_step" in names(log) and "asca_ssm_fwd" in names(log)


@pytest.mark.parametrize("lens", [4, [4], [4, 4], [4, 4, 4, 4], [[4, 4, 4]]])
def test_lengths_of_another_number_of_sequences(model, lens):
    m, log = model
    st = m.new_state(3)
    refused(log, m.prompt, np.zeros((3, 5), int), st, lens)
    m.prompt(np.zeros((3, 5), int), st, [4, 0, 9])
    assert "asca_ssm_fwd" in names(log)
