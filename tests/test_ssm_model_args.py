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


def test_ids_outside_the_table(model):
    m, log = model
    st = m.new_state(2)
    for bad in (17, -1, 1 << 31, 1 << 32):
        refused(log, m.step, np.array([0, bad]), st)
        refused(log, m.prompt, np.array([[0, 1], [bad, 1]]), st)
        refused(log, m.prompt, np.array([[0, 1], [1, bad]]), st, [2, 2])
        refused(log, m.prompt, np.array([[0, 1], [bad, 1]]), st, [2, 0])   # its logits are of this row
        refused(log, m.forward_backward, np.array([0, 1, 2, bad]), np.zeros(4, int), 2)
    m.step(np.array([0, 16], np.uint8), st)
    m.step([0, 16], st)


def test_ids_past_a_prompts_length_do_not_matter(model):
    m, log = model
    st = m.new_state(3)
    del log[:]
    m.prompt(np.array([[1, 2, 99], [3, -1, -1], [4, 99, 99]]), st, [2, 1, 0])
    up = [a for n, a in log if n == "upload" and a.size == 9]
    assert len(up) == 1 and up[0].min() >= 0 and up[0].max() < 17
    np.testing.assert_array_equal(up[0].reshape(3, 3)[[0, 0, 1, 2], [0, 1, 0, 0]], [1, 2, 3, 4])


def test_no_rows(model):
    m, log = model
    st = m.new_state(2)
    refused(log, m.prompt, np.zeros((2, 0), int), st)         # there is no row to give logits of
    refused(log, m.prompt, np.zeros((2, 0), int), st, [0, 0])
    none = m.new_state(0)
    refused(log, m.prompt, np.zeros((0, 4), int), none)
    refused(log, m.step, [], none)
    refused(log, m.step, np.zeros((2, 2), int), st)           # two ids for a sequence
    for batch in (2, 0, -1):
        refused(log, m.forward_backward, [], [], batch)
    refused(log, m.forward_backward, np.zeros(4, int), np.zeros(4, int), 0)
    refused(log, m.forward_backward, np.zeros(4, int), np.zeros(4, int), -2)


def test_training_rows_lie_one_after_another(model):
    m, log = model
    refused(log, m.forward_backward, np.zeros((2, 5), int), np.zeros((2, 5), int), 2)   # two rows, by their length
    m.forward_backward(np.zeros(10, int), np.zeros(10, int), 2)
    assert "asca_ssm_bwd" in names(log)
