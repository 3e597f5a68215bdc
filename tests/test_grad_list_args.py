"""GradList's checks of its tensors before any device call.  CPU only: the library's
calls and device buffers are replaced by recorders."""
import pytest

from asca_amd import gpu, model


class Buf(gpu.DevBuf):
    __slots__ = ()

    def __init__(self, nbytes):
        self.nbytes, self.ptr = int(nbytes), 1 << 20

    def free(self):
        pass


@pytest.fixture
def log(monkeypatch):
    calls: list = []
    monkeypatch.setattr(gpu, "DevBuf", Buf)
    monkeypatch.setattr(gpu._lib, "call", lambda name, *a: calls.append(name))
    return calls


@pytest.mark.parametrize("dtype,size", [(gpu.F32, 4), (gpu.BF16, 2)])
def test_a_buffer_smaller_than_its_tensor(log, dtype, size):
    small, right = Buf(9 * size), Buf(10 * size)
    for src, dst in (([(small, 10)], None), ([(right, 10), (small, 10)], None), ([(right, 10)], [small])):
        with pytest.raises(ValueError):
            gpu.GradList(src, dst, dtype=dtype)
    assert not log
    gpu.GradList([(right, 10), (small, 9), (1 << 20, 10)], [right, small, right], dtype=dtype)
    assert log == ["asca_grads_create"]


def test_clipping_a_closed_model(log):
    m = model.DeviceModel.__new__(model.DeviceModel)
    m._h, m._grad_list, m._ptr, m.tensors, m._bufs = 1, None, {"grads": 1 << 20}, [("w", 0, 3, 4)], {}
    m.clip_grads(1.0, sync=False)
    m.close()
    del log[:]
    with pytest.raises(RuntimeError):   # its gradients' memory is freed
        m.clip_grads(1.0, sync=False)
    assert not log
