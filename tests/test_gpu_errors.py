"""A failed call leaves nothing behind that a later one is blamed for."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_the_call_after_a_refused_allocation_works(g):
    from asca_amd import _lib
    from asca_amd.model import DeviceModel

    x = np.ones((3, 8), np.float32)
    want = g.block_norm(x)
    m = DeviceModel(16, 512, 4, 1, 1, 16)
    f = C.c_void_p(1 << 12)   # never dereferenced: the first of the call's buffers alone is 1 TB
    with pytest.raises(_lib.AscaError) as ei:
        _lib.call("asca_model_decode_step", m._h, f, 500_000_000, f, f, None)
    assert ei.value.code == 6, str(ei.value)
    got = g.block_norm(x)
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
    m.close()
