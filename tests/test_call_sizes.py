"""Calls over many tables at the sizes where a launch has more threads than a grid's dimension takes (2^32): answered, or refused before
anything is queued."""
import ctypes

import numpy as np
import pytest

from conftest import pkg

abi, hip, dm = pkg("abi"), pkg("hip"), pkg("devmem")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


class Far:
    """`nbytes` of zeros on the card, and numbers put to or taken from any place in it."""

    def __init__(self, nbytes):
        self.b = dm.DeviceBuffer(nbytes)
        assert dm.rt().hipMemset(ctypes.c_void_p(self.b.ptr), 0, ctypes.c_size_t(nbytes)) == 0
        dm.synchronize()

    def put(self, at, a):
        assert dm.rt().hipMemcpy(ctypes.c_void_p(self.b.ptr + at), ctypes.c_void_p(a.ctypes.data), ctypes.c_size_t(a.nbytes), 1) == 0

    def take(self, at, shape):
        a = np.empty(shape, np.float32)
        assert dm.rt().hipMemcpy(ctypes.c_void_p(a.ctypes.data), ctypes.c_void_p(self.b.ptr + at), ctypes.c_size_t(a.nbytes), 2) == 0
        return a


def test_more_tiles_than_a_launch_takes_are_refused(gpu):
    """2^22 tables of a query each, 8 heads: 2^25 workgroups. Nothing is read: the arrays are as long as the sizes say all the same."""
    tables, hd = 2**22, 16
    offsets, q = Far((tables + 1) * 4), Far(tables * 8 * hd * 4)
    k = dm.DeviceBuffer(8 * hd * 4)
    try:
        with pytest.raises(ValueError):
            gpu.attend_packed_dev(q.b.ptr, k.ptr, k.ptr, offsets.b.ptr, offsets.b.ptr, tables, tables, 1, 8, 8, hd, q.b.ptr)
        gpu.sync()
    finally:
        offsets.b.free()
        q.b.free()
        k.free()
