"""Where `pages.PagePool` takes its memory: on its handle's card, whichever is current, with the handle's errors; a runtime of two cards
stands in. And a replacement that fails, with a stand-in for the card."""
import ctypes
import os

import numpy as np
import pytest

from conftest import pkg

abi, hip, pages, devmem = pkg("abi"), pkg("hip"), pkg("pages"), pkg("devmem")


class Runtime:
    """hipGetDevice, hipSetDevice, hipMalloc and hipFree of two cards."""

    def __init__(self, current, status=0):
        self.current, self.status, self.made = current, status, []

    def hipGetDevice(self, p):
        p._obj.value = self.current
        return 0

    def hipSetDevice(self, ordinal):
        if not 0 <= ordinal < 2:
            return 101
        self.current = ordinal
        return 0

    def hipMalloc(self, p, nbytes):
        self.made.append((self.current, nbytes))
        p._obj.value = 1 << 20
        return self.status

    def hipFree(self, p):
        return 0


class Handle:
    def __init__(self, ordinal):
        self.ordinal = ordinal


@pytest.fixture
def built():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libtah_hip.so not built")


SIZES = dict(layers=2, heads=2, hd=16, pages=10, page_rows=16)


@pytest.mark.parametrize("ordinal", [0, 1])
@pytest.mark.parametrize("current", [0, 1])
def test_memory_is_the_handles_cards(built, monkeypatch, ordinal, current):
    rt = Runtime(current)
    monkeypatch.setattr(devmem, "_rt", rt)
    pool = pages.PagePool(Handle(ordinal), **SIZES)
    assert rt.made == [(ordinal, pool.bytes())] and rt.current == current
    pool.free()


@pytest.mark.parametrize("status,error", [(2, hip.BudgetError), (1, hip.CardError), (101, hip.CardError)])
def test_failures_are_the_handles(built, monkeypatch, status, error):
    rt = Runtime(0, status)
    monkeypatch.setattr(devmem, "_rt", rt)
    with pytest.raises(error):
        pages.PagePool(Handle(1), **SIZES)
    assert rt.current == 0
    with pytest.raises(hip.CardError):  # no such card
        pages.PagePool(Handle(2), **SIZES)
    assert rt.current == 0


@pytest.mark.gpu
def test_a_handle_knows_its_card():
    gpu = hip.Gpu(0)
    assert gpu.ordinal == 0
    pool = pages.PagePool(gpu, **SIZES)
    before = ctypes.c_int(-1)
    assert devmem.rt().hipGetDevice(ctypes.byref(before)) == 0 and before.value == 0
    pool.hold("a", 0, [(np.ones((3, 32), np.float32), np.ones((3, 32), np.float32))] * 2)
    assert np.all(np.abs(pool.attend("a", 0, 1, np.ones((1, 32), np.float32), 32, 2) - 1) <= 2.0**-20)
    pool.free()
    gpu.close()
