"""Stored records at the ends of what a call takes: the longest chunks, steps that no packing would choose."""
import os

import numpy as np
import pytest

from conftest import pkg

abi, hip, dm = pkg("abi"), pkg("hip"), pkg("devmem")


# ---- without a card ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", [abi.KV_F32, abi.KV_I16, abi.KV_I8, abi.KV_I4])
def test_the_longest_records_sizes(fmt):
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libtah_hip.so not built")
    for rc in (0, 1, 64, 2 ** 31 - 65, 2 ** 31 - 64, 2 ** 31 - 63, 2 ** 31 - 1):
        assert abi.lib().tah_kv_record(fmt, 16, rc) == abi.kv_record(fmt, 16, rc)


# ---- the card ------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [abi.KV_I16, abi.KV_I8, abi.KV_I4])
def test_chunks_past_what_a_call_takes_are_refused(fmt):
    """Rows of a chunk are numbered in 32 bits with room above. Under a budget of 1 MB, so that a call that was let
    through would end before it read anything."""
    g = hip.Gpu(0)
    g.set_work_budget(1 << 20)
    some = np.zeros(64, np.float32)
    at, bytes_at = some.ctypes.data_as(abi.F32P), some.ctypes.data_as(abi.U8P)
    for rows in (2 ** 31 - 1, 2 ** 31 - 1000):
        assert g._l.tah_pack(g._h, at, 1, rows, fmt, bytes_at) == abi.E_ARG
        assert g._l.tah_unpack(g._h, bytes_at, 1, rows, rows, fmt, at) == abi.E_ARG
        assert g._l.tah_unpack(g._h, bytes_at, 1, rows, 2 ** 31 - 1, fmt, at) == abi.E_ARG
    assert g._l.tah_pack(g._h, at, 1, 2 ** 31 - 1024, fmt, bytes_at) == abi.E_BUDGET
    assert g._l.tah_unpack(g._h, bytes_at, 1, 2 ** 31 - 1024, 2 ** 31 - 1, fmt, at) == abi.E_BUDGET
    g.close()
