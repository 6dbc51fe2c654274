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
