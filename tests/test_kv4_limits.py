"""Stored records at the ends of what a call takes: the longest chunks, steps that no packing would choose."""
import os

import numpy as np
import pytest

import kv4_plain as P
import test_kv4_kernels as K
from conftest import pkg

abi, hip, M = pkg("abi"), pkg("hip"), pkg("model")


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


def bf16_bits(x):
    return int(np.float32(x).view(np.uint32)) >> 16


def with_steps_of_its_own(rec, d, rc, j, s, z, code, other=None):
    """A record's coordinate j as a step s and an offset z (bfloat16 numbers) and one code throughout, or two in turn."""
    ng, half = -(-rc // 64), (rc + 1) // 2
    rec[:8 * d * ng].view(np.uint16).reshape(2 * d, ng, 2)[j] = bf16_bits(s), bf16_bits(z)
    codes = rec[8 * d * ng:].reshape(2 * d, half)
    codes[j] = (code + 8) + 16 * ((code if other is None else other) + 8)
    if rc % 2:
        codes[j, -1] &= 15


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 16])
@pytest.mark.parametrize("nq", [3, 40, 1100])
def test_steps_that_no_packing_would_choose(width, nq):
    """Records that hold steps and offsets far larger than any value they stand for (a level beside 0 used throughout), or
    negative ones: attention over them is attention over what they stand for, as for any record."""
    print(f"steps of other packings: heads of {width}, {nq} queries", flush=True)
    g = hip.Gpu(0)
    heads, rows, chunk = 8, 3000, 1000
    d = heads * width
    cfg = dict(M.FULL_CLASSIFIER, col_num_blocks=1, row_num_blocks=1, icl_num_blocks=1)
    if width == 16:
        cfg = dict(cfg, icl_nhead=8, embed_dim=16, row_num_cls=8)
    w = g.weights(M.Model.random(cfg, seed=5))
    k, v, q = (a[:, :d].copy() for a in K.inputs(np.random.default_rng(nq), rows, heads, nq))
    third = slice(3 * width, 4 * width)
    for a in (k, v):
        a[:, third] *= 0.55 / a[:, third].std()
    q[:, third] *= 0.5 / q[:, third].std()
    rec = P.pack_layer(P.chunk_layout(k, v, chunk), d, rows, chunk)
    size = P.record(d, chunk)
    for ci in range(3):
        one = rec[ci * size:(ci + 1) * size]
        for at in (0, d):
            with_steps_of_its_own(one, d, chunk, at + 5, 2.0 ** 20, 2.0 ** 23, -8)        # 0
            with_steps_of_its_own(one, d, chunk, at + 9, -(2.0 ** 18), 2.0 ** 20, 4)      # 0, by a negative step
            with_steps_of_its_own(one, d, chunk, at + width + 3, 512.0, -3584.0, 7)       # 0, in another head
            with_steps_of_its_own(one, d, chunk, at + 2 * width + 1, -0.25, 0.125, 3)     # -0.625
            with_steps_of_its_own(one, d, chunk, at + 3 * width + 2, 4.0, 32.0, -8, -7)   # 0 and 4, the head's largest
    k4, v4 = P.unpack_layer(rec, d, rows, chunk)
    for a in (k4, v4):
        assert not a[:, [5, 9, width + 3]].any() and np.all(a[:, 2 * width + 1] == -0.625)
        assert np.all(a[::2, 3 * width + 2] == 0) and np.all(a[1::2, 3 * width + 2] == 4)
    vm = g.load(w, abi.KV_I4, rows, chunk, [rec], np.ones((1, d), np.float32))
    got, was_many = K.attend(g, vm, q)
    vm.free()
    w.free()
    g.close()
    assert was_many == (width == 64 and nq == 1100)
    e, want = got - P.attention(q, k4, v4, heads), P.attention(q, k4, v4, heads)
    share = lambda x: np.sqrt((x.astype(np.float64).reshape(nq, heads, width) ** 2).mean((0, 2)))
    print(f"  error {np.max(share(e) / share(want)):.1e}", flush=True)
    assert np.all(share(e) < K.LIMIT * share(want))
