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


def test_rows_past_two_to_the_thirty(gpu):
    """2^30 + 100 rows of one head of 16 (64 GiB; keys and values the same), of which the last 40 and some before fall on pages."""
    rows, hd, page = 2**30 + 100, 16, 16
    far = Far(rows * hd * 4)
    try:
        rng = np.random.default_rng(1)
        first, last = rng.standard_normal((page, hd)).astype(np.float32), rng.standard_normal((40, hd)).astype(np.float32)
        far.put(0, first)
        far.put((rows - 40) * hd * 4, last)
        pool = dm.DeviceBuffer(4 * abi.page_bytes(abi.KV_F32, 1, hd, page))
        # table 0: the first 16 rows; table 1: all others, of which the last 40 are its rows 0 .. 39; rows before them are on no page
        table = dm.DeviceBuffer.of(np.array([[2, -1, -1], [1, 3, 0]], np.int32))
        starts, offsets = dm.DeviceBuffer.of(np.array([0, -(rows - page - 40)], np.int32)), dm.DeviceBuffer.of(np.array([0, page, rows], np.int32))
        d = abi.Pages(pool=pool.ptr, table=table.ptr, kv_format=abi.KV_F32, kv_heads=1, hd=hd, page_rows=page, pages=4, tables=2, ld=3)
        print("write", flush=True)
        gpu.pages_write_dev(d, starts.ptr, offsets.ptr, far.b.ptr, far.b.ptr, rows)
        gpu.sync()
        # back into the same place: all other rows zeros, which they were
        far.put(0, np.full((page, hd), 9.0, np.float32))
        far.put((rows - 45) * hd * 4, np.full((45, hd), 9.0, np.float32))
        print("read", flush=True)
        gpu.pages_read_dev(d, starts.ptr, offsets.ptr, far.b.ptr, far.b.ptr, rows)
        gpu.sync()
        assert np.array_equal(far.take(0, (page, hd)), first)
        assert np.array_equal(far.take((rows - 40) * hd * 4, (40, hd)), last)
        assert not np.any(far.take((rows - 45) * hd * 4, (5, hd)))
    finally:
        far.b.free()


def test_queries_past_two_to_the_twenty_six(gpu):
    """2^26 + 5 queries of a head of 16 over a table of two rows, a third of which the join puts together where their units are cut."""
    nq, hd, page = 2**26 + 5, 16, 16
    q, out = Far(nq * hd * 4), Far(nq * hd * 4)
    try:
        pool = dm.DeviceBuffer.of(np.zeros(abi.page_bytes(abi.KV_F32, 1, hd, page), np.uint8))
        kv = np.arange(2 * hd, dtype=np.float32).reshape(2, hd)
        d = abi.Pages(pool=pool.ptr, kv_format=abi.KV_F32, kv_heads=1, hd=hd, page_rows=page, pages=1, tables=1, ld=1)
        gpu.pages_write(d, [[0]], [0], [0, 2], np.zeros((2, hd), np.float32), kv)
        table, lengths = dm.DeviceBuffer.of(np.zeros((1, 1), np.int32)), dm.DeviceBuffer.of(np.array([2], np.int32))
        offsets = dm.DeviceBuffer.of(np.array([0, nq], np.int32))
        d.table = table.ptr
        gpu.pages_attend_dev(d, lengths.ptr, q.b.ptr, offsets.ptr, nq, 1, out.b.ptr)
        gpu.sync()
        want = kv.mean(0)  # scores of 0: both rows alike
        for a in (0, 2**24, 2**26 - 2000, nq - 2000):
            got = out.take(a * hd * 4, (2000, hd))
            assert np.all(np.abs(got - want) <= 2.0**-20 * 32), a
    finally:
        q.b.free()
        out.b.free()


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


def test_many_tables_of_a_row(gpu):
    """65,536 tables of a row each, 8 heads of 64: within the default working memory, of which tiles of 64 rows a table would take 17
    GB. Each query's answer is its row."""
    tables, heads, hd = 65536, 8, 64
    rng = np.random.default_rng(3)
    v = rng.standard_normal((tables, heads * hd)).astype(np.float32)
    at = np.arange(tables + 1, dtype=np.int32)
    before = gpu.work_budget()
    gpu.release()
    gpu.set_work_budget(16 << 30)
    try:
        got = gpu.attend_packed(v[::-1], v, v, at, heads, heads, True)
    finally:
        gpu.set_work_budget(before)
    # A number and its weight in two halves each, off by 2^-11 2^-11 of themselves, and the product of their low halves left out, 2^-11
    # 2^-11: 3 x 2^-22; three products added, a reciprocal (two units) and two products in f32: 7 x 2^-24; 2^-39 of the row's largest
    # (below 8) where a low half is below fp16's normal numbers.
    assert np.all(np.abs(got - v) <= (3 * 2.0**-22 + 7 * 2.0**-24) * np.abs(v) + 2.0**-36)
