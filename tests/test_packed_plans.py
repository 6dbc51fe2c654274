"""Attention of packed tables where its work is divided in each of the ways there are: units of tiles that are a workgroup's each, long
and short, runs of blocks, and both, with more tables than a wavefront has lanes; a sample of queries against 64 bits. `division`
states the rule, so that each case says which way it takes."""
import numpy as np
import pytest

import pages_plain as P
from conftest import pkg
from test_packed import flat, inputs
from test_pages import check, dev, gpu, offsets_of  # noqa: F401 (fixtures)

hip, dm = pkg("hip"), pkg("devmem")
pytestmark = pytest.mark.gpu


def division(q_counts, kv_counts, heads, kv_heads, hd, causal):
    """(units of a head that are a workgroup's each, units of a head, blocks of the longest)"""
    width, tables, nq = (32 if hd <= 32 else 64 if hd <= 64 else 128), len(q_counts), sum(q_counts)
    waves = 8 if (nq // 2048 >= tables if width == 128 else not causal and nq // 4096 >= tables) else 4
    share = 0
    while share < 5 and (heads // kv_heads) % (2 << share) == 0:
        share += 1
    runs, queries, heads = 256 if waves == 8 else 768 if width == 32 else 512, (32 * waves) >> share, heads >> share
    units = sum(-(-n // queries) for n in q_counts)
    blocks = [-(-m // 64) for n, m in zip(q_counts, kv_counts) if n]
    rounds, even = units * heads // runs, not causal and min(blocks) + 1 >= max(blocks)
    own = rounds * runs // heads
    if max(blocks) <= 8 or (not even and rounds >= 2):
        own = units
    return own, units, max(blocks)


def sample(rng, n):
    """Some of n queries, the first and last and those about the borders of tiles and blocks among them."""
    some = {i + d for i in range(0, n, 128) for d in (-1, 0)} | {0, n - 1}
    return sorted({i for i in some if 0 <= i < n and rng.random() < 0.2} | set(rng.integers(0, n, 12).tolist()) | {0, n - 1})


def compare(rng, got, q, k, v, q_counts, kv_counts, causal, what):
    a = b = 0
    outs, offs, gots = [], [], []
    for n, m in zip(q_counts, kv_counts):
        if n:
            some, limits = sample(rng, n), P.limits_of(m, n, causal)
            out, off = P.attention(q[a:a + n][some], k[b:b + m], v[b:b + m], [limits[i] for i in some])
            outs, offs, gots = outs + [out], offs + [off], gots + [got[a:a + n][some]]
        a, b = a + n, b + m
    check(np.concatenate(gots), np.concatenate(outs), np.concatenate(offs), what)


MIXED, WHOLE, RUNS = "units of whole rounds and runs of the rest", "units only", "runs only"
CASES = [
    (MIXED, [4300], [600], 16, 16, 64, False), (MIXED, [4300], [4300], 16, 16, 64, False), (MIXED, [9000], [9000], 8, 1, 64, True),
    (MIXED, [1500] * 6, [1500] * 6, 8, 8, 64, True), (MIXED, [2500, 2300], [1000, 990], 16, 16, 128, False),
    (MIXED, [3] * 130, [641] * 130, 4, 4, 64, False), (MIXED, [40] * 200, [700] * 200, 4, 4, 32, True),
    (MIXED, [9] * 100 + [0] * 40 + [9] * 100, [577] * 240, 3, 3, 128, False),
    (WHOLE, [4000, 1500, 3000, 700], [4000, 1500, 3000, 700], 16, 16, 64, False),
    (WHOLE, [4000, 1500, 3000, 700], [4000, 1500, 3000, 700], 16, 16, 64, True),
    (WHOLE, [4000, 1500, 3000, 700, 9], [4000, 1500, 3000, 700, 2000], 16, 8, 128, True),
    (WHOLE, [600, 40] * 70, [600, 900] * 70, 4, 4, 64, True), (WHOLE, [30] * 150, [10] * 150, 2, 2, 32, False),
    (RUNS, [3, 1] * 35, [641, 5000] * 35, 4, 2, 64, False), (RUNS, [1] * 70 + [0] * 80 + [300], [700] * 150 + [9000], 2, 2, 64, True),
    (RUNS, [2] * 100, [1300] * 100, 2, 1, 128, True), (RUNS, [5] * 300, [600] * 300, 2, 2, 32, False)]


@pytest.mark.parametrize("way,q_counts,kv_counts,heads,kv_heads,hd,causal", CASES, ids=[f"{i}" for i in range(len(CASES))])
def test_ways_of_dividing(gpu, way, q_counts, kv_counts, heads, kv_heads, hd, causal):
    own, units, longest = division(q_counts, kv_counts, heads, kv_heads, hd, causal)
    assert {MIXED: 0 < own < units, WHOLE: own == units, RUNS: own == 0}[way] and (longest > 8 or way == WHOLE)
    rng = np.random.default_rng(units + hd)
    q, k, v = inputs(rng, sum(q_counts), sum(kv_counts), heads, kv_heads, hd)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(q_counts), heads, kv_heads, causal, offsets_of(kv_counts)).reshape(q.shape)
    compare(rng, got, q, k, v, q_counts, kv_counts, causal, f"{way}: {own} of {units} units a head")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ld", [2**22 - 1, 2**22 + 3])
def test_rows_far_apart(gpu, ld, causal):
    """Keys and values 16 MiB from row to row, about where short tables are no longer read where they stand."""
    import ctypes

    rng = np.random.default_rng(ld)
    counts, hd = [40, 27], 64
    n = sum(counts)
    q, k, v = inputs(rng, n, n, 1, 1, hd)
    far = dm.DeviceBuffer(4 * (ld * (n - 1) + 3 * hd))
    qd, of, od = dm.DeviceBuffer.of(flat(q)), dm.DeviceBuffer.of(offsets_of(counts)), dm.DeviceBuffer(q.nbytes)
    try:
        for r in range(n):
            row = np.concatenate([k[r].ravel(), np.full(hd, np.nan, np.float32), v[r].ravel()])
            assert dm.rt().hipMemcpy(ctypes.c_void_p(far.ptr + 4 * ld * r), ctypes.c_void_p(row.ctypes.data), ctypes.c_size_t(row.nbytes), 1) == 0
        gpu.attend_packed_dev(qd.ptr, far.ptr, far.ptr + 8 * hd, of.ptr, of.ptr, 2, n, n, 1, 1, hd, od.ptr, causal, 0, ld)
        gpu.sync()
        compare(rng, od.download(q.shape), q, k, v, counts, counts, causal, f"{ld} floats apart, causal {causal}")
    finally:
        for b in (far, qd, of, od):
            b.free()
