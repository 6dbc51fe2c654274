"""Rows of many tables into pages and back, bit for bit, and attention over the pages within the sum of its worst roundings, against
the statements in `pages_plain`."""
import ctypes

import numpy as np
import pytest

import pages_plain as P
from conftest import pkg

abi, hip, dm = pkg("abi"), pkg("hip"), pkg("devmem")
pytestmark = pytest.mark.gpu
FORMATS = [abi.KV_F32, abi.KV_I16, abi.KV_I8]


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


def described(pool, tables, ld, pool_ptr, table_ptr=0):
    return abi.Pages(pool=pool_ptr, table=table_ptr, kv_format=pool.fmt, kv_heads=pool.heads, hd=pool.hd, page_rows=pool.rows,
                     pages=pool.pages, tables=tables, ld=ld)


def tables_of(rng, lengths, rows, extra=2, ld=None):
    """Pages anywhere in a pool for tables of these lengths: (table [tables][ld], pages)."""
    need = [-(-n // rows) for n in lengths]
    ld = ld or max(1, max(need))
    total = sum(need) + extra
    order = rng.permutation(total).astype(np.int32)
    table, at = np.full((len(lengths), ld), -1, np.int32), 0
    for t, n in enumerate(need):
        table[t, :n] = order[at:at + n]
        at += n
    return table, total


def values(rng, n, heads, hd, scale=0.55):
    return (rng.standard_normal((n, heads, hd)) * scale + rng.standard_normal((heads, hd)) * 0.3).astype(np.float32)


def offsets_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


class Device:
    """Arrays on the card, freed together."""

    def __init__(self):
        self.held = []

    def of(self, a):
        b = dm.DeviceBuffer.of(np.ascontiguousarray(a))
        self.held.append(b)
        return b

    def free(self):
        for b in self.held:
            b.free()


@pytest.fixture
def dev():
    d = Device()
    yield d
    d.free()


# ---- rows into pages and back ---------------------------------------------------------------------------------------------
COUNTS = [(1, 0), (0, 5), (15, 1), (16, 0), (17, 7), (64, 61), (65, 3), (130, 200), (0, 0), (333, 15)]  # rows, where they begin


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,hd", [(16, 1, 16), (32, 3, 48), (64, 8, 64), (128, 2, 128), (256, 5, 80)])
def test_rows_are_stored_and_read(gpu, dev, fmt, rows, heads, hd):
    rng = np.random.default_rng(fmt * 100 + rows)
    lengths = [s + n for n, s in COUNTS]
    table, pages = tables_of(rng, lengths, rows)
    pool = P.Pool(fmt, heads, hd, rows, pages, fill=0xA5)
    card = dev.of(pool.bytes)
    counts, starts = [n for n, _ in COUNTS], [s for _, s in COUNTS]
    offsets = offsets_of(counts)
    n = int(offsets[-1])
    k, v = values(rng, n, heads, hd), values(rng, n, heads, hd, 3.0)
    k[0], v[min(5, n - 1)] = 0.0, 1e-41  # rows of nothing, and of steps too small
    k[1, 0, 3], k[1, 0, 5], v[2, 0, 0], v[2, 0, 1] = np.nan, np.inf, -np.inf, np.nan
    k[3] *= 1e37
    d = described(pool, len(COUNTS), table.shape[1], card.ptr)
    gpu.pages_write(d, table, starts, offsets, k.reshape(n, -1), v.reshape(n, -1))
    for t in range(len(COUNTS)):
        for i in range(counts[t]):
            at = starts[t] + i
            pool.write(table[t, at // rows], at % rows, k[offsets[t] + i], v[offsets[t] + i])
    got = card.download(pool.bytes.shape, np.uint8)
    assert np.array_equal(got, pool.bytes)
    gk, gv = gpu.pages_read(d, table, starts, offsets)
    for t in range(len(COUNTS)):
        for i in range(counts[t]):
            at, r = starts[t] + i, offsets[t] + i
            wk, wv = pool.read(table[t, at // rows], at % rows)
            assert np.array_equal(gk[r].reshape(heads, hd), wk.astype(np.float32), equal_nan=True)
            assert np.array_equal(gv[r].reshape(heads, hd), wv.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("fmt", [abi.KV_I16, abi.KV_I8])
def test_ties_and_their_neighbours(gpu, dev, fmt):
    """Numbers whose quotient by the step is a half, and the floats next to it, where a product with 1 / step would round over."""
    top, hd, rng = P.TOP[fmt], 128, np.random.default_rng(3)
    n = 64
    k = np.zeros((n, 1, hd), np.float32)
    for r in range(n):
        big = np.float32(rng.uniform(0.5, 2.0) * 2.0 ** int(rng.integers(-20, 20)))
        s = np.float32(big / np.float32(top))
        c = rng.integers(0, top, hd) + 0.5
        x = (c * np.float64(s)).astype(np.float32)
        x[1::3], x[2::3] = np.nextafter(x[1::3], np.float32(0)), np.nextafter(x[2::3], np.float32(np.inf))
        x *= rng.choice([-1, 1], hd).astype(np.float32)
        x[r % hd] = big
        k[r, 0] = np.clip(x, -big, big)
    pool = P.Pool(fmt, 1, hd, 64, 1)
    card = dev.of(pool.bytes)
    d = described(pool, 1, 1, card.ptr)
    gpu.pages_write(d, [[0]], [0], [0, n], k.reshape(n, hd), -k.reshape(n, hd))
    for r in range(n):
        pool.write(0, r, k[r], -k[r])
    assert np.array_equal(card.download(pool.bytes.shape, np.uint8), pool.bytes)


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_on_no_page_and_behind_the_last(gpu, dev, fmt):
    """On device memory: ids outside the pool, rows outside their table's pages, negative starts and rows past the last table are
    left alone; rows on no page are read as zeros; rows far apart."""
    rng = np.random.default_rng(8 + fmt)
    heads, hd, rows, ld = 2, 32, 16, 3
    pool = P.Pool(fmt, heads, hd, rows, 4, fill=0x33)
    table = np.array([[2, -1, 1], [7, 0, 3], [4, 2**31 - 1, -2**31]], np.int32)
    starts, offsets = np.array([-3, 10, 0], np.int32), np.array([0, 60, 110, 120], np.int32)
    n, total, far = 120, 131, heads * hd + 5
    k, v = np.zeros((total, far), np.float32), np.zeros((total, far), np.float32)
    k[:, :heads * hd], v[:, :heads * hd] = rng.standard_normal((2, total, heads * hd)).astype(np.float32)
    card, tb, st, of = dev.of(pool.bytes), dev.of(table), dev.of(starts), dev.of(offsets)
    kd, vd = dev.of(k), dev.of(v)
    d = described(pool, 3, ld, card.ptr, tb.ptr)
    gpu.pages_write_dev(d, st.ptr, of.ptr, kd.ptr, vd.ptr, total, far)
    gpu.sync()
    on = {}
    for t in range(3):
        for r in range(offsets[t], offsets[t + 1]):
            at = int(starts[t]) + r - int(offsets[t])
            if 0 <= at < ld * rows and 0 <= table[t, at // rows] < 4:
                on[r] = (table[t, at // rows], at % rows)
                pool.write(*on[r], k[r, :heads * hd].reshape(heads, hd), v[r, :heads * hd].reshape(heads, hd))
    assert np.array_equal(card.download(pool.bytes.shape, np.uint8), pool.bytes)
    ko, vo = dev.of(np.full((total, far), 7.0, np.float32)), dev.of(np.full((total, far), 7.0, np.float32))
    gpu.pages_read_dev(d, st.ptr, of.ptr, ko.ptr, vo.ptr, total, far)
    gpu.sync()
    gk, gv = ko.download((total, far)), vo.download((total, far))
    assert np.all(gk[n:] == 7.0) and np.all(gv[n:] == 7.0)
    assert np.all(gk[:, heads * hd:] == 7.0) and np.all(gv[:, heads * hd:] == 7.0)
    for r in range(n):
        wk, wv = pool.read(*on[r]) if r in on else (np.zeros((heads, hd)), np.zeros((heads, hd)))
        assert np.array_equal(gk[r, :heads * hd].reshape(heads, hd), wk.astype(np.float32))
        assert np.array_equal(gv[r, :heads * hd].reshape(heads, hd), wv.astype(np.float32))


def test_many_tables_of_a_row_each(gpu, dev):
    """More tables than a workgroup keeps in LDS, every third without a row."""
    rng = np.random.default_rng(5)
    T, heads, hd, rows = 2500, 1, 16, 16
    counts = [0 if t % 3 == 0 else 1 for t in range(T)]
    starts = rng.integers(0, rows, T).astype(np.int32)
    table = np.arange(T, dtype=np.int32)[:, None]
    offsets = offsets_of(counts)
    n = int(offsets[-1])
    pool = P.Pool(abi.KV_I8, heads, hd, rows, T)
    card = dev.of(pool.bytes)
    k, v = values(rng, n, heads, hd), values(rng, n, heads, hd)
    d = described(pool, T, 1, card.ptr)
    gpu.pages_write(d, table, starts, offsets, k.reshape(n, -1), v.reshape(n, -1))
    for t in range(T):
        if counts[t]:
            pool.write(t, starts[t], k[offsets[t]], v[offsets[t]])
    assert np.array_equal(card.download(pool.bytes.shape, np.uint8), pool.bytes)


# ---- attention over pages -------------------------------------------------------------------------------------------------
def filled(rng, fmt, heads, hd, rows, lengths, scale=0.55, garbage=0xFF):
    """A pool with tables of random rows; what no table holds is garbage (NaN in f32 and in steps)."""
    table, pages = tables_of(rng, lengths, rows)
    pool = P.Pool(fmt, heads, hd, rows, pages, fill=garbage)
    for t, n in enumerate(lengths):
        k, v = values(rng, n, heads, hd, scale), values(rng, n, heads, hd, scale)
        for i in range(n):
            pool.write(table[t, i // rows], i % rows, k[i], v[i])
    return pool, table


def wanted(pool, table, lengths, q, counts, causal):
    """The outputs and how far off they may be, queries of all tables."""
    out, off, at = np.zeros(q.shape), np.zeros(q.shape), 0
    for t, n in enumerate(counts):
        k, v = pool.rows_of(table[t], lengths[t])
        out[at:at + n], off[at:at + n] = P.attention(q[at:at + n], k, v, P.limits_of(lengths[t], n, causal))
        at += n
    return out, off


def check(got, out, off, what, rms=2.0**-20):
    """Every output within its worst roundings, and all of them together (roundings being of either sign, the terms' 2^-22 add up
    to about as much of their sum) within 2^-20 of their root mean square: a query, weight, key or value in one half would be
    2^-13 off."""
    size = lambda a: np.sqrt(np.mean(np.square(a)))
    worst, mean = np.max(np.abs(got - out) / np.maximum(off, 1e-30)), size(got - out) / max(size(out), 1e-30)
    say(f"{what}: worst error {np.abs(got - out).max():.2e}, {worst:.3f} of what it may be, root mean square {mean:.1e}")
    assert np.all(np.isfinite(got)) and np.all(np.abs(got - out) <= off) and mean <= rms


LENGTHS = [0, 1, 15, 16, 17, 63, 64, 65, 300, 1111]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,kv_heads,group,hd,new,causal", [
    (64, 8, 1, 64, 1, False), (16, 2, 4, 64, 1, True), (16, 1, 8, 128, 3, True), (256, 2, 2, 128, 9, False), (32, 3, 1, 48, 2, True),
    (128, 1, 3, 16, 17, True), (16, 4, 1, 80, 1, False), (64, 2, 1, 64, 40, True), (128, 1, 16, 64, 2, False)])
def test_attention_over_pages(gpu, dev, fmt, rows, kv_heads, group, hd, new, causal):
    rng = np.random.default_rng(fmt + rows + hd + new)
    pool, table = filled(rng, fmt, kv_heads, hd, rows, LENGTHS)
    counts = [max(0, new - i % 3) for i in range(len(LENGTHS))]
    heads, n = kv_heads * group, sum(counts)
    q = (rng.standard_normal((n, heads, hd)) * 0.4).astype(np.float32)
    card = dev.of(pool.bytes)
    d = described(pool, len(LENGTHS), table.shape[1], card.ptr)
    got = gpu.pages_attend(d, table, LENGTHS, q.reshape(n, -1), offsets_of(counts), heads, causal).reshape(q.shape)
    out, off = wanted(pool, table, LENGTHS, q, counts, causal)
    check(got, out, off, f"format {fmt}, pages of {rows}, {heads}/{kv_heads} heads of {hd}, {new} queries")


@pytest.mark.parametrize("fmt,length", [(abi.KV_I8, 40000), (abi.KV_I16, 30001), (abi.KV_F32, 20011)])
def test_one_long_table_and_many_short(gpu, dev, fmt, length):
    """Rows that many workgroups share, units that end inside a wavefront's run, and short ones between."""
    rng = np.random.default_rng(length)
    lengths = [5, length, 70, 0, 700, 1, 3000]
    pool, table = filled(rng, fmt, 1, 64, 64, lengths)
    counts, heads = [1, 2, 1, 1, 3, 1, 1], 2
    q = (rng.standard_normal((sum(counts), heads, 64)) * 0.4).astype(np.float32)
    card = dev.of(pool.bytes)
    d = described(pool, len(lengths), table.shape[1], card.ptr)
    got = gpu.pages_attend(d, table, lengths, q.reshape(len(q), -1), offsets_of(counts), heads).reshape(q.shape)
    check(got, *wanted(pool, table, lengths, q, counts, False), f"format {fmt}, a table of {length}")


@pytest.mark.parametrize("fmt", FORMATS)
def test_magnitudes(gpu, dev, fmt):
    """Keys, values and queries far from 1, rows a million times larger than others, a certain row among many."""
    rng = np.random.default_rng(40 + fmt)
    lengths = [200, 200, 200, 200]
    pool, table = filled(rng, fmt, 1, 64, 32, lengths)
    for t, (sk, sv) in enumerate([(1e-12, 1e12), (1e9, 1e-20), (1.0, 1e6), (30.0, 1.0)]):
        for i in range(200):
            k, v = (rng.standard_normal((2, 1, 64)) * 0.5).astype(np.float32)
            big = 1e6 if t == 2 and i % 50 == 7 else 1.0
            pool.write(table[t, i // 32], i % 32, (k * sk).astype(np.float32), (v * sv / 1e6 * big).astype(np.float32))
    q = (rng.standard_normal((4, 1, 64)) * 0.4).astype(np.float32)
    q[0] *= 1e12
    q[1] *= 1e-9
    card = dev.of(pool.bytes)
    d = described(pool, 4, table.shape[1], card.ptr)
    got = gpu.pages_attend(d, table, lengths, q.reshape(4, -1), [0, 1, 2, 3, 4], 1).reshape(q.shape)
    check(got, *wanted(pool, table, lengths, q, [1] * 4, False), f"format {fmt}, magnitudes", 2.0**-16)  # scores up to 100


def test_numbers_that_are_not_finite(gpu, dev):
    """f32 pages: a key or value that is not finite makes NaN of the queries that see it, a value of its coordinate alone, and
    nothing of the queries before it, of other tables or of rows behind a table's end."""
    rng = np.random.default_rng(77)
    rows, hd, n = 16, 64, 70
    for where, kind in [(65, "value"), (65, "key"), (3, "value"), (200, "value"), (200, "key")]:
        pool, table = filled(rng, abi.KV_F32, 1, hd, rows, [n + 250, 90])
        length = n  # rows from here on are another time's
        page, slot = table[0, where // rows], where % rows
        bad = np.float32(np.inf if where == 65 else np.nan)
        if kind == "value":
            pool.values[page, 0, 5, slot] = bad
        else:
            pool.keys[page, 0, slot, 9] = bad
        q = (rng.standard_normal((12, 2, hd)) * 0.4).astype(np.float32)
        card = dev.of(pool.bytes)
        d = described(pool, 2, table.shape[1], card.ptr)
        got = gpu.pages_attend(d, table, [length, 90], q.reshape(12, -1), [0, 10, 12], 2, True).reshape(q.shape)
        clean = P.Pool(abi.KV_F32, 1, hd, rows, pool.pages)
        clean.bytes[:] = pool.bytes
        (clean.values[page, 0] if kind == "value" else clean.keys[page, 0].T)[:, slot] = 0.25
        out, off = wanted(clean, table, [length, 90], q, [10, 2], True)
        sees = np.zeros(q.shape, bool)
        for i, lim in enumerate(P.limits_of(length, 10, True)):
            if where < lim:
                sees[i, :, 5 if kind == "value" else slice(None)] = True
        assert np.all(np.isnan(got[sees])), (where, kind)
        blind = np.ones(q.shape, bool)
        blind[:10] = np.array([where >= lim for lim in P.limits_of(length, 10, True)])[:, None, None]
        say(f"{kind} {bad} at row {where}: {int(sees.sum())} outputs see it")
        assert np.all(np.abs(got[blind] - out[blind]) <= off[blind]), (where, kind)
        if kind == "value":
            others = ~sees & ~blind  # the other coordinates: as ever
            if where < length:
                full = P.Pool(abi.KV_F32, 1, hd, rows, pool.pages)
                full.bytes[:] = pool.bytes
                full.values[page, 0, 5, slot] = 0.25
                out, off = wanted(full, table, [length, 90], q, [10, 2], True)
                assert np.all(np.abs(got[others] - out[others]) <= off[others])


def test_a_query_that_is_not_finite_is_alone(gpu, dev):
    rng = np.random.default_rng(12)
    pool, table = filled(rng, abi.KV_I8, 2, 64, 64, [100, 300])
    q = (rng.standard_normal((5, 4, 64)) * 0.4).astype(np.float32)
    q[1, 2, 7], q[3, 0, 0] = np.nan, np.inf
    card = dev.of(pool.bytes)
    d = described(pool, 2, table.shape[1], card.ptr)
    got = gpu.pages_attend(d, table, [100, 300], q.reshape(5, -1), [0, 2, 5], 4).reshape(q.shape)
    bad = np.zeros((5, 4), bool)
    bad[1, 2] = bad[3, 0] = True
    assert np.all(np.isnan(got[bad]))
    out, off = wanted(pool, table, [100, 300], np.where(np.isfinite(q), q, 0).astype(np.float32), [2, 3], False)
    assert np.all(np.abs(got - out)[~bad] <= off[~bad])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [16, 128])
def test_missing_pages_lengths_and_spare_queries_on_device_memory(gpu, dev, fmt, rows):
    """Rows on no page are not seen, lengths past the table's pages count as the pages, negative ones as none; pages shared by
    two tables; queries far apart; queries past the last table's are left as they were."""
    rng = np.random.default_rng(fmt + rows)
    kv_heads, heads, hd = 2, 4, 64
    lengths = [300, 300, 40, 256]
    pool, table = filled(rng, fmt, kv_heads, hd, rows, lengths)
    table[1, 0] = table[0, 0]  # shared
    table[0, 1] = pool.pages + 5
    if table.shape[1] > 2:
        table[3, 2] = -7
    told = np.array([300, 300, -4, 10**9], np.int32)
    counts, far = [2, 1, 1, 3], heads * hd + 3
    n = sum(counts) + 4
    q = np.zeros((n, far), np.float32)
    q[:, :heads * hd] = rng.standard_normal((n, heads * hd)) * 0.4
    card, tb, ln, of, qd = dev.of(pool.bytes), dev.of(table), dev.of(told), dev.of(offsets_of(counts)), dev.of(q)
    od = dev.of(np.full((n, heads * hd), 5.0, np.float32))
    d = described(pool, 4, table.shape[1], card.ptr, tb.ptr)
    gpu.pages_attend_dev(d, ln.ptr, qd.ptr, of.ptr, n, heads, od.ptr, False, far)
    gpu.sync()
    got = od.download((n, heads, hd))
    assert np.all(got[sum(counts):] == 5.0)
    at = 0
    for t, c in enumerate(counts):
        length = min(max(int(told[t]), 0), table.shape[1] * rows)
        there = [i for i in range(length) if 0 <= table[t, i // rows] < pool.pages]
        qs = q[at:at + c, :heads * hd].reshape(c, heads, hd)
        k = np.stack([pool.read(table[t, i // rows], i % rows)[0] for i in there]) if there else np.zeros((0, kv_heads, hd))
        v = np.stack([pool.read(table[t, i // rows], i % rows)[1] for i in there]) if there else np.zeros((0, kv_heads, hd))
        out, off = P.attention(qs, k, v, [len(there)] * c)
        check(got[at:at + c], out, off, f"table {t}")
        at += c


def test_a_pool_past_four_gigabytes(gpu, dev):
    """The last pages of a pool of 4.5 GB: offsets past 32 bits, written, read and attended."""
    rng = np.random.default_rng(6)
    heads, hd, rows = 8, 128, 256
    size = abi.page_bytes(abi.KV_F32, heads, hd, rows)
    pages = 4608 * 2**20 // size
    card = dm.DeviceBuffer(pages * size)
    dev.held.append(card)
    table = np.array([[pages - 1, pages - 3]], np.int32)
    n = 300
    k, v = values(rng, n, heads, hd), values(rng, n, heads, hd)
    d = abi.Pages(pool=card.ptr, kv_format=abi.KV_F32, kv_heads=heads, hd=hd, page_rows=rows, pages=pages, tables=1, ld=2)
    gpu.pages_write(d, table, [0], [0, n], k.reshape(n, -1), v.reshape(n, -1))
    gk, gv = gpu.pages_read(d, table, [0], [0, n])
    assert np.array_equal(gk, k.reshape(n, -1)) and np.array_equal(gv, v.reshape(n, -1))
    q = (rng.standard_normal((2, heads, hd)) * 0.3).astype(np.float32)
    got = gpu.pages_attend(d, table, [n], q.reshape(2, -1), [0, 2], heads).reshape(q.shape)
    check(got, *P.attention(q, k, v, [n, n]), "behind 4 GB")


# ---- captured, and from two handles ------------------------------------------------------------------------------------------
class Graph:
    """What `work` queues on the handle's stream, captured."""

    def __init__(self, gpu, work):
        rt, vp = dm.rt(), ctypes.c_void_p
        self.rt, self.stream = rt, vp(gpu.stream)
        graph, self.exec = vp(), vp()
        assert rt.hipStreamBeginCapture(self.stream, ctypes.c_int(1)) == 0
        try:
            work()
        finally:
            rc = rt.hipStreamEndCapture(self.stream, ctypes.byref(graph))
        assert rc == 0
        assert rt.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)) == 0
        assert rt.hipGraphDestroy(graph) == 0

    def replay(self):
        assert self.rt.hipGraphLaunch(self.exec, self.stream) == 0

    def free(self):
        assert self.rt.hipGraphExecDestroy(self.exec) == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_tables_grow_in_a_captured_step(gpu, dev, fmt):
    """A serving step captured once: a new row written into each table, its query answered over the row and those before it. Replayed as the
    tables grow (the starts and lengths change on the card), with eager calls between, and checked against the
    eager calls bit for bit, and against 64 bits."""
    rng = np.random.default_rng(fmt)
    kv_heads, heads, hd, rows, T = 2, 4, 64, 16, 5
    lengths = np.array([0, 15, 16, 100, 333], np.int32)
    steps = 4
    pool, table = filled(rng, fmt, kv_heads, hd, rows, list(lengths + steps))
    card, tb, of = dev.of(pool.bytes), dev.of(table), dev.of(offsets_of([1] * T))
    st, ln = dev.of(lengths), dev.of(lengths)
    zero = np.zeros((T, kv_heads * hd), np.float32)
    kd, vd, qd = dev.of(zero), dev.of(zero), dev.of(np.zeros((T, heads * hd), np.float32))
    od, oe = dev.of(np.zeros((T, heads * hd), np.float32)), dev.of(np.zeros((T, heads * hd), np.float32))
    d = described(pool, T, table.shape[1], card.ptr, tb.ptr)

    def step(out):
        gpu.pages_write_dev(d, st.ptr, of.ptr, kd.ptr, vd.ptr, T)
        gpu.pages_attend_dev(d, ln.ptr, qd.ptr, of.ptr, T, heads, out.ptr, True)

    step(od)
    gpu.sync()
    card.upload(pool.bytes)
    g = Graph(gpu, lambda: step(od))
    try:
        for i in range(steps):
            k, v = values(rng, T, kv_heads, hd), values(rng, T, kv_heads, hd)
            q = (rng.standard_normal((T, heads, hd)) * 0.4).astype(np.float32)
            for b, a in ((kd, k), (vd, v), (qd, q), (st, lengths + i), (ln, lengths + i + 1)):
                b.upload(a)
            g.replay()
            gpu.sync()
            got = od.download((T, heads, hd))
            for t in range(T):
                at = lengths[t] + i
                pool.write(table[t, at // rows], at % rows, k[t], v[t])
            assert np.array_equal(card.download(pool.bytes.shape, np.uint8), pool.bytes)
            step(oe)
            gpu.sync()
            assert np.array_equal(oe.download((T, heads, hd)), got)
            check(got, *wanted(pool, table, lengths + i + 1, q, [1] * T, True), f"step {i}")
    finally:
        g.free()


def test_two_handles_give_the_same(gpu, dev):
    rng = np.random.default_rng(31)
    pool, table = filled(rng, abi.KV_I8, 8, 64, 64, [700, 1200, 30])
    q = (rng.standard_normal((3, 8, 64)) * 0.4).astype(np.float32)
    card = dev.of(pool.bytes)
    d = described(pool, 3, table.shape[1], card.ptr)
    other = hip.Gpu(0)
    try:
        a = gpu.pages_attend(d, table, [700, 1200, 30], q.reshape(3, -1), [0, 1, 2, 3], 8)
        b = other.pages_attend(d, table, [700, 1200, 30], q.reshape(3, -1), [0, 1, 2, 3], 8)
    finally:
        other.close()
    assert np.array_equal(a, b)
    assert np.array_equal(a, gpu.pages_attend(d, table, [700, 1200, 30], q.reshape(3, -1), [0, 1, 2, 3], 8))


# ---- refusals -----------------------------------------------------------------------------------------------------------------
def test_refusals(gpu, dev):
    pool = P.Pool(abi.KV_I8, 2, 64, 64, 4)
    card = dev.of(pool.bytes)
    table = np.array([[0, 1], [2, 3]], np.int32)
    good = described(pool, 2, 2, card.ptr)
    k = np.zeros((3, 128), np.float32)
    q = np.zeros((2, 256), np.float32)
    write = lambda d=good, table=table, starts=(0, 0), offsets=(0, 2, 3), k=k, v=k: gpu.pages_write(d, table, starts, offsets, k, v)
    attend = lambda d=good, table=table, lengths=(5, 128), q=q, offsets=(0, 1, 2), heads=4: gpu.pages_attend(d, table, lengths, q,
                                                                                                        offsets, heads)
    write(), attend()

    def other(**kw):
        d = abi.Pages.from_buffer_copy(good)
        for name, value in kw.items():
            setattr(d, name, value)
        return d

    bad = [dict(kv_format=abi.KV_I4), dict(kv_format=-1), dict(kv_format=9), dict(page_rows=0), dict(page_rows=48), dict(page_rows=8),
           dict(page_rows=512), dict(pool=None), dict(pool=card.ptr + 8), dict(pages=0), dict(pages=-1)]
    for kw in bad:
        for call in (write, attend):
            with pytest.raises(ValueError):
                call(d=other(**kw))
    for hd in (0, 8, 24, 72, 136, 144, -16):
        width = max(0, 2 * hd)
        with pytest.raises(ValueError):
            gpu.pages_write(other(hd=hd), table, (0, 0), (0, 2, 3), np.zeros((3, width), np.float32), np.zeros((3, width), np.float32))
    for kw in [dict(starts=(-1, 0)), dict(starts=(127, 0)), dict(starts=(0, 128)), dict(offsets=(1, 2, 3)), dict(offsets=(0, 3, 2)),
               dict(offsets=(0, 2, 4)), dict(offsets=(0, 2)), dict(starts=(0,)), dict(starts=(0.5, 0)), dict(table=table[:1]),
               dict(table=np.array([[0, 1], [4, 3]])), dict(table=np.array([[0, 1], [-1, 3]])), dict(k=k[:, :-1], v=k[:, :-1]),
               dict(k=k[:2]), dict(starts=(0, 2**40)), dict(table=np.array([[0, 1], [0, 3]]), starts=(0, 1))]:
        with pytest.raises(ValueError):
            write(**kw)
    for kw in [dict(lengths=(-1, 3)), dict(lengths=(129, 3)), dict(lengths=(1, 2, 3)), dict(heads=3), dict(heads=0), dict(heads=1),
               dict(offsets=(0, 2, 1)), dict(offsets=(0, 1, 3)), dict(table=np.array([[9, 1], [2, 3]])), dict(q=q[:, 1:])]:
        with pytest.raises(ValueError):
            attend(**kw)
    with pytest.raises(ValueError):
        gpu.pages_read(good, np.array([[0, 1], [-1, 3]]), (0, 0), (0, 2, 3))
    # on device memory: pointers, strides and sizes
    of, st = dev.of(np.array([0, 2, 3], np.int32)), dev.of(np.zeros(2, np.int32))
    kd, tb = dev.of(k), dev.of(table)
    on_card = other(table=tb.ptr)
    gpu.pages_write_dev(on_card, st.ptr, of.ptr, kd.ptr, kd.ptr, 3)
    for args in [(good, st.ptr, of.ptr, kd.ptr, kd.ptr, 3), (on_card, 0, of.ptr, kd.ptr, kd.ptr, 3), (on_card, st.ptr, 0, kd.ptr, kd.ptr, 3),
                 (on_card, st.ptr, of.ptr, kd.ptr + 2, kd.ptr, 3), (on_card, st.ptr, of.ptr, kd.ptr, 0, 3), (on_card, st.ptr, of.ptr, kd.ptr, kd.ptr, -1),
                 (on_card, st.ptr, of.ptr, kd.ptr, kd.ptr, 3, 127), (on_card, st.ptr, of.ptr, kd.ptr, kd.ptr, 2**31 - 1)]:
        with pytest.raises(ValueError):
            gpu.pages_write_dev(*args)
        with pytest.raises(ValueError):
            gpu.pages_read_dev(*args)
    qd = dev.of(q)
    for args in [(good, st.ptr, qd.ptr, of.ptr, 2, 4, qd.ptr), (on_card, st.ptr, qd.ptr, of.ptr, 2, 3, qd.ptr),
                 (on_card, st.ptr, qd.ptr + 1, of.ptr, 2, 4, qd.ptr), (on_card, st.ptr, qd.ptr, of.ptr, -2, 4, qd.ptr),
                 (on_card, st.ptr, qd.ptr, of.ptr, 2, 4, qd.ptr, False, 255), (on_card, st.ptr, qd.ptr, of.ptr, 2**30, 4, qd.ptr),
                 (other(table=tb.ptr, tables=2**24, ld=2**20), st.ptr, qd.ptr, of.ptr, 2**28, 4, qd.ptr)]:
        with pytest.raises(ValueError):
            gpu.pages_attend_dev(*args)
    gpu.sync()


def test_page_sizes():
    l = abi.lib()
    for fmt in FORMATS:
        for heads, hd, rows in ((1, 16, 16), (8, 64, 64), (3, 128, 256), (2, 48, 32)):
            assert l.tah_page_bytes(fmt, heads, hd, rows) == abi.page_bytes(fmt, heads, hd, rows)
    assert l.tah_page_bytes(abi.KV_I8, 8, 64, 64) == 8 * (2 * 64 * 64 + 2 * 64 * 4)
    for args in ((abi.KV_I4, 8, 64, 64), (0, 0, 64, 64), (0, 8, 60, 64), (0, 8, 64, 24), (0, 8, 144, 64), (7, 8, 64, 64)):
        assert l.tah_page_bytes(*args) == 0
