"""Attention of packed tables in full precision against 64 bits, within the sum of its worst roundings and, together, to f32's
precision (`pages_plain.attention`)."""
import numpy as np
import pytest

import pages_plain as P
from conftest import pkg
from test_pages import Device, Graph, check, offsets_of, say, values

abi, hip, dm = pkg("abi"), pkg("hip"), pkg("devmem")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


@pytest.fixture
def dev():
    d = Device()
    yield d
    d.free()


def wanted(q, k, v, q_counts, kv_counts, causal):
    out, off, a, b = np.zeros(q.shape), np.zeros(q.shape), 0, 0
    for n, m in zip(q_counts, kv_counts):
        out[a:a + n], off[a:a + n] = P.attention(q[a:a + n], k[b:b + m], v[b:b + m], P.limits_of(m, n, causal))
        a, b = a + n, b + m
    return out, off


def inputs(rng, n, m, heads, kv_heads, hd):
    return ((rng.standard_normal((n, heads, hd)) * 0.4).astype(np.float32), values(rng, m, kv_heads, hd), values(rng, m, kv_heads, hd))


def flat(a):
    return a.reshape(len(a), -1)


SHORT = [1, 0, 31, 32, 33, 63, 64, 65, 127, 129, 200]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kv_heads,group,hd", [(8, 1, 64), (2, 4, 64), (1, 3, 16), (3, 1, 48), (1, 2, 128), (2, 1, 80), (1, 8, 32)])
def test_tables_of_all_lengths(gpu, kv_heads, group, hd, causal):
    rng = np.random.default_rng(hd + group)
    n, heads = sum(SHORT), kv_heads * group
    q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(SHORT), heads, kv_heads, causal).reshape(q.shape)
    check(got, *wanted(q, k, v, SHORT, SHORT, causal), f"{heads}/{kv_heads} heads of {hd}, causal {causal}")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_tables(gpu, hd, causal):
    rng = np.random.default_rng(hd)
    counts = [700, 5, 1300]
    q, k, v = inputs(rng, sum(counts), sum(counts), 2, 1, hd)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), 2, 1, causal).reshape(q.shape)
    check(got, *wanted(q, k, v, counts, counts, causal), f"heads of {hd}, causal {causal}")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd", [(6, 1, 32), (12, 2, 64), (16, 1, 64), (32, 1, 16), (64, 1, 32), (24, 3, 128), (7, 1, 48)])
def test_heads_that_share_keys(gpu, heads, kv_heads, hd, causal):
    """Groups of every kind (odd, even, more than a wavefront's columns), tables short and long enough to be cut, more queries than
    rows and fewer."""
    rng = np.random.default_rng(heads)
    q_counts, kv_counts = [900, 3, 0, 41, 130, 17], [900, 3, 5, 700, 60, 17]
    q, k, v = inputs(rng, sum(q_counts), sum(kv_counts), heads, kv_heads, hd)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(q_counts), heads, kv_heads, causal, offsets_of(kv_counts)).reshape(q.shape)
    check(got, *wanted(q, k, v, q_counts, kv_counts, causal), f"{heads}/{kv_heads} heads of {hd}, causal {causal}")


@pytest.mark.parametrize("hd,rows,causal", [(32, 4300, False), (64, 4300, False), (128, 2300, False), (128, 2300, True)])
def test_one_long_table(gpu, hd, rows, causal):
    """Long enough alone for the larger tiles of queries, not long enough with another."""
    rng = np.random.default_rng(rows)
    for counts in ([rows], [3, rows - 40]):
        n = sum(counts)
        q, k, v = inputs(rng, n, n, 2, 1, hd)
        got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), 2, 1, causal).reshape(q.shape)
        check(got, *wanted(q, k, v, counts, counts, causal), f"{counts} rows, heads of {hd}, causal {causal}")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_counts,kv_counts", [
    ([1], [5000]), ([3, 0, 2], [0, 100, 4000]), ([10, 20, 1], [4, 20, 0]), ([40, 300], [1000, 299]), ([1, 1, 1, 1], [64, 128, 1, 63])])
def test_queries_and_rows_of_different_counts(gpu, q_counts, kv_counts, causal):
    """Few queries over many rows (several key ranges joined), queries before a table's first row, tables without queries or
    without rows."""
    rng = np.random.default_rng(sum(q_counts))
    q, k, v = inputs(rng, sum(q_counts), sum(kv_counts), 4, 2, 64)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(q_counts), 4, 2, causal, offsets_of(kv_counts)).reshape(q.shape)
    out, off = wanted(q, k, v, q_counts, kv_counts, causal)
    check(got, out, off, f"{q_counts} over {kv_counts}, causal {causal}")
    assert not np.any(got[np.all(out == 0, axis=(1, 2))])


def test_no_rows_at_all(gpu):
    q = np.ones((3, 128), np.float32)
    none = np.zeros((0, 128), np.float32)
    assert not np.any(gpu.attend_packed(q, none, none, [0, 1, 3], 2, 2, False, [0, 0, 0]))
    assert gpu.attend_packed(none, q, q, [0, 0], 2, 2, True, [0, 3]).shape == (0, 128)


@pytest.mark.parametrize("causal", [False, True])
def test_magnitudes(gpu, causal):
    """Tables, blocks and rows of very different sizes side by side: none takes another's precision."""
    rng = np.random.default_rng(2)
    counts = [150, 150, 150, 300]
    q, k, v = inputs(rng, 750, 750, 2, 1, 64)
    q[:150], k[:150] = q[:150] * np.float32(1e10), k[:150] * np.float32(1e-10)
    v[:150] *= np.float32(1e-25)
    q[150:300], k[150:300] = q[150:300] * np.float32(1e-18), k[150:300] * np.float32(1e18)
    v[150:300] *= np.float32(1e25)
    v[450:514] *= np.float32(1e-30)  # a block of tiny values before, and one of large ones behind it
    v[578:642] *= np.float32(1e6)
    k[700:] *= np.float32(1e-8)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), 2, 1, causal).reshape(q.shape)
    out, off = wanted(q, k, v, counts, counts, causal)
    at = 0
    for n in counts:
        check(got[at:at + n], out[at:at + n], off[at:at + n], f"rows {at} to {at + n}")
        at += n


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["value", "key", "query"])
def test_numbers_that_are_not_finite(gpu, hd, kind):
    """One makes NaN of the queries that see it (a value of its coordinate alone), and nothing of the others: those before it in a
    block that both read, other heads', other tables'."""
    rng = np.random.default_rng(hd)
    counts, heads, kv_heads = [100, 260, 40], 4, 2
    n = sum(counts)
    for where, bad in ((100 + 70, np.nan), (100 + 133, np.inf), (100 + 259, -np.inf)):
        q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
        clean = [a.copy() for a in (q, k, v)]
        dims = 7 if kind == "value" else slice(None)
        {"query": q, "key": k, "value": v}[kind][where, 1, 7] = bad
        got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), heads, kv_heads, True).reshape(q.shape)
        sees = np.zeros(q.shape, bool)
        if kind == "query":
            sees[where, 1] = True
        else:
            sees[where:360, 2:4, dims] = True
        out, off = wanted(*clean, counts, counts, True)
        say(f"{kind} {bad} at row {where}: {int(sees.sum())} outputs see it")
        assert np.all(np.isnan(got[sees])) and np.all(np.abs(got - out)[~sees] <= off[~sees])


@pytest.mark.parametrize("hd", [16, 32, 64])
@pytest.mark.parametrize("kind", ["value", "key", "query"])
def test_numbers_that_are_not_finite_in_short_tables(gpu, hd, kind):
    """The same for tables whose blocks only one or two tiles of queries read."""
    rng = np.random.default_rng(hd + 1)
    counts, heads = [128, 200, 90], 2
    n = sum(counts)
    for where, bad in ((128 + 3, np.nan), (128 + 133, np.inf), (128 + 199, -np.inf)):
        q, k, v = inputs(rng, n, n, heads, heads, hd)
        clean = [a.copy() for a in (q, k, v)]
        dims = 7 if kind == "value" else slice(None)
        {"query": q, "key": k, "value": v}[kind][where, 1, 7] = bad
        got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), heads, heads, True).reshape(q.shape)
        sees = np.zeros(q.shape, bool)
        sees[where:where + 1 if kind == "query" else 328, 1, dims] = True
        out, off = wanted(*clean, counts, counts, True)
        say(f"{kind} {bad} at row {where}: {int(sees.sum())} outputs see it")
        assert np.all(np.isnan(got[sees])) and np.all(np.abs(got - out)[~sees] <= off[~sees])


@pytest.mark.parametrize("beside", [np.nan, 1e30])
@pytest.mark.parametrize("hd", [16, 48, 64, 80, 112])
def test_what_stands_beside_the_heads(gpu, dev, hd, beside):
    """Rows of one head among columns, and between rows of no table, that hold anything: short tables, tables whose tiles are made
    first, one long enough to be cut, and a table with rows but no queries."""
    rng = np.random.default_rng(hd)
    counts, ld = [100, 7, 250, 300, 64, 1100], hd + 11
    n = sum(counts)
    q, k, v = inputs(rng, n, n, 1, 1, hd)
    around = np.full((2, n + 8, ld), beside, np.float32)
    around[0, 4:-4, 5:5 + hd], around[1, 4:-4, 5:5 + hd] = flat(k), flat(v)
    at, rows, skip = offsets_of(counts), dev.of(around), 4 * (4 * ld + 5)
    asked = [c if i != 4 else 0 for i, c in enumerate(counts)]
    keep = np.concatenate([np.arange(at[i], at[i] + a) for i, a in enumerate(asked)])
    qd, qo, ko = dev.of(flat(q[keep])), dev.of(offsets_of(asked)), dev.of(at)
    for causal in (False, True):
        od = dev.of(np.full((len(keep), hd), 3.0, np.float32))
        gpu.attend_packed_dev(qd.ptr, rows.ptr + skip, rows.ptr + 4 * (n + 8) * ld + skip, qo.ptr, ko.ptr, len(counts), len(keep), n, 1, 1,
                              hd, od.ptr, causal, 0, ld)
        gpu.sync()
        check(od.download((len(keep), 1, hd)), *wanted(q[keep], k, v, asked, counts, causal), f"beside {beside}, causal {causal}")


def test_strides_and_spare_rows_on_device_memory(gpu, dev):
    """Queries, keys and values as parts of wider rows at odd distances; queries past the last table's are left as they were, and
    rows past it, NaN here, are not read as any table's."""
    rng = np.random.default_rng(4)
    counts, heads, kv_heads, hd = [70, 1, 333], 4, 2, 64
    n, total, far = sum(counts), sum(counts) + 9, (heads + 2 * kv_heads) * hd + 1
    rows = np.full((total, far), np.nan, np.float32)
    q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
    rows[:n, :heads * hd] = flat(q)
    rows[:n, heads * hd:(heads + kv_heads) * hd], rows[:n, (heads + kv_heads) * hd:-1] = flat(k), flat(v)
    rd, of = dev.of(rows), dev.of(offsets_of(counts))
    for causal in (False, True):
        od = dev.of(np.full((total, heads * hd), 3.0, np.float32))
        gpu.attend_packed_dev(rd.ptr, rd.ptr + 4 * heads * hd, rd.ptr + 4 * (heads + kv_heads) * hd, of.ptr, of.ptr, 3, total, total,
                              heads, kv_heads, hd, od.ptr, causal, far, far)
        gpu.sync()
        got = od.download((total, heads, hd))
        assert np.all(got[n:] == 3.0)
        check(got[:n], *wanted(q, k, v, counts, counts, causal), f"strided, causal {causal}")


def test_more_tables_than_a_wavefront(gpu):
    rng = np.random.default_rng(9)
    counts = [int(c) for c in rng.integers(0, 9, 500)]
    n = sum(counts)
    q, k, v = inputs(rng, n, n, 2, 2, 32)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), 2, 2, True).reshape(q.shape)
    check(got, *wanted(q, k, v, counts, counts, True), "500 tables")


def test_against_the_attention_of_one_table(gpu):
    """A table alone is what `attend_rows` gives, and what it gives packed with others (where its rows may go in fewer key ranges),
    all to f32's precision."""
    rng = np.random.default_rng(14)
    q, k, v = inputs(rng, 500, 500, 8, 8, 64)
    one = gpu.attend_rows(flat(q), flat(k), flat(v), 512, 8)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), [0, 500], 8, 8)
    size = np.sqrt(np.mean(np.square(one)))
    assert np.sqrt(np.mean(np.square(got - one))) <= 2.0**-19 * size  # each 2^-20 from 64 bits
    p, m, w = inputs(rng, 300, 300, 8, 8, 64)
    both = gpu.attend_packed(*(np.concatenate([flat(a), flat(b)]) for a, b in ((p, q), (m, k), (w, v))), [0, 300, 800], 8, 8)
    assert np.sqrt(np.mean(np.square(both[300:] - got))) <= 2.0**-19 * size


def test_captured_and_replayed(gpu, dev):
    """Captured, replayed with other rows and with the tables cut elsewhere, with eager calls between, and from another handle: the
    eager call's bits."""
    rng = np.random.default_rng(20)
    heads, hd, n = 4, 64, 400
    qd, kd, vd = (dev.of(np.zeros((n, heads * hd), np.float32)) for _ in range(3))
    od, oe = dev.of(np.zeros((n, heads * hd), np.float32)), dev.of(np.zeros((n, heads * hd), np.float32))
    of = dev.of(offsets_of([100, 300]))
    call = lambda g, out: g.attend_packed_dev(qd.ptr, kd.ptr, vd.ptr, of.ptr, of.ptr, 2, n, n, heads, heads, hd, out.ptr, True)
    call(gpu, od)
    gpu.sync()
    graph, other = Graph(gpu, lambda: call(gpu, od)), hip.Gpu(0)
    try:
        for counts in ([100, 300], [399, 1], [200, 150]):
            q, k, v = inputs(rng, n, n, heads, heads, hd)
            for b, a in ((qd, q), (kd, k), (vd, v), (of, offsets_of(counts))):
                b.upload(a)
            graph.replay()
            gpu.sync()
            m = sum(counts)
            got = od.download((n, heads, hd))[:m]
            for g in (gpu, other):
                call(g, oe)
                g.sync()
                assert np.array_equal(oe.download((n, heads, hd))[:m], got)
            check(got, *wanted(q[:m], k[:m], v[:m], counts, counts, True), f"replayed, {counts}")
    finally:
        graph.free()
        other.close()


def test_fitted_in_order_stored_and_grown(gpu, dev):
    """The three operators as they are used together: tables' rows attended in order, stored in pages, new rows added to each table, and
    answered from the pages. Exact pages give what attending the grown tables from scratch gives, and i16 pages what their
    numbers say."""
    rng = np.random.default_rng(33)
    heads, kv_heads, hd, rows = 4, 2, 64, 32
    before, after = [90, 0, 33], [93, 2, 64]
    n = sum(after)
    q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
    at = offsets_of(after)
    whole = gpu.attend_packed(flat(q), flat(k), flat(v), at, heads, kv_heads, True).reshape(q.shape)
    for fmt in (abi.KV_F32, abi.KV_I16):
        pool = P.Pool(fmt, kv_heads, hd, rows, 9)
        card = dev.of(pool.bytes)
        table = np.array([[3, 0, 7], [5, -1, -1], [8, 1, 4]], np.int32)
        d = abi.Pages(pool=card.ptr, kv_format=fmt, kv_heads=kv_heads, hd=hd, page_rows=rows, pages=9, tables=3, ld=3)
        first = np.concatenate([np.arange(at[t], at[t] + before[t]) for t in range(3)])
        rest = np.concatenate([np.arange(at[t] + before[t], at[t + 1]) for t in range(3)])
        gpu.pages_write(d, table, [0, 0, 0], offsets_of(before), flat(k[first]), flat(v[first]))
        new = [a - b for a, b in zip(after, before)]
        gpu.pages_write(d, table, before, offsets_of(new), flat(k[rest]), flat(v[rest]))
        got = gpu.pages_attend(d, table, after, flat(q[rest]), offsets_of(new), heads, True).reshape(len(rest), heads, hd)
        if fmt == abi.KV_F32:
            size = np.sqrt(np.mean(np.square(whole[rest])))
            assert np.sqrt(np.mean(np.square(got - whole[rest]))) <= 2.0**-19 * size
        sk, sv = gpu.pages_read(d, table, [0, 0, 0], at)
        out, off = wanted(q, sk.reshape(k.shape), sv.reshape(v.shape), after, after, True)
        check(got, out[rest], off[rest], f"grown, format {fmt}")


def test_refusals(gpu, dev):
    q, k = np.zeros((6, 256), np.float32), np.zeros((5, 128), np.float32)
    call = lambda q=q, k=k, v=k, qo=(0, 2, 6), heads=4, kv_heads=2, ko=(0, 5, 5): gpu.attend_packed(q, k, v, qo, heads, kv_heads, False, ko)
    call()
    for kw in [dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(heads=4, kv_heads=1), dict(q=q[:, :-1]), dict(v=k[:4]),
               dict(qo=(0, 2, 7)), dict(qo=(1, 2, 6)), dict(qo=(0, 3, 2)), dict(ko=(0, 6, 6)), dict(ko=(0, 5)), dict(qo=(0,), ko=(0,)),
               dict(qo=(0, 1.5, 2)), dict(k=k[:, :40], v=k[:, :40], q=q[:, :80]), dict(k=k.reshape(-1), v=k)]:
        with pytest.raises(ValueError):
            call(**kw)
    wide = np.zeros((2, 288), np.float32)
    with pytest.raises(ValueError):
        gpu.attend_packed(wide, wide, wide, [0, 2], 2, 2)  # heads of 144
    qd, of = dev.of(q), dev.of(np.array([0, 2, 6], np.int32))
    good = [qd.ptr, qd.ptr, qd.ptr, of.ptr, of.ptr, 2, 6, 6, 2, 2, 128, qd.ptr]
    for i, value in [(0, 0), (1, 0), (2, 0), (3, 0), (4, 0), (11, 0), (0, qd.ptr + 2), (4, of.ptr + 1), (5, 0), (5, -1), (6, -1), (7, -3),
                     (8, 3), (9, 0), (10, 0), (10, 8), (10, 136), (6, 2**31 - 5), (7, 2**31 - 5)]:
        args = list(good)
        args[i] = value
        with pytest.raises(ValueError):
            gpu.attend_packed_dev(*args)
    for ld in ((255, 0), (0, 255), (-1, 0)):
        with pytest.raises(ValueError):
            gpu.attend_packed_dev(*good, False, *ld)
    with pytest.raises(MemoryError):  # the tiles of 2^27 rows: 2^27 x 2 x 128 x 8 bytes
        gpu.attend_packed_dev(*good[:6], 6, 2**27, *good[8:])
    gpu.sync()
