"""Attention of packed tables and over pages where rows of one table are of very different sizes: blocks of zeros and of missing
rows beside tiny values, against 64 bits within the sum of the worst roundings of what a query sees (`pages_plain.attention`)."""
import numpy as np
import pytest

import pages_plain as P
from conftest import pkg
from test_packed import flat, inputs, wanted
from test_pages import FORMATS, check, described, dev, gpu, offsets_of, values  # noqa: F401 (fixtures)

abi = pkg("abi")
pytestmark = pytest.mark.gpu

# counts of rows: all read by few tiles of queries; made into tiles first (more readers, or heads over 64 wide); long, cut into runs
SHAPES = [([130, 200], 2, 2, 32), ([130, 200], 2, 2, 64), ([700, 90], 2, 1, 64), ([130, 200], 2, 1, 128), ([200, 130], 8, 1, 64),
          ([1500], 1, 1, 64), ([1500], 2, 2, 32)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("tiny", [1e-8, 1e-12, 1e-25, 1e-36])
@pytest.mark.parametrize("counts,heads,kv_heads,hd", SHAPES)
def test_packed_blocks_of_zeros(gpu, counts, heads, kv_heads, hd, tiny, causal):
    """64 rows whose values are all zeros, before or behind rows of tiny ones."""
    for zeros in (0, 1, 3):
        rng = np.random.default_rng(hd + zeros)
        n = sum(counts)
        q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
        v *= np.float32(tiny)
        at = 0
        for c in counts:
            for b in range(zeros % 2, -(-c // 64), 2) if zeros < 3 else [0]:
                v[at + 64 * b:min(at + 64 * b + 64, at + c)] = 0.0
            at += c
        got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), heads, kv_heads, causal).reshape(q.shape)
        got = got.astype(np.float64) / tiny
        out, off = (a / tiny for a in wanted(q, k, v, counts, counts, causal))
        at = 0
        for c in counts:
            check(got[at:at + c], out[at:at + c], off[at:at + c], f"zeros {zeros}, {c} rows, heads of {hd}, {tiny}, causal {causal}")
            at += c


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tiny", [1e-8, 1e-12, 1e-25])
@pytest.mark.parametrize("hd,group", [(64, 1), (64, 20), (128, 2)])
def test_pages_of_zeros_and_missing_pages(gpu, dev, fmt, tiny, hd, group):
    """Tables with 64 rows of zeros or on no page, before or behind rows of tiny values; each asked 250 times at once, so that
    a wavefront has several of their blocks."""
    rng = np.random.default_rng(hd + group)
    rows, T, length, copies = 32, 4, 200, 250
    pool = P.Pool(fmt, 1, hd, rows, T * 7, fill=0)
    table = rng.permutation(T * 7).astype(np.int32).reshape(T, 7)
    k, v = values(rng, T * length, 1, hd).reshape(T, length, 1, hd), (values(rng, T * length, 1, hd) * np.float32(tiny)).reshape(T, length, 1, hd)
    v[0, :64], v[1, 64:128], v[1, 192:] = 0.0, 0.0, 0.0
    there = np.ones((T, length), bool)
    there[2, :64] = there[3, 64:128] = False
    for t in range(T):
        for i in range(length):
            pool.write(table[t, i // rows], i % rows, k[t, i], v[t, i])
    told = table.copy()
    told[2, :2] = told[3, 2:4] = -1
    told, n = np.repeat(told, copies, 0), T * copies
    q = (rng.standard_normal((n, group, hd)) * 0.4).astype(np.float32)
    card, tb, ln, of = dev.of(pool.bytes), dev.of(told), dev.of(np.full(n, length, np.int32)), dev.of(offsets_of([1] * n))
    qd, od = dev.of(q), dev.of(np.zeros(q.shape, np.float32))
    gpu.pages_attend_dev(described(pool, n, 7, card.ptr, tb.ptr), ln.ptr, qd.ptr, of.ptr, n, group, od.ptr)
    gpu.sync()
    got = od.download(q.shape).astype(np.float64) / tiny
    for t in range(T):
        kt, vt = pool.rows_of(table[t], length)
        asked = slice(copies * t, copies * (t + 1))
        out, off = P.attention(q[asked], kt[there[t]], vt[there[t]], [int(there[t].sum())] * copies)
        check(got[asked], out / tiny, off / tiny, f"format {fmt}, table {t}, {tiny}")


LARGE = 1e37


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("counts,heads,kv_heads,hd", SHAPES + [([2300], 2, 1, 128), ([4300], 1, 1, 64)])
def test_packed_values_near_the_largest_float(gpu, counts, heads, kv_heads, hd, causal):
    """Outputs are means of values: finite where those are, also where several states are put together."""
    rng = np.random.default_rng(hd)
    n = sum(counts)
    q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
    got = gpu.attend_packed(flat(q), flat(k), flat(v * np.float32(LARGE)), offsets_of(counts), heads, kv_heads, causal).reshape(q.shape)
    check(got.astype(np.float64) / LARGE, *wanted(q, k, v, counts, counts, causal), f"{counts} rows, heads of {hd}, causal {causal}")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd,lengths,counts,causal", [(64, [9000], [2], False), (64, [3000, 2500], [9, 8], True), (128, [5000], [3], True),
                                                      (64, [300] * 40, [40] * 40, True)])
def test_pages_values_near_the_largest_float(gpu, dev, fmt, hd, lengths, counts, causal):
    """One query's parts joined by four wavefronts, many queries' by one, a workgroup's parts joined in it, and none."""
    rng = np.random.default_rng(hd + len(lengths))
    rows, ld = 64, -(-max(lengths) // 64)
    table = np.arange(len(lengths) * ld, dtype=np.int32).reshape(len(lengths), ld)
    pool = P.Pool(fmt, 1, hd, rows, table.size)
    for t, n in enumerate(lengths):
        for i in range(n):
            pool.write(table[t, i // rows], i % rows, *(values(rng, 1, 1, hd)[0] * np.float32(f) for f in (1.0, LARGE)))
    q = (rng.standard_normal((sum(counts), 2, hd)) * 0.4).astype(np.float32)
    card = dev.of(pool.bytes)
    got = gpu.pages_attend(described(pool, len(lengths), ld, card.ptr), table, lengths, flat(q), offsets_of(counts), 2, causal).reshape(q.shape)
    at = 0
    for t, n in enumerate(counts):
        k, v = pool.rows_of(table[t], lengths[t])
        out, off = P.attention(q[at:at + n], k, v / LARGE, P.limits_of(lengths[t], n, causal))
        # Values without a mean: the outputs are their weights' chance, 1 / sqrt(rows) of a value, and so are the weights' errors'. A
        # weight's: a score of 128 products of 0.5 by 0.4 (a sum of about 2) added in f32, 2^-24 sqrt(132 / 3) 2 = 8e-7, its products'
        # halves 2^-22 0.2 sqrt(128) 1.7 = 9e-7, the exponent's argument below 16 2^-21 0.69 / sqrt(3) = 2e-7, exp2 1e-7: 1.3e-6
        # together, of which a head's outputs have three times as much at most.
        check(got[at:at + n].astype(np.float64) / LARGE, out, off, f"format {fmt}, table {t}", 3 * 1.3e-6)
        at += n


def by_tables(counts):
    at = 0
    for c in counts:
        yield at, at + c
        at += c


@pytest.mark.parametrize("kind", ["key", "value"])
@pytest.mark.parametrize("larger", [1e4, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("counts,heads,kv_heads,hd", SHAPES)
def test_packed_rows_that_a_query_does_not_see(gpu, counts, heads, kv_heads, hd, larger, kind):
    """In order: a row of a block far larger than those before it takes nothing from the queries that do not see it, and is what those
    see that do; with as many queries as rows, and fewer."""
    rng = np.random.default_rng(hd + heads)
    n = sum(counts)
    for queries in (counts, [max(1, c // 3) for c in counts]):
        q, k, v = inputs(rng, sum(queries), n, heads, kv_heads, hd)
        rows = [a + int(f * (b - a)) for a, b in by_tables(counts) for f in (0.41, 0.87)]
        for r in rows:
            {"key": k, "value": v}[kind][r] *= np.float32(larger)
        got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(queries), heads, kv_heads, True, offsets_of(counts)).reshape(q.shape)
        out, off = wanted(q, k, v, queries, counts, True)
        if kind == "value" or larger < 1e6:  # scores past 2^22 have no fractions to speak of
            assert np.all(np.isfinite(got)) and np.all(np.abs(got - out) <= off)
        # where one row outweighs all others the roundings of its weight do not cancel: together only those that see neither
        for (a, b), (qa, qb) in zip(by_tables(counts), by_tables(queries)):
            at = qa + np.array([i for i, m in enumerate(P.limits_of(b - a, qb - qa, True)) if not any(a <= r < a + m for r in rows)], int)
            if len(at):
                check(got[at], out[at], off[at], f"{kind} {larger}, {qb - qa} over {b - a}")


@pytest.mark.parametrize("counts,heads,kv_heads,hd", SHAPES)
def test_packed_blocks_that_a_query_does_not_see(gpu, counts, heads, kv_heads, hd):
    """In order: blocks of values 2^140 times those of the blocks before them."""
    rng = np.random.default_rng(hd)
    n = sum(counts)
    q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
    v *= np.float32(1e-6)
    for a, b in by_tables(counts):
        v[a + (b - a) // 128 * 64:b] *= np.float32(2.0**100)
        v[a + (b - a) // 128 * 64:b] *= np.float32(2.0**40)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), heads, kv_heads, True).reshape(q.shape).astype(np.float64)
    out, off = wanted(q, k, v, counts, counts, True)
    for a, b in by_tables(counts):
        c = a + (b - a) // 128 * 64
        if c > a:
            check(got[a:c] * 1e6, out[a:c] * 1e6, off[a:c] * 1e6, f"{b - a} rows, before")
        check(got[c:b] * 1e-36, out[c:b] * 1e-36, off[c:b] * 1e-36, f"{b - a} rows, from there on")


@pytest.mark.parametrize("counts,heads,kv_heads,hd", SHAPES)
def test_packed_blocks_that_weigh_nothing(gpu, counts, heads, kv_heads, hd):
    """A block of values 1e12 times the others', whose scores are 90 below theirs: the others' outputs, to their own precision."""
    rng = np.random.default_rng(hd)
    n = sum(counts)
    for last in (False, True):
        q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
        q[:, :, 0], k[:, :, 0] = 8.0, 0.0
        left = np.ones(n, bool)
        for a, b in by_tables(counts):
            at = a + ((b - a - 1) // 64 * 64 if last else 0)
            left[at:min(at + 64, b)] = False
        k[~left, :, 0] = -12.0
        v[~left] *= np.float32(1e12)
        got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), heads, kv_heads).reshape(q.shape)
        rows = [int(left[a:b].sum()) for a, b in by_tables(counts)]
        # what the block adds: e^-80 1e12, at most 2e-23
        check(got, *wanted(q, k[left], v[left], counts, rows, False), f"the {'last' if last else 'first'} block")


def asked_often(gpu, dev, pool, table, lengths, q, counts, heads, causal, copies):
    """The outputs of queries of a few tables, asked `copies` times in one call, so that a wavefront has several of their blocks."""
    T, n = len(lengths), sum(counts)
    card, tb = dev.of(pool.bytes), dev.of(np.tile(table, (copies, 1)))
    ln, of, qd = dev.of(np.tile(np.array(lengths, np.int32), copies)), dev.of(offsets_of(counts * copies)), dev.of(np.tile(q, (copies, 1, 1)))
    od = dev.of(np.zeros((copies * n,) + q.shape[1:], np.float32))
    gpu.pages_attend_dev(described(pool, T * copies, table.shape[1], card.ptr, tb.ptr), ln.ptr, qd.ptr, of.ptr, copies * n, heads, od.ptr,
                         causal)
    gpu.sync()
    return od.download((copies, n) + q.shape[1:]).astype(np.float64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kind", ["key", "value"])
@pytest.mark.parametrize("larger", [1e4, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("hd,group,copies", [(64, 1, 1), (64, 4, 150), (128, 2, 150), (48, 1, 300)])
def test_pages_rows_that_a_query_does_not_see(gpu, dev, fmt, kind, larger, hd, group, copies):
    """In order: a row far larger than those before it takes nothing from the queries that do not see it."""
    rng = np.random.default_rng(hd + group)
    rows, kv_heads, lengths, counts = 32, 2, [100, 37, 130], [20, 18, 40]
    table = rng.permutation(15).astype(np.int32).reshape(3, 5)
    pool = P.Pool(fmt, kv_heads, hd, rows, 15, fill=0xFF)
    large = [[n - 7, n - 15] for n in lengths]
    for t, n in enumerate(lengths):
        for i in range(n):
            k, v = values(rng, 1, kv_heads, hd)[0], values(rng, 1, kv_heads, hd)[0]
            f = np.float32(larger if i in large[t] else 1.0)
            pool.write(table[t, i // rows], i % rows, *((k * f, v) if kind == "key" else (k, v * f)))
    q = (rng.standard_normal((sum(counts), kv_heads * group, hd)) * 0.4).astype(np.float32)
    got = asked_often(gpu, dev, pool, table, lengths, q, counts, kv_heads * group, True, copies)
    at = 0
    for t, n in enumerate(counts):
        k, v = pool.rows_of(table[t], lengths[t])
        limits = P.limits_of(lengths[t], n, True)
        out, off = P.attention(q[at:at + n], k, v, limits)
        blind = np.array([i for i, m in enumerate(limits) if m <= min(large[t])])
        for c in sorted({0, 1 % copies, copies // 2, copies - 1}):
            one = got[c, at:at + n]
            if kind == "value" or larger < 1e6:
                assert np.all(np.isfinite(one)) and np.all(np.abs(one - out) <= off)
            check(one[blind], out[blind], off[blind], f"format {fmt}, {kind} {larger}, table {t}, copy {c}", 3 * 1.3e-6)
        at += n


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd,group,copies", [(64, 1, 1), (64, 4, 150), (128, 2, 150)])
def test_pages_blocks_apart(gpu, dev, fmt, hd, group, copies):
    """Blocks of values 2^100 times those before them, which the first queries do not see; and such a block whose scores are 90 below
    the others', which weighs nothing."""
    rng = np.random.default_rng(hd + group)
    rows, lengths, counts = 64, [200, 192], [20, 40]
    table = rng.permutation(8).astype(np.int32).reshape(2, 4)
    q = (rng.standard_normal((sum(counts), group, hd)) * 0.4).astype(np.float32)
    q[:, :, 0] = 8.0
    for weighs in (True, False):
        pool = P.Pool(fmt, 1, hd, rows, 8, fill=0xFF)
        # the last 8 rows of the first, the last 32 of the second; or the block from row 64 on
        large = [lambda i, n: i >= 192, lambda i, n: i >= 160] if weighs else [lambda i, n: 64 <= i < 128] * 2
        for t, n in enumerate(lengths):
            k, v = values(rng, n, 1, hd), values(rng, n, 1, hd)
            k[:, :, 0] = 0.0
            for i in range(n):
                if large[t](i, n):
                    v[i] *= np.float32(2.0**100)
                    k[i, :, 0] = 0.0 if weighs else -22.5
                pool.write(table[t, i // rows], i % rows, k[i], v[i])
        got = asked_often(gpu, dev, pool, table, lengths, q, counts, group, True, copies)
        at = 0
        for t, n in enumerate(counts):
            k, v = pool.rows_of(table[t], lengths[t])
            limits = P.limits_of(lengths[t], n, True)
            if not weighs:  # e^-150 2^100, at most 1e-35
                left = np.array([not large[t](i, lengths[t]) for i in range(lengths[t])])
                k, v, limits = k[left], v[left], [int(left[:m].sum()) for m in limits]
            out, off = P.attention(q[at:at + n], k, v, limits)
            sees = np.array([weighs and any(large[t](i, lengths[t]) for i in range(m)) for m in limits])
            for c in sorted({0, copies // 2, copies - 1}):
                one = got[c, at:at + n]
                assert np.all(np.isfinite(one)) and np.all(np.abs(one - out) <= off)
                if not np.all(sees):
                    check(one[~sees], out[~sees], off[~sees], f"format {fmt}, table {t}, copy {c}, weighs {weighs}")
            at += n


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd,group,causal", [(64, 1, False), (64, 20, True), (128, 2, True)])
def test_pages_small_queries_of_large_keys(gpu, dev, fmt, hd, group, causal):
    """Scores of ordinary size, of queries of 1e-34 and keys of 1e34, beside a table of ordinary ones and queries of zeros."""
    rng = np.random.default_rng(hd)
    lengths, counts = [150, 90, 70], [4, 3, 2]
    table = rng.permutation(9).astype(np.int32).reshape(3, 3)
    pool = P.Pool(fmt, 1, hd, 64, 9, fill=0xFF)
    q = (rng.standard_normal((sum(counts), group, hd)) * 0.4).astype(np.float32)
    q[:4] *= np.float32(1e-34)
    q[8] = 0.0
    for t, n in enumerate(lengths):
        for i in range(n):
            k, v = values(rng, 1, 1, hd)[0], values(rng, 1, 1, hd)[0]
            pool.write(table[t, i // 64], i % 64, k * np.float32(1e34 if t == 0 else 1.0), v)
    card = dev.of(pool.bytes)
    got = gpu.pages_attend(described(pool, 3, 3, card.ptr), table, lengths, flat(q), offsets_of(counts), group, causal).reshape(q.shape)
    at = 0
    for t, n in enumerate(counts):
        out, off = P.attention(q[at:at + n], *pool.rows_of(table[t], lengths[t]), P.limits_of(lengths[t], n, causal))
        check(got[at:at + n], out, off, f"format {fmt}, table {t}", 3 * 1.3e-6)
        at += n


@pytest.mark.parametrize("counts,heads,kv_heads,hd,causal", [
    ([4300], 1, 1, 64, False), ([4300], 2, 1, 32, False), ([2300], 2, 1, 128, True), ([2300], 1, 1, 128, False), ([900, 130], 2, 2, 64, True),
    ([900, 130], 2, 1, 32, False), ([600, 130], 1, 1, 128, True)])
def test_packed_rows_of_all_sizes(gpu, counts, heads, kv_heads, hd, causal):
    """Keys and values of sizes 2^-20 to 1 from row to row, in tiles of 256 and of 128 columns, blocks of even rows before, between and
    behind."""
    rng = np.random.default_rng(hd + heads)
    n = sum(counts)
    q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
    f = np.exp2(-rng.integers(0, 21, (2, n, 1, 1))).astype(np.float32)
    f[:, np.arange(n) // 64 % 5 < 2] = 1.0
    k, v = k * f[0], v * f[1]
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), heads, kv_heads, causal).reshape(q.shape)
    some = np.unique(np.concatenate([np.arange(0, n, 31), [n - 1]])) if n > 2000 else np.arange(n)
    at = 0
    for c in counts:
        mine = some[(some >= at) & (some < at + c)]
        limits = P.limits_of(c, c, causal)
        out, off = P.attention(q[mine], k[at:at + c], v[at:at + c], [limits[i - at] for i in mine])
        check(got[mine], out, off, f"{c} rows, heads of {hd}, causal {causal}")
        at += c


@pytest.mark.parametrize("counts,heads,kv_heads,hd", SHAPES)
def test_packed_rows_apart_and_numbers_that_are_not_finite(gpu, counts, heads, kv_heads, hd):
    """In order, in one block: a value that is not finite, a key that is not finite and a large row, each behind the other."""
    rng = np.random.default_rng(hd)
    n = sum(counts)
    q, k, v = inputs(rng, n, n, heads, kv_heads, hd)
    clean_k, clean_v = k.copy(), v.copy()
    sees_value, sees_key = np.zeros(n, bool), np.zeros(n, bool)
    blind = np.zeros(n, bool)
    for a, b in by_tables(counts):
        v[a + 70, 0, 7], v[a + 75] = np.inf, v[a + 75] * np.float32(1e10)
        k[a + 80, 0, 3] = np.nan
        sees_value[a + 70:b], sees_key[a + 80:b], blind[a:a + 70] = True, True, True
        clean_v[a + 75] *= np.float32(1e10)
    got = gpu.attend_packed(flat(q), flat(k), flat(v), offsets_of(counts), heads, kv_heads, True).reshape(q.shape)
    out, off = wanted(q, clean_k, clean_v, counts, counts, True)
    check(got[blind], out[blind], off[blind], f"{counts}, heads of {hd}")
    group = heads // kv_heads
    first = np.arange(heads) < group  # the heads that read the one with such numbers
    nan = np.zeros(q.shape, bool)
    nan[:, first, 7] |= sees_value[:, None]
    nan[:, first] |= sees_key[:, None, None]
    assert np.all(np.isnan(got[nan])) and np.all(np.abs(got - out)[~nan] <= off[~nan])
