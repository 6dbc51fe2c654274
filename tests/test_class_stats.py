"""Rows of class scores read as distributions (`tah_class_stats`, `table.class_report`): entropy, log probabilities of
given classes and the most probable classes, against the definition in float64."""
import ctypes
import os

import numpy as np
import pytest

from conftest import pkg

abi, hip, T, dm = pkg("abi"), pkg("hip"), pkg("table"), pkg("devmem")


def say(*a):
    print(*a, flush=True)


def plain(x, given, top, temperature):
    """The definition in float64 (the inputs are float32): stats, ids."""
    x64 = x.astype(np.float64)
    rows, n = x.shape
    stats = np.full((rows, 1 + given.shape[1] + top), np.nan)
    ids = np.empty((rows, top), np.int32)
    for r in range(rows):
        v = x64[r]
        order = sorted(range(n), key=lambda i: (np.isnan(v[i]), -v[i] if not np.isnan(v[i]) else 0.0, i)) if n <= 512 else \
            np.argsort(np.where(np.isnan(v), np.inf, -v), kind="stable")
        ids[r] = order[:top]
        if np.isnan(v).any() or v.max() == np.inf:
            logp, ent = np.full(n, np.nan), np.nan
        elif v.max() == -np.inf:
            logp, ent = v, 0.0
        else:
            u = (v - v.max()) / temperature
            best = int(np.argmax(v))
            rest = np.exp(np.delete(u, best)).sum()
            logp = u - np.log1p(rest)
            with np.errstate(invalid="ignore"):
                ent = np.log1p(rest) - np.where(np.exp(u) > 0, np.exp(u) * u, 0.0).sum() / (1.0 + rest)
        stats[r, 0] = ent
        for i, g in enumerate(given[r]):
            if 0 <= g < n:
                stats[r, 1 + i] = logp[g]
        stats[r, 1 + given.shape[1]:] = logp[ids[r]]
    return stats, ids


def scores(rng, rows, n, kind):
    x = (rng.standard_normal((rows, n)) * rng.uniform(0.2, 8.0, (rows, 1))).astype(np.float32)
    if kind == "special":
        x[0::9] = np.round(x[0::9])              # ties
        x[1::9] = 2.5                            # all equal
        x[2::9, : n // 2] = -np.inf              # half of them ruled out
        x[3::9] = -np.inf                        # all of them
        x[4::9, n // 2] = np.nan
        x[5::9, n // 3] = np.inf
        x[6::9] *= 1e30                          # one class certain
        x[7::9, ::2] = 0.0
        x[7::9, 1::2] = -0.0                     # equal zeros
        x[8::9] = np.sort(x[8::9], axis=1)       # the most probable last, side by side
    return x


def bound(want, x, temperature):
    """A score's difference from the largest and its quotient are off by 2^-24 each, so a weight by 2^-23 of the quotient u
    beside the exponential's own 2^-22; u is at most 104 where a weight counts. Sums of positive terms keep the terms'
    relative error, plus 2^-24 for each of at most 40 + n / 256 additions in a row; the logarithm's and the last sums' own
    roundings are 2^-22 of the result."""
    n = x.shape[1]
    rel = 104 * 2.0 ** -23 + 2.0 ** -22 + (40 + n / 256) * 2.0 ** -24
    return rel + 2.0 ** -22 * np.abs(want)


def compare(got, want, x, temperature):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    err = np.abs(got[ok] - want[ok])
    say(f"  worst {err.max() if err.size else 0:.2e}")
    assert np.all(err <= bound(want[ok], x, temperature))


# ---- without a card ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["plain", "special"])
def test_the_host_report_is_the_definition(kind):
    rng = np.random.default_rng(4)
    x = scores(rng, 40, 11, kind)
    labels = rng.integers(-1, 11, 40)
    got = T.class_report(x, 3, 0.9, labels, 4)
    want, ids = plain(x, labels[:, None], 4, 3 * 0.9)
    assert np.array_equal(got["top"], ids)
    for a, b in ((got["entropy"], want[:, 0]), (got["log_p"], want[:, 1]), (got["top_log_p"], want[:, 2:])):
        assert np.allclose(a, b, rtol=1e-12, atol=1e-12, equal_nan=True)
    p = T.finish_proba(x[:1].astype(np.float64), 3, 0.9)
    if kind == "plain":
        assert np.allclose(np.exp(got["top_log_p"][0]), p[0][got["top"][0]])


def test_the_host_report_refuses():
    x = np.zeros((3, 4))
    for labels, top in (([0, 1], 1), ([0, 1, 4], 1), ([0, 1, -2], 1), ([0.0, 1.0, 2.0], 1), ([0, 1, 2], 5), (None, -1)):
        with pytest.raises(ValueError):
            T.class_report(x, 1, 1.0, labels, top)


def test_null_handles_are_refused():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libtah_hip.so not built")
    some = ctypes.c_void_p(4096)
    assert abi.lib().tah_class_stats_dev(None, some, 1, 2, 0, 1.0, None, 0, 0, some, None) == abi.E_ARG
    assert abi.lib().tah_class_stats(None, None, 1, 2, 1.0, None, 0, 0, None, None) == abi.E_ARG


# ---- the card ------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["plain", "special"])
@pytest.mark.parametrize("rows,n,k,top", [(1, 1, 1, 1), (1, 2, 0, 0), (300, 2, 1, 2), (1000, 3, 0, 3), (65, 10, 2, 10),
                                          (130, 16, 1, 1), (130, 17, 1, 17), (64, 64, 3, 5), (9, 65, 64, 64),
                                          (70, 999, 1, 20), (37, 1024, 0, 64), (20, 1025, 1, 3), (11, 5000, 2, 64),
                                          (9, 16384, 1, 7), (10, 16385, 1, 64), (9, 70001, 1, 33), (1, 300000, 1, 64), (2, 1 << 20, 1, 64), (3, 8193, 1, 40), (200, 24, 2, 24), (99, 40, 1, 40),
                                          (41, 33, 1, 5), (77, 100, 2, 8), (77, 128, 0, 0), (50, 129, 1, 3), (33, 256, 1, 8),
                                          (33, 200, 3, 9), (31, 257, 1, 5), (40, 600, 1, 10), (5, 4096, 1, 20), (5, 4097, 0, 64),
                                          (4, 8192, 2, 3)])
def test_class_stats(gpu, kind, rows, n, k, top):
    say(f"class stats {rows} x {n}, {k} given, {top} best, {kind}")
    rng = np.random.default_rng(rows * 7 + n)
    x = scores(rng, rows, n, kind)
    given = rng.integers(-1, n, (rows, k))
    temperature = 0.9 if kind == "plain" else 1.7
    got, ids = gpu.class_stats(x, given, top, temperature)
    want, wids = plain(x, given, top, np.float64(1.0) / np.float64(np.float32(1.0) / np.float32(temperature)))
    assert np.array_equal(ids, wids)
    compare(got, want, x, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,ld", [(33, 7, 12), (33, 16, 17), (20, 300, 303), (5, 2000, 2001), (5, 40000, 40007)])
def test_rows_apart(gpu, rows, n, ld):
    """Rows of scores with others between them, starting off a 16-byte line; nothing written past the outputs."""
    say(f"class stats {rows} x {n}, {ld} apart")
    rng = np.random.default_rng(n)
    wide = np.full((rows, ld), np.nan, np.float32)
    wide[:, :n] = scores(rng, rows, n, "plain")
    given = rng.integers(0, n, (rows, 2)).astype(np.int32)
    given[0] = (-7, n)  # outside: NaN
    top = 5
    flat = np.concatenate([np.full(1, np.nan, np.float32), wide.reshape(-1)])
    bx, bg = dm.DeviceBuffer.of(flat), dm.DeviceBuffer.of(given)
    bs, bi = dm.DeviceBuffer.of(np.full(rows * 8 + 8, 3.0, np.float32)), dm.DeviceBuffer.of(np.full(rows * top + 8, -9, np.int32))
    gpu.class_stats_dev(bx.ptr + 4, rows, n, bg.ptr, 2, top, bs.ptr, bi.ptr, ld=ld)
    gpu.sync()
    st, ids = bs.download(rows * 8 + 8), bi.download(rows * top + 8, np.int32)
    want, wids = plain(wide[:, :n], given, top, 1.0)
    assert np.all(st[rows * 8:] == 3.0) and np.all(ids[rows * top:] == -9)
    assert np.array_equal(ids[:rows * top].reshape(rows, top), wids)
    compare(st[:rows * 8].reshape(rows, 8), want, wide[:, :n], 1.0)
    for b in (bx, bg, bs, bi):
        b.free()


@pytest.mark.gpu
def test_confident_rows_keep_their_precision(gpu):
    """One class far ahead: log p of it is minus the others' weight, which float32 holds to 2^-20 of itself although 1 + it
    rounds to 1."""
    x = np.zeros((40, 10), np.float32)
    x[:, 3] = np.arange(40, dtype=np.float32) * 2
    st, ids = gpu.class_stats(x, np.full(40, 3), 1)
    rest = 9 * np.exp(-2.0 * np.arange(40))
    assert np.array_equal(ids[1:, 0], np.full(39, 3)) and ids[0, 0] == 0
    assert np.all(np.abs(st[:, 1] + np.log1p(rest)) <= 2.0 ** -16 * np.log1p(rest))
    ent = np.log1p(rest) + rest / (1 + rest) * 2.0 * np.arange(40)
    assert np.all(np.abs(st[:, 0] - ent) <= 2.0 ** -15 * ent)


@pytest.mark.gpu
def test_class_stats_refused(gpu):
    x = np.zeros((2, 5), np.float32)
    for given, top, temperature in (([0, 5], 0, 1.0), ([0, -2], 0, 1.0), ([0], 0, 1.0), ([0.0, 1.0], 0, 1.0), (None, 6, 1.0),
                                    (None, -1, 1.0), (None, 1, 0.0), (None, 1, -1.0), (None, 1, np.nan), (None, 1, np.inf),
                                    (None, 1, 1e-45), (np.zeros((2, 65), int), 0, 1.0)):
        with pytest.raises(ValueError):
            gpu.class_stats(x, given, top, temperature)
    b = dm.DeviceBuffer(4096)
    # no rows: a call that was let through would read nothing
    for args in ((None, 0, 5, b.ptr, 1, 1, b.ptr, b.ptr), (b.ptr, -1, 5, b.ptr, 1, 1, b.ptr, b.ptr),
                 (b.ptr, 0, 0, b.ptr, 1, 0, b.ptr, b.ptr), (b.ptr, 0, 5, None, 1, 1, b.ptr, b.ptr),
                 (b.ptr, 0, 5, b.ptr, 1, 1, b.ptr, None), (b.ptr, 0, 5, b.ptr, 65, 1, b.ptr, b.ptr),
                 (b.ptr, 0, 5, b.ptr, 1, 6, b.ptr, b.ptr), (b.ptr, 0, (1 << 20) + 1, b.ptr, 1, 1, b.ptr, b.ptr)):
        with pytest.raises(ValueError):
            gpu.class_stats_dev(*args)
    with pytest.raises(ValueError):
        gpu.class_stats_dev(b.ptr, 0, 5, b.ptr, 1, 1, b.ptr, b.ptr, ld=4)
    for off in ((1, 0, 0, 0), (0, 2, 0, 0), (0, 0, 3, 0), (0, 0, 0, 1)):
        with pytest.raises(ValueError):
            gpu.class_stats_dev(b.ptr + off[0], 0, 5, b.ptr + off[1], 1, 1, b.ptr + off[2], b.ptr + off[3])
    for n in (1, 5, 1024, 2000, 1 << 20):  # no rows: nothing to do, however many classes
        gpu.class_stats_dev(b.ptr, 0, n, b.ptr, 1, 1, b.ptr, b.ptr)
        st, ids = gpu.class_stats(np.zeros((0, n), np.float32), None, 1)
        assert st.shape == (0, 2) and ids.shape == (0, 1)
    gpu.sync()
    b.free()


@pytest.mark.gpu
def test_report_card_matches_host(gpu):
    rng = np.random.default_rng(12)
    sums = scores(rng, 200, 14, "special").astype(np.float64) * 4
    labels = rng.integers(-1, 14, 200)
    a, b = T.class_report(sums, 4, 0.9, labels, 3, gpu=gpu), T.class_report(sums.astype(np.float32), 4, 0.9, labels, 3)
    assert np.array_equal(a["top"], b["top"])
    for k in ("entropy", "log_p", "top_log_p"):
        assert np.allclose(a[k], b[k], rtol=2e-6, atol=2e-5, equal_nan=True)
    assert "log_p" not in T.class_report(sums, 4, 0.9, gpu=gpu)
