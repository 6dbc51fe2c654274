"""Class scores read as distributions where rows are unusual: a NaN beside classes ruled out, classes all but certain."""
import numpy as np
import pytest

import test_class_stats as S
from conftest import pkg

hip, T = pkg("hip"), pkg("table")


def order(row):
    """Class ids in order: larger scores first, the lower id among equals, NaN after every number."""
    return sorted(range(len(row)), key=lambda i: (np.isnan(row[i]), 0.0 if np.isnan(row[i]) else -row[i], i))


def unusual_rows(rng, rows, n):
    """Scores with both a NaN and a class ruled out, at different places: numbers beside them, or nothing else."""
    x = rng.standard_normal((rows, n)).astype(np.float32)
    x[rng.random((rows, n)) < 0.4] = -np.inf
    x[rng.random((rows, n)) < 0.3] = np.nan
    x[0, ::2], x[0, 1::2] = np.nan, -np.inf
    x[1, ::2], x[1, 1::2] = -np.inf, np.nan
    return x


# ---- without a card ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [2, 3, 11])
def test_the_host_orders_nan_after_every_number(n):
    assert T.class_report([[np.nan, -np.inf, 1.0]], 1, 1.0, top=3)["top"].tolist() == [[2, 1, 0]]
    x = unusual_rows(np.random.default_rng(n), 40, n)
    assert T.class_report(x, 1, 1.0, top=n)["top"].tolist() == [order(row) for row in x]


def test_the_host_keeps_a_certain_rows_precision():
    """One class far ahead: log p of it is minus the others' weight, although 1 and that weight round to 1. float64's
    roundings are 2^-53 each: the exponents' (of at most 80, so 2^-53 * 80 of a weight) and a few more."""
    x = np.zeros((41, 10))
    x[:, 3] = np.arange(41) * 2.0
    rep = T.class_report(x, 1, 1.0, np.full(41, 3), 2)
    rest = 9 * np.exp(-x[:, 3])
    log_p, entropy = -np.log1p(rest), np.log1p(rest) + rest * x[:, 3] / (1 + rest)
    for got, want in ((rep["log_p"], log_p), (rep["top_log_p"][1:, 0], log_p[1:]), (rep["entropy"], entropy)):
        assert np.all(np.abs(got - want) <= 100 * 2.0 ** -53 * np.abs(want))
    pair = T.class_report([[0.0, 50.0]], 1, 1.0, [1])
    assert abs(pair["log_p"][0] + np.exp(-50.0)) <= 60 * 2.0 ** -53 * np.exp(-50.0)


@pytest.mark.parametrize("members,temperature", [(1, 0.0), (0, 0.9), (2, -1.0), (1, np.nan), (1, np.inf)])
def test_the_host_refuses_what_is_no_temperature(members, temperature):
    with pytest.raises(ValueError):
        T.class_report(np.zeros((2, 3)), members, temperature, [0, 1], 1)


# ---- the card ------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n,top", [(3, 3), (10, 10), (50, 50), (100, 8), (200, 64), (1000, 64), (2000, 64), (20000, 64)])
def test_the_card_orders_nan_after_every_number(gpu, n, top):
    print(f"order of rows with NaN and -inf: {n} classes, {top} best", flush=True)
    x = unusual_rows(np.random.default_rng(n), 9, n)
    x[2, : n - top // 2 - 1] = np.nan  # fewer numbers than are wanted
    x[3] = np.nan
    st, ids = gpu.class_stats(x, None, top)
    assert np.all(np.isnan(st[np.isnan(x).any(1)]))
    assert ids.tolist() == [order(row)[:top] for row in x]


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.9, 1.0, 2.5, 100.0, 1e38])
@pytest.mark.parametrize("n,top", [(2, 2), (7, 3), (50, 5), (100, 8), (200, 20), (1000, 10), (2000, 10), (40000, 10)])
def test_scores_further_apart_than_a_float_holds(gpu, n, top, temperature):
    """Finite scores whose difference passes float32's largest: at a high temperature the quotient does not. What does is
    -inf, as it rounds."""
    print(f"scores far apart: {n} classes, temperature {temperature}", flush=True)
    rng = np.random.default_rng(n)
    x = (rng.uniform(-1, 1, (6, n)) * 3.4e38).astype(np.float32)
    x[0, 0], x[0, 1] = 3.4e38, -3.4e38
    x[1] = -np.finfo(np.float32).max  # masks of the lowest value, one row of nothing else
    x[2, ::2] = -np.finfo(np.float32).max
    x[2, 1::2] = rng.standard_normal(n // 2)
    given = np.stack([np.zeros(6, int), np.full(6, n - 1), rng.integers(0, n, 6)], 1)
    st, ids = gpu.class_stats(x, given, top, temperature)
    inv = np.float64(np.float32(1.0) / np.float32(temperature))
    want, wids = S.plain(x, given, top, 1.0 / inv)
    with np.errstate(over="ignore"):
        beyond = np.isinf(want.astype(np.float32))
    assert np.array_equal(ids, wids)
    assert np.array_equal(np.isinf(st), beyond) and np.all(st[beyond] < 0)
    ok = ~beyond
    assert np.all(np.abs(st[ok] - want[ok]) <= S.bound(want[ok], x, temperature))
