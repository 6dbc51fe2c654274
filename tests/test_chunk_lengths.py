"""Chunks longer than the table, up to 2^31 - 1 rows: the table is one chunk of its own length, at the fit, in the exact
attention and in what is loaded from the fit."""
import numpy as np
import pytest

from conftest import pkg

abi, hip, fit, M, B, C = pkg("abi"), pkg("hip"), pkg("fit"), pkg("model"), pkg("bundle"), pkg("cache")
pytestmark = pytest.mark.gpu
LONGEST = 2 ** 31 - 1


@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


@pytest.fixture(scope="module", params=[64, 16])
def network(gpu, request):
    """Heads of this width (64: layers held as tiles)."""
    cfg = dict(M.FULL_CLASSIFIER, col_num_blocks=1, row_num_blocks=1, icl_num_blocks=2)
    if request.param == 16:
        cfg = dict(cfg, icl_nhead=8, embed_dim=16, row_num_cls=8)
    w = gpu.weights(M.Model.random(cfg, seed=5))
    yield w
    w.free()


@pytest.mark.parametrize("rows", [2, 77, 300])
@pytest.mark.parametrize("fmt", [abi.KV_F32, abi.KV_I16, abi.KV_I8, abi.KV_I4])
def test_a_fit_in_one_chunk(gpu, network, fmt, rows):
    print(f"fit in one chunk: format {fmt}, {rows} rows, width {network.model.d}", flush=True)
    rng = np.random.default_rng(rows)
    x, xt = rng.standard_normal((rows, 3)).astype(np.float32), rng.standard_normal((5, 3)).astype(np.float32)
    y = (np.arange(rows) % 2).astype(np.float32)
    scores = []
    records = []
    for chunk in (max(rows, 8), LONGEST):
        f = fit.fit_raw(gpu, network, x, y, 2, chunk=chunk, kv_format=fmt)
        records.append(f.layers[0])
        vm = C.Cache.open(B.Bundle(f.write())).load(gpu, network)[0]
        scores.append(gpu.predict(network, vm, xt, 2))
        vm.free()
    assert all(np.array_equal(a, b) for a, b in zip(*records)) and np.array_equal(*scores)
    assert np.all(np.isfinite(scores[0]))


@pytest.mark.parametrize("d,heads", [(128, 2), (32, 4)])
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_exact_attention_over_one_chunk(gpu, rows, d, heads):
    print(f"exact attention over one chunk: {rows} rows, {heads} heads of {d // heads}", flush=True)
    rng = np.random.default_rng(rows)
    q, kv = rng.standard_normal((rows, d)).astype(np.float32), rng.standard_normal(2 * rows * d).astype(np.float32)
    a, b = (gpu.attend(q, kv, rows, chunk, d, heads) for chunk in (rows, LONGEST))
    assert np.array_equal(a, b)
