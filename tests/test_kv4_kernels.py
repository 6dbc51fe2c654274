"""Each attention kernel over 4-bit tiles against 64 bits, to the precision of f32 arithmetic: the call's own kernel is
told apart by the launch probe (which counts the many-query kernel's launches and no others), and the limit is one that
queries or weights held in a single fp16 would not keep, which is checked here on the CPU."""
import numpy as np
import pytest

import kv4_plain as P
from conftest import pkg

abi, hip, M, dm = pkg("abi"), pkg("hip"), pkg("model"), pkg("devmem")

# The largest root mean square error over a head's outputs, as a share of the outputs' own. Inputs as `inputs` makes them:
# scores of standard deviation SPREAD, under whose softmax a key's expected score is SPREAD^2, about 6. Roundings are
# independent and half a step at most (2^-24 of a float32, uniform: 2^-24 / sqrt 3).
#  * A score is 64 terms of a query's high half and 64 of its low: at most 128 additions whose partial sums grow to the
#    score: 2^-24 / sqrt 3 * sqrt 128 * 6.25 / sqrt 3 = 1.4e-6, times the value's distance from the output, over keys that
#    average to a quarter of it: under 1e-6 of the output. The halves leave 2^-22 of a query, the sums of a score of 10 or
#    so times log2 e in the exponent 2^-21 / sqrt 3 of a weight, which average alike: 3e-7.
#  * The sums over the keys: 32 keys a product, high and low, so 10,000 rows are 625 additions to a growing sum,
#    2^-24 / sqrt 3 * sqrt 625 / sqrt 3 = 5e-7; a weight sum takes 2,500 of its own in a lane, of which four join: 5e-7.
# Together under 1.4e-6. The limit is the next power of two with room for 100,000 rows' sums.
LIMIT = 2.0 ** -18
SPREAD = 2.5


def say(*a):
    print(*a, flush=True)


def inputs(rng, rows, heads, nq, k_scale=1.0, v_scale=1.0):
    """Keys, values [rows][d] and queries [nq][d]. A value is the key's own coordinate seven on (of the head), so that an
    output follows its query and an error in a query is not averaged away; each head's keys and values, by 2^-8 to 2^8,
    have a magnitude of their own that its queries undo."""
    d = 64 * heads
    k = rng.standard_normal((rows, d)) * 0.55
    v = np.roll(k.reshape(rows, heads, 64), 7, 2).reshape(rows, d)
    size = np.repeat(2.0 ** rng.integers(-8, 9, heads), 64)
    q = rng.standard_normal((nq, d)) * (SPREAD / (0.55 * 8)) / (k_scale * size)
    return (k * k_scale * size).astype(np.float32), (v * v_scale * size[::-1]).astype(np.float32), q.astype(np.float32)


def worst_head(got, want, heads):
    """The largest over heads of the root mean square error over the outputs' own."""
    e, w = (np.asarray(a, np.float64).reshape(-1, heads, 64) for a in (got - want, want))
    return float(np.sqrt((e ** 2).mean((0, 2)) / (w ** 2).mean((0, 2))).max())


# ---- what the limit tells apart, without a card ------------------------------------------------------------------------
def halves(x, parts):
    """float32 x as a sum of `parts` fp16 numbers, each row's largest magnitude first brought below 2^14."""
    e = 14 - np.frexp(np.abs(x).max(1, keepdims=True))[1]
    left, out = np.ldexp(x, e).astype(np.float32), np.zeros_like(x, np.float32)
    for _ in range(parts):
        h = left.astype(np.float16).astype(np.float32)
        out, left = out + h, left - h
    return np.ldexp(out, -e)


def one_head(q, k, v, query_parts, weight_parts):
    """Attention of one head in float32 with the queries and the weights as so many fp16 parts."""
    s = halves(q, query_parts) @ k.T
    w = np.exp(s - s.max(1, keepdims=True))
    return (halves(w, weight_parts) @ v) / w.sum(1, keepdims=True)


@pytest.mark.parametrize("rows", [64, 3000, 10000])
def test_the_limit_needs_both_halves(rows):
    k, v, q = inputs(np.random.default_rng(rows), rows, 1, 200)
    k, v = (P.eleven_bits(a.astype(np.float64)).astype(np.float32) for a in (k, v))
    want = P.attention(q, k, v, 1)
    right = worst_head(one_head(q, k, v, 2, 2), want, 1)
    say(f"  {rows} rows: {right:.1e}, of a limit of {LIMIT:.1e}")
    assert right < LIMIT / 2
    for parts in ((1, 2), (2, 1)):
        short = worst_head(one_head(q, k, v, *parts), want, 1)
        say(f"  query and weight in {parts} parts: {short:.1e}")
        assert short > 4 * LIMIT


# ---- the card ------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def networks(gpu):
    """Networks of one in-context layer by their number of heads of 64."""
    held = {}

    def get(heads):
        if heads not in held:
            cfg = dict(M.FULL_CLASSIFIER, col_num_blocks=1, row_num_blocks=1, icl_num_blocks=1, icl_nhead=heads,
                       row_num_cls=heads // 2)
            held[heads] = gpu.weights(M.Model.random(cfg, seed=5))
        return held[heads]

    yield get
    for w in held.values():
        w.free()


def layer(gpu, w, k, v, chunk):
    """The layer held on the card, and the keys and values that its records stand for."""
    rows, d = k.shape
    kv = dm.DeviceBuffer.of(P.chunk_layout(k, v, chunk))
    size = abi.layer_bytes(abi.KV_I4, rows, chunk, d)
    rec = dm.DeviceBuffer(size)
    gpu.pack_dev(kv.ptr, d, rows, chunk, abi.KV_I4, rec.ptr)
    gpu.sync()
    records = rec.download(size, np.uint8)
    kv.free()
    rec.free()
    return gpu.load(w, abi.KV_I4, rows, chunk, [records], np.ones((1, d), np.float32)), P.unpack_layer(records, d, rows, chunk)


def attend(gpu, vm, q):
    """The outputs, and whether the many-query kernel gave them."""
    gpu.probe_attention(4)
    out = gpu.attend_resident(vm, 0, q)
    launches, _ = gpu.probe_read()
    gpu.probe_attention(0)
    return out, launches == 1


def check(gpu, w, heads, rows, chunk, nq, many, **scales):
    k, v, q = inputs(np.random.default_rng(rows + nq), rows, heads, nq, **scales)
    vm, (k4, v4) = layer(gpu, w, k, v, chunk)
    got, was_many = attend(gpu, vm, q)
    vm.free()
    err = worst_head(got, P.attention(q, k4, v4, heads), heads)
    say(f"  many-query kernel: {was_many}; error {err:.1e}")
    assert was_many == many
    assert err < LIMIT


@pytest.mark.gpu
@pytest.mark.parametrize("heads,rows,chunk,nq", [
    (8, 1, 256, 8192), (8, 64, 256, 8192), (8, 65, 256, 4097),    # one key range, written as it is
    (8, 3000, 256, 1025), (8, 10000, 256, 513), (8, 10000, 256, 600), (8, 10000, 256, 2048),
    (8, 20001, 100, 200),                                         # chunks of two blocks, the second short; a last row alone
    (8, 1000, 48, 2049), (8, 130, 1, 3000),                       # every block short
    (8, 40000, 256, 193), (4, 60000, 256, 250),                   # more than 16 key ranges
    (4, 20001, 1000, 700), (16, 10000, 256, 400)])
def test_many_queries(gpu, networks, heads, rows, chunk, nq):
    say(f"many queries over i4: {heads} heads, {rows} rows in chunks of {chunk}, {nq} queries")
    check(gpu, networks(heads), heads, rows, chunk, nq, True)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,rows,chunk,nq", [
    (8, 1, 256, 1), (8, 1000, 256, 1), (8, 100000, 256, 1), (8, 20001, 100, 13), (8, 50000, 256, 16), (8, 130, 1, 16),
    (8, 64, 256, 17), (4, 5003, 256, 100), (8, 3000, 256, 769), (8, 3000, 256, 2048), (16, 20000, 256, 33), (2, 777, 48, 40)])
def test_fewer_queries(gpu, networks, heads, rows, chunk, nq):
    say(f"few queries over i4: {heads} heads, {rows} rows in chunks of {chunk}, {nq} queries")
    check(gpu, networks(heads), heads, rows, chunk, nq, False)


@pytest.mark.gpu
@pytest.mark.parametrize("k_scale,v_scale", [(2.0 ** 11, 2.0 ** -10), (2.0 ** -40, 2.0 ** 60), (2.0 ** 60, 2.0 ** -60)])
@pytest.mark.parametrize("nq", [5, 40, 1100])
def test_magnitudes(gpu, networks, k_scale, v_scale, nq):
    say(f"magnitudes over i4: keys by {k_scale:.0e}, values by {v_scale:.0e}, {nq} queries")
    check(gpu, networks(8), 8, 3000, 256, nq, nq == 1100, k_scale=k_scale, v_scale=v_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [16, 40, 600])
def test_a_query_that_is_no_number(gpu, networks, nq):
    """A NaN or an infinity in a query: no number for that head of it, and nothing changed in the others."""
    say(f"queries that are no numbers over i4: {nq} queries")
    k, v, q = inputs(np.random.default_rng(nq), 10000, 8, nq)
    vm, _ = layer(gpu, networks(8), k, v, 256)
    want, was_many = attend(gpu, vm, q)
    bad = q.copy()
    bad[3, 70] = np.nan
    bad[nq - 1, 5] = np.inf
    got, _ = attend(gpu, vm, bad)
    vm.free()
    assert was_many == (nq == 600)
    hit = np.zeros(want.shape, bool)
    hit[3, 64:128] = hit[nq - 1, :64] = True
    assert np.all(np.isnan(got[hit])) and np.array_equal(got[~hit], want[~hit])
