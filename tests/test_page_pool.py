"""`pages.PagePool`: which pages are whose, on the host with a stand-in for the card; and on the card, problems held from a fit's
records, served together and grown, against the models the card holds whole and the operators' statement."""
import threading

import numpy as np
import pytest

import pages_plain as P
from conftest import pkg

abi, hip, pages, devmem = pkg("abi"), pkg("hip"), pkg("pages"), pkg("devmem")


class Memory:
    """Stands in for a DeviceBuffer."""

    def __init__(self, nbytes):
        self.nbytes, self.ptr = nbytes, 1 << 20

    def free(self):
        self.ptr = None


class Card:
    """Stands in for a Gpu: a dict of rows by (pool address, page, slot)."""

    def __init__(self):
        self.rows, self.calls, self.fail = {}, [], False

    def places(self, p, table, starts, offsets):
        for t in range(p.tables):
            for i in range(offsets[t + 1] - offsets[t]):
                at = starts[t] + i
                yield p.pool, int(table[t][at // p.page_rows]), at % p.page_rows

    def pages_write(self, p, table, starts, offsets, k, v):
        if self.fail and self.fail == p.pool:
            raise hip.CardError("graphics card: gone")
        for r, place in enumerate(self.places(p, table, starts, offsets)):
            assert 0 <= place[1] < p.pages
            self.rows[place] = (k[r], v[r])

    def pages_read(self, p, table, starts, offsets):
        got = [self.rows[place] for place in self.places(p, table, starts, offsets)]
        return tuple(np.array([g[i] for g in got]).reshape(len(got), -1) for i in (0, 1))

    def pages_attend(self, p, table, lengths, q, offsets, heads, causal):
        self.calls.append((p.pool, table.copy(), list(lengths), q.shape, list(offsets), heads, causal))
        return np.arange(q.size, dtype=np.float32).reshape(q.shape)


@pytest.fixture
def pool(monkeypatch):
    if not __import__("os").path.exists(abi.LIB_PATH):
        pytest.skip("libtah_hip.so not built")
    monkeypatch.setattr(devmem, "DeviceBuffer", Memory)
    return pages.PagePool(Card(), layers=2, heads=2, hd=16, pages=10, page_rows=16)


def kv(n, seed=0, layers=2, d=32):
    rng = np.random.default_rng(seed)
    return [tuple(rng.standard_normal((2, n, d)).astype(np.float32)) for _ in range(layers)]


def same(pool, name, layers):
    for l, (k, v) in enumerate(layers):
        gk, gv = pool.read(*name, l)
        assert np.array_equal(gk, k) and np.array_equal(gv, v)


def test_held_grown_dropped(pool):
    a, b, more = kv(20, 1), kv(1, 2), kv(13, 3)
    pool.hold("a", 0, a)
    pool.hold("b", 3, b)
    assert (pool.rows("a", 0), pool.rows("b", 3), pool.rows("c", 0), pool.free_pages) == (20, 1, 0, 7)
    pool.grow("a", 0, more)  # 33 rows: a third page
    assert pool.rows("a", 0) == 33 and pool.free_pages == 6
    same(pool, ("a", 0), [tuple(np.concatenate(x) for x in zip(p, q)) for p, q in zip(a, more)])
    same(pool, ("b", 3), b)
    pool.grow("b", 3, kv(15, 4))  # fills its page
    assert pool.free_pages == 6
    pool.grow("b", 3, kv(0))
    assert pool.rows("b", 3) == 16
    assert pool.drop("a", 0) and not pool.drop("a", 0)
    assert pool.free_pages == 9 and pool.rows("a", 0) == 0
    pool.hold("b", 3, kv(144, 5))  # in place of what it was: all pages but one were free
    assert pool.free_pages == 1
    same(pool, ("b", 3), kv(144, 5))


def test_too_few_pages_change_nothing(pool):
    a = kv(100, 1)
    pool.hold("a", 0, a)
    with pytest.raises(hip.BudgetError):
        pool.hold("b", 0, kv(49))
    with pytest.raises(hip.BudgetError):
        pool.grow("a", 0, kv(61))
    with pytest.raises(hip.BudgetError):
        pool.hold("a", 0, kv(161))
    assert (pool.rows("a", 0), pool.rows("b", 0), pool.free_pages) == (100, 0, 3)
    same(pool, ("a", 0), a)
    pool.hold("a", 0, kv(160, 7))
    assert pool.free_pages == 0


def test_a_failed_write_gives_its_pages_back(pool):
    a = kv(20, 1)
    pool.hold("a", 0, a)
    pool.gpu.fail = pool._memory.ptr + pool.layer_bytes  # the second layer's
    with pytest.raises(hip.CardError):
        pool.grow("a", 0, kv(20, 2))
    pool.gpu.fail = False
    assert pool.rows("a", 0) == 20 and pool.free_pages == 8
    same(pool, ("a", 0), a)
    pool.gpu.fail = pool._memory.ptr
    with pytest.raises(hip.CardError):
        pool.hold("b", 0, kv(20, 2))
    assert pool.free_pages == 8 and pool.attend("b", 0, 0, np.zeros((1, 32), np.float32), 32, 2) is None


def test_questions_of_many_problems(pool):
    pool.hold("a", 0, kv(20))
    pool.hold("b", 0, kv(40))
    pool.hold("none", 0, kv(0))
    q = np.zeros((3, 64), np.float32)
    out = pool.attend_many(1, [("b", 0, q), ("none", 0, q[:1]), ("a", 0, q[:2])], heads=4, causal=True)
    assert [o.shape for o in out] == [(3, 64), (1, 64), (2, 64)] and out[2][0, 0] == 4 * 64
    address, table, lengths, shape, offsets, heads, causal = pool.gpu.calls[-1]
    assert address == pool._memory.ptr + pool.layer_bytes and lengths == [40, 0, 20] and offsets == [0, 3, 4, 6] and causal
    assert table.shape == (3, 3) and np.all(table[1] == -1) and table[2, 2] == -1 and np.all(table[0] >= 0)
    assert pool.attend_many(0, [], heads=2) == []
    assert pool.attend("a", 0, 0, q, 64, 4).shape == (3, 64)
    assert pool.attend("c", 0, 0, q, 64, 4) is None and pool.attend("a", 0, 0, q, 48, 3) is None
    assert pool.attend("a", 0, 2, q, 64, 4) is None and pool.attend("a", 0, 0, q, 60, 4) is None


def test_refusals(pool):
    pool.hold("a", 0, kv(20))
    for layers in (kv(5)[:1], kv(5) + kv(5), [kv(5)[0], kv(6)[0]], [kv(5)[0], (kv(5)[0][0],)], kv(5, d=31)):
        with pytest.raises(ValueError):
            pool.hold("b", 0, layers)
        with pytest.raises(ValueError):
            pool.grow("a", 0, layers)
    for call in (lambda: pool.grow("b", 0, kv(1)), lambda: pool.read("b", 0, 0),
                 lambda: pool.attend_many(0, [("b", 0, np.zeros((1, 32), np.float32))], 2)):
        with pytest.raises(LookupError):
            call()
    for call in (lambda: pool.read("a", 0, 2), lambda: pool.attend_many(-1, [("a", 0, np.zeros((1, 32), np.float32))], 2),
                 lambda: pool.attend_many(0, [("a", 0, np.zeros((1, 31), np.float32))], 2)):
        with pytest.raises(ValueError):
            call()
    for bad in (dict(layers=0), dict(pages=0), dict(hd=24), dict(heads=0), dict(page_rows=24), dict(kv_format=abi.KV_I4)):
        with pytest.raises(ValueError):
            pages.PagePool(Card(), **{**dict(layers=2, heads=2, hd=16, pages=10, page_rows=16), **bad})
    assert pool.free_pages == 8 and pool.rows("a", 0) == 20


# ---- on the card --------------------------------------------------------------------------------------------------------------
def records(rng, rows, chunk, d, layers):
    """Layers' f32 records, and their keys and values [rows][d]."""
    out = []
    for _ in range(layers):
        k, v = (rng.standard_normal((2, rows, d)) * 0.5).astype(np.float32)
        rec = np.concatenate([np.concatenate([k[a:a + chunk].T.reshape(-1), v[a:a + chunk].T.reshape(-1)]) for a in range(0, rows, chunk)])
        out.append((rec.view(np.uint8), k, v))
    return out


@pytest.mark.gpu
def test_problems_from_records_served_together_and_grown():
    """Problems put into pages from their stored records answer as the models that the card holds whole do; then they grow, and
    answer as the operators' statement says."""
    M = pkg("model")
    gpu = hip.Gpu(0)
    m = M.Model.random(dict(M.FULL_CLASSIFIER, col_num_blocks=1, row_num_blocks=1, icl_num_blocks=2), seed=5)
    w = gpu.weights(m)
    rng = np.random.default_rng(3)
    d, heads, chunk = m.d, 8, 48
    pool = pages.PagePool(gpu, layers=2, heads=heads, hd=d // heads, pages=40, kv_format=abi.KV_F32, page_rows=32)
    card, asked = hip.CardAttend(gpu, w), []
    made = {("a", 0): 333, ("a", 1): 17, ("b", 0): 100}
    kvs = {}
    for (prefix, node), rows in made.items():
        layers = records(rng, rows, chunk, d, 2)
        kvs[(prefix, node)] = [(k, v) for _, k, v in layers]
        pool.hold_records(prefix, node, abi.KV_F32, rows, chunk, [rec for rec, _, _ in layers])
        card.hold(prefix, node, gpu.load(w, abi.KV_F32, rows, chunk, [rec for rec, _, _ in layers], np.ones((2, d), np.float32)))
        asked.append((prefix, node, (rng.standard_normal((int(rng.integers(1, 5)), d)) * 0.4).astype(np.float32)))
        assert all(np.array_equal(a, b) for a, b in zip(pool.read(prefix, node, 1), kvs[(prefix, node)][1]))
    for layer in range(2):
        together = pool.attend_many(layer, asked, heads)
        for (prefix, node, q), got in zip(asked, together):
            one = card.attend(prefix, node, layer, q, d, heads)
            size = np.sqrt(np.mean(np.square(one)))
            assert np.sqrt(np.mean(np.square(got - one))) <= 2.0**-19 * size  # each 2^-20 from 64 bits
            assert np.sqrt(np.mean(np.square(pool.attend(prefix, node, layer, q, d, heads) - one))) <= 2.0**-19 * size
    assert pool.attend("b", 1, 0, asked[0][2], d, heads) is None
    free = pool.free_pages
    pool.drop("a", 1)
    for name in (("a", 0), ("b", 0)):
        more = [(k, v) for _, k, v in records(rng, 40, 40, d, 2)]
        pool.grow(*name, more)
        kvs[name] = [tuple(np.concatenate(x) for x in zip(p, q)) for p, q in zip(kvs[name], more)]
    assert free - pool.free_pages == 1  # one page back, and for 373 and 140 rows one each
    for layer in range(2):
        q = {name: (rng.standard_normal((3, d)) * 0.4).astype(np.float32) for name in (("a", 0), ("b", 0))}
        got = pool.attend_many(layer, [(*name, a) for name, a in q.items()], heads, causal=True)
        for (name, a), o in zip(q.items(), got):
            k, v = (x.reshape(len(x), heads, -1) for x in kvs[name][layer])
            out, off = P.attention(a.reshape(3, heads, -1), k, v, P.limits_of(len(k), 3, True))
            assert np.all(np.abs(o.reshape(out.shape) - out) <= off)
    pool.free()
    gpu.close()


@pytest.mark.gpu
def test_two_threads_share_a_pool():
    """One thread's problem grows while another's answers: every answer is of the rows it had."""
    gpu = hip.Gpu(0)
    d, heads = 128, 2
    pool = pages.PagePool(gpu, layers=1, heads=heads, hd=64, pages=64, kv_format=abi.KV_F32, page_rows=16)
    rng = np.random.default_rng(8)
    k, v, q = (rng.standard_normal((3, 300, d)) * 0.4).astype(np.float32)
    pool.hold("still", 0, [(k[:77], v[:77])])
    pool.hold("grows", 0, [(k[:1], v[:1])])
    want = pool.attend("still", 0, 0, q[:2], d, heads)
    wrong = []

    def grow():
        for i in range(1, 300):
            pool.grow("grows", 0, [(k[i:i + 1], v[i:i + 1])])

    def ask():
        for _ in range(200):
            if not np.array_equal(pool.attend("still", 0, 0, q[:2], d, heads), want):
                wrong.append(1)

    threads = [threading.Thread(target=f) for f in (grow, ask)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and pool.rows("grows", 0) == 300
    gk, gv = pool.read("grows", 0, 0)
    assert np.array_equal(gk, k) and np.array_equal(gv, v)
    pool.free()
    gpu.close()


@pytest.mark.parametrize("error", [hip.CardError, hip.BudgetError])
def test_a_replacement_that_fails_leaves_what_was_held(pool, error):
    """Where enough pages are free for the new rows beside the old ones; else the old ones' pages are taken first."""
    a = kv(40, 1)
    pool.hold("a", 0, a)
    write, layer = pool.gpu.pages_write, []

    def fails_at_the_second_layer(p, *args):
        layer.append(p.pool)
        if p.pool != pool._memory.ptr:
            raise error("graphics card: gone")
        write(p, *args)

    pool.gpu.pages_write = fails_at_the_second_layer
    with pytest.raises(error):
        pool.hold("a", 0, kv(112, 2))  # seven pages, as many as are free
    assert len(layer) == 2 and pool.rows("a", 0) == 40 and pool.free_pages == 7
    same(pool, ("a", 0), a)
    with pytest.raises(error):
        pool.hold("a", 0, kv(113, 2))
    assert pool.rows("a", 0) == 0 and pool.free_pages == 10
    pool.gpu.pages_write = write
    pool.hold("a", 0, kv(160, 3))
    same(pool, ("a", 0), kv(160, 3))
