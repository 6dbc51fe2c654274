"""The 4-bit cache and the class statistics as they are used together: a fit in 4 bits served and its answers read as
distributions without leaving the card; the in-context stage without allocating; captured work replayed; two handles at
once; a problem held on the card. Captured work, and the same by another handle, is the eager call's bit for bit."""
import ctypes
import threading

import numpy as np
import pytest

import kv4_plain as P
import test_class_stats as S
from conftest import pkg

abi, hip, fit, M, B, C = pkg("abi"), pkg("hip"), pkg("fit"), pkg("model"), pkg("bundle"), pkg("cache")
T, dm = pkg("table"), pkg("devmem")
pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


def network(layers=1):
    return M.Model.random(dict(M.FULL_CLASSIFIER, col_num_blocks=1, row_num_blocks=1, icl_num_blocks=layers), seed=5)


def records(gpu, rng, rows, chunk, d):
    """A layer's 4-bit records, packed on the card."""
    kv = dm.DeviceBuffer.of((rng.standard_normal(2 * rows * d) * 0.5).astype(np.float32))
    size = abi.layer_bytes(abi.KV_I4, rows, chunk, d)
    rec = dm.DeviceBuffer(size)
    gpu.pack_dev(kv.ptr, d, rows, chunk, abi.KV_I4, rec.ptr)
    gpu.sync()
    out = rec.download(size, np.uint8)
    kv.free()
    rec.free()
    return out


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


def test_fit_serve_and_read_the_answers(gpu):
    """Fit in 4 bits, the bundle reopened, rows predicted and their scores read as distributions with nothing copied to the
    host between; the same by `class_report` from the downloaded scores, and by its definition in 64 bits."""
    m = M.Model.random(M.FULL_CLASSIFIER, seed=2)
    w = gpu.weights(m)
    rng = np.random.default_rng(21)
    x = rng.standard_normal((700, 9)).astype(np.float32)
    y = rng.integers(0, 4, 700).astype(np.float32)
    f = fit.fit_raw(gpu, w, x, y, 4, chunk=256, kv_format=abi.KV_I4)
    vm = C.Cache.open(B.Bundle(f.write())).load(gpu, w)[0]
    held = hip.VramModel.model_bytes(w, abi.KV_I4, 700, 256) + hip.VramModel.columns_bytes(w, 9, 1)
    assert vm.bytes() == held
    for n in (1, 37, 300):
        xt = rng.standard_normal((n, 9)).astype(np.float32)
        labels = rng.integers(0, 4, n).astype(np.int32)
        bx, bl, bo = dm.DeviceBuffer.of(xt), dm.DeviceBuffer.of(labels), dm.DeviceBuffer(n * 16)
        bs, bi = dm.DeviceBuffer(n * 16), dm.DeviceBuffer(n * 8)
        gpu.predict_dev(w, vm, bx.ptr, n, 4, bo.ptr)
        gpu.class_stats_dev(bo.ptr, n, 4, bl.ptr, 1, 2, bs.ptr, bi.ptr, temperature=0.9)
        gpu.sync()
        sums, st, ids = bo.download((n, 4)), bs.download((n, 4)), bi.download((n, 2), np.int32)
        assert np.array_equal(sums, gpu.predict(w, vm, xt, 4))
        want, wids = S.plain(sums, labels[:, None], 2, np.float64(1.0) / np.float64(np.float32(1.0) / np.float32(0.9)))
        assert np.array_equal(ids, wids)
        S.compare(st, want, sums, 0.9)
        rep = T.class_report(sums, 1, 0.9, labels, 2, gpu=gpu)
        assert np.array_equal(rep["top"], ids) and np.array_equal(rep["log_p"], st[:, 1]) and np.array_equal(rep["entropy"], st[:, 0])
        p = T.finish_proba(sums.astype(np.float64), 1, 0.9)
        # a log probability's difference is the probability's relative one; both softmaxes have no more than 2^-18 of it
        assert np.abs(np.exp(rep["log_p"]) - p[np.arange(n), labels]).max() < 2.0 ** -17
        for b in (bx, bl, bo, bs, bi):
            b.free()
    vm.free()
    w.free()


def test_a_held_problem(gpu):
    """A member in 4 bits held on the card: its answers through `CardAttend`, and its bytes among the formats'."""
    m = network(2)
    w = gpu.weights(m)
    rng = np.random.default_rng(4)
    x = rng.standard_normal((500, 5)).astype(np.float32)
    y = rng.integers(0, 3, 500).astype(np.float32)
    f = fit.fit_raw(gpu, w, x, y, 3, chunk=100, kv_format=abi.KV_I4)
    c = C.Cache.open(B.Bundle(f.write()))
    vm = c.load(gpu, w)[0]
    card = hip.CardAttend(gpu, w)
    card.hold("", 0, vm)
    xt = rng.standard_normal((21, 5)).astype(np.float32)
    a = card.rows("", xt, 3)
    assert np.array_equal(a, gpu.predict(w, vm, xt, 3)) and np.all(np.isfinite(a))
    sizes = [hip.VramModel.model_bytes(w, fmt, 500, 100) for fmt in (abi.KV_F32, abi.KV_I16, abi.KV_I8, abi.KV_I4)]
    assert sizes == sorted(sizes, reverse=True)
    up = lambda n: -(-n // 256) * 256
    blocks = 5 * 2  # of 64 keys, chunks of 100 rows
    assert sizes[-1] == 2 * (up(blocks * 8 * 4608) + 256) + up(2 * m.d * 4)  # a layer's tiles and its heads' maxima; the scales
    vm.free()
    w.free()


def test_a_class_tree(gpu):
    """More classes than the network tells apart: every problem of the tree in 4 bits, each its f32 self of the values that
    its records stand for."""
    m = network(2)
    w = gpu.weights(m)
    rng = np.random.default_rng(6)
    x = rng.standard_normal((900, 4)).astype(np.float32)
    y = (np.arange(900) % 25).astype(np.float32)
    f = fit.fit_raw(gpu, w, x, y, 25, chunk=101, kv_format=abi.KV_I4)
    c = C.Cache.open(B.Bundle(f.write()))
    vms = c.load(gpu, w)
    assert len(vms) > 1
    h = (rng.standard_normal((30, m.d)) * 0.5).astype(np.float32)
    for i, vm in enumerate(vms):
        plain = [gpu.unpack(r, m.d, vm.rows, vm.chunk, abi.KV_I4).view(np.uint8) for r in c.layers(i, m.icl_layers)]
        vp = gpu.load(w, abi.KV_F32, vm.rows, vm.chunk, plain, c.scales(i))
        for n in (1, 30):
            a, b = gpu.in_context(w, vm, h[:n], 10), gpu.in_context(w, vp, h[:n], 10)
            say(f"  problem {i}, {vm.rows} rows, {n} queries: worst {np.abs(a - b).max():.2e}")
            assert np.all(np.isfinite(a)) and np.abs(a - b).max() < 5e-5
        vp.free()
        vm.free()
    w.free()


@pytest.mark.parametrize("rows,chunk,calls", [(2000, 256, (256, 4)), (2000, 256, (3, 1)), (40000, 256, (256, 16)), (333, 100, (200, 17))])
def test_stage_without_allocating(gpu, rows, chunk, calls):
    say(f"stage without allocating over i4: {rows} rows, calls of {calls}")
    m = network(2)
    g = hip.Gpu(0)
    w = g.weights(m)
    rng = np.random.default_rng(rows)
    recs = [records(g, rng, rows, chunk, m.d) for _ in range(2)]
    g.release()
    vm = g.load(w, abi.KV_I4, rows, chunk, recs, (0.125 * (1 + 0.1 * rng.standard_normal((2, m.d)))).astype(np.float32))
    h = (rng.standard_normal((max(calls), m.d)) * 0.5).astype(np.float32)
    bh, bo, bp = dm.DeviceBuffer.of(h), dm.DeviceBuffer(max(calls) * 40), dm.DeviceBuffer(max(calls) * 40)
    got = []
    for nq in calls:
        g._check(g._l.tah_stage_dev_noalloc(g._h, w._h, vm._h, ctypes.c_void_p(bh.ptr), nq, 10, ctypes.c_void_p(bo.ptr)))
        g.sync()
        got.append(bo.download((nq, 10)))
        assert g.working() == (0, 0)
    for nq, a in zip(calls, got):
        g.in_context_dev(w, vm, bh.ptr, nq, 10, bp.ptr)
        g.sync()
        assert np.all(np.isfinite(a)) and np.array_equal(a, bp.download((nq, 10)))
    for b in (bh, bo, bp):
        b.free()
    vm.free()
    w.free()
    g.close()


def test_captured_and_replayed(gpu):
    """Two graphs of a handle's calls, which share its working memory, replayed in turns on its stream with new inputs and
    eager work between."""
    m = network()
    d, rows, chunk = m.d, 3001, 100
    w = gpu.weights(m)
    rng = np.random.default_rng(9)
    vm = gpu.load(w, abi.KV_I4, rows, chunk, [records(gpu, rng, rows, chunk, d)], np.ones((1, d), np.float32))
    size = abi.layer_bytes(abi.KV_I4, 130, 100, d)
    kv, rec, back = dm.DeviceBuffer(8 * 130 * d), dm.DeviceBuffer(size), dm.DeviceBuffer(8 * 130 * d)
    q, o1, o40, o300 = (dm.DeviceBuffer(300 * d * 4) for _ in range(4))
    x = [dm.DeviceBuffer(3 * 50000 * 4), dm.DeviceBuffer(200 * 10 * 4), dm.DeviceBuffer(5 * 70000 * 4)]
    shapes = ((3, 50000), (200, 10), (5, 70000))
    given = dm.DeviceBuffer.of(np.arange(200, dtype=np.int32) % 10)
    st = [dm.DeviceBuffer(r * 9 * 4) for r, _ in shapes]
    ids = [dm.DeviceBuffer(r * 7 * 4) for r, _ in shapes]

    def classes(i):
        gpu.class_stats_dev(x[i].ptr, *shapes[i], given.ptr, 1, 7, st[i].ptr, ids[i].ptr, temperature=0.7)

    def first():
        gpu.pack_dev(kv.ptr, d, 130, 100, abi.KV_I4, rec.ptr)
        gpu.unpack_dev(rec.ptr, d, 130, 100, abi.KV_I4, back.ptr)
        gpu.attend_resident_dev(vm, 0, q.ptr, 1, o1.ptr)
        gpu.attend_resident_dev(vm, 0, q.ptr, 300, o300.ptr)
        classes(0)

    def second():
        classes(1)
        gpu.attend_resident_dev(vm, 0, q.ptr, 40, o40.ptr)
        classes(2)

    outs = ((o1, d), (o40, 40 * d), (o300, 300 * d), (back, 260 * d)) + tuple((s, r * 9) for s, (r, _) in zip(st, shapes)) + \
        tuple((i, r * 7) for i, (r, _) in zip(ids, shapes))

    def load():
        kv.upload(rng.standard_normal(260 * d).astype(np.float32))
        q.upload((rng.standard_normal(300 * d) * 0.4).astype(np.float32))
        for b, (r, n) in zip(x, shapes):
            b.upload(rng.standard_normal((r, n)).astype(np.float32) * 3)

    def results():
        gpu.sync()
        return [b.download(n) for b, n in outs]

    load()
    first()  # the working memory is there before the capture
    second()
    gpu.sync()
    a, b = Graph(gpu, first), Graph(gpu, second)
    for turn in range(4):
        load()
        first()
        second()
        want = results()
        assert all(np.all(np.isfinite(v)) for v in want[:7])
        for buf, _ in outs:
            buf.upload(np.full(buf.nbytes // 4, np.nan, np.float32))
        for g in ((a, b), (b, a))[turn % 2]:
            g.replay()
        got = results()
        assert all(np.array_equal(u.view(np.uint32), v.view(np.uint32)) for u, v in zip(got, want))
    a.free()
    b.free()
    for buf in (kv, rec, back, q, o1, o40, o300, given, *x, *st, *ids):
        buf.free()
    vm.free()
    w.free()


def test_two_handles_at_once(gpu):
    """Two handles' calls from two threads, each over its own problem: the results of each alone."""
    m = network()
    d = m.d
    hands = []
    for i, (rows, chunk, nq, n) in enumerate(((9000, 256, 33, 40000), (4001, 100, 1, 3000))):
        g = hip.Gpu(0)
        w = g.weights(m)
        rng = np.random.default_rng(i)
        vm = g.load(w, abi.KV_I4, rows, chunk, [records(g, rng, rows, chunk, d)], np.ones((1, d), np.float32))
        q = (rng.standard_normal((nq, d)) * 0.4).astype(np.float32)
        x = rng.standard_normal((20, n)).astype(np.float32)
        hands.append((g, w, vm, q, x))

    def work(g, w, vm, q, x):
        return [g.attend_resident(vm, 0, q), *g.class_stats(x, None, 30, 0.8)]

    alone = [work(*h) for h in hands]
    got = [[], []]

    def run(i):
        for _ in range(20):
            got[i].append(work(*hands[i]))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20
        for r in got[i]:
            assert all(np.array_equal(u, v) for u, v in zip(r, alone[i]))
    for g, w, vm, *_ in hands:
        vm.free()
        w.free()
        g.close()


def test_no_queries_and_chunks_past_the_table(gpu):
    m = network()
    w = gpu.weights(m)
    rng = np.random.default_rng(2)
    rec = records(gpu, rng, 70, 70, m.d)
    b = dm.DeviceBuffer.of(np.full(m.d, 5.0, np.float32))
    q = (rng.standard_normal((3, m.d)) * 0.4).astype(np.float32)
    got = []
    for chunk in (70, 2 ** 31 - 1):
        vm = gpu.load(w, abi.KV_I4, 70, chunk, [rec], np.ones((1, m.d), np.float32))
        gpu.attend_resident_dev(vm, 0, b.ptr, 0, b.ptr)
        gpu.sync()
        got.append(gpu.attend_resident(vm, 0, q))
        assert gpu.attend_resident(vm, 0, q[:0]).shape == (0, m.d)
        vm.free()
    assert np.all(b.download(m.d) == 5.0) and np.array_equal(got[0], got[1])
    k4, v4 = P.unpack_layer(rec, m.d, 70, 70)
    assert np.abs(got[0] - P.attention(q, k4, v4, 8)).max() < P.attention_bound(q, k4, v4, 8)
    b.free()
    w.free()
