"""Keys and values held in 4 bits (`TAH_KV_I4`): the record's sizes and its statement in numpy here on the CPU; packing
(bit for bit), unpacking, the attention over it, the in-context stage and a fit in 4 bits on the card."""
import ctypes
import os

import numpy as np
import pytest

import kv4_plain as P
from conftest import pkg

abi, hip, fit, M, B, C = pkg("abi"), pkg("hip"), pkg("fit"), pkg("model"), pkg("bundle"), pkg("cache")
dm = pkg("devmem")


def say(*a):
    print(*a, flush=True)


# ---- the record, without a card ------------------------------------------------------------------------------------
def test_record_sizes():
    assert abi.kv_record(abi.KV_I4, 512, 256) == 2 * 512 * (16 + 128)  # 4.5 bits a number
    assert abi.kv_record(abi.KV_I4, 16, 1) == 2 * 16 * 5
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libtah_hip.so not built")
    for d, rc in ((512, 256), (512, 100), (16, 1), (16, 63), (16, 64), (16, 65), (7, 129)):
        assert abi.lib().tah_kv_record(abi.KV_I4, d, rc) == abi.kv_record(abi.KV_I4, d, rc) == P.record(d, rc)


@pytest.mark.parametrize("rc", [1, 2, 63, 64, 65, 130])
def test_a_value_is_within_half_a_step(rc):
    rng = np.random.default_rng(rc)
    d = 8
    c = (rng.standard_normal((2 * d, rc)) * rng.uniform(1e-3, 50, (2 * d, 1)) + rng.standard_normal((2 * d, 1)) * 10).astype(np.float32)
    rec = P.pack(c, d, rc)
    assert rec.size == abi.kv_record(abi.KV_I4, d, rc)
    got = P.unpack(rec, d, rc)
    ng = -(-rc // 64)
    steps = (rec[:8 * d * ng].view(np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(2 * d, ng, 2)
    s = steps[:, np.arange(rc) // 64, 0]
    level = np.abs(steps[:, np.arange(rc) // 64, 1]) + 8 * s
    assert np.all(np.abs(got - c) <= s * (0.5 + 2.0 ** -20) + level * 2.0 ** -11)


def test_a_bundle_of_an_unknown_format_is_refused():
    meta = lambda fmt: {"meta": np.array([70, 3, 2, 32, fmt, 1, 1], np.int32), "tree": np.zeros(0, np.int32)}
    with pytest.raises(B.BundleError):
        C.Cache.open(B.Bundle(B.write(None, meta(4))))


def test_null_handles_are_refused():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libtah_hip.so not built")
    l = abi.lib()
    some = ctypes.c_void_p(4096)
    assert l.tah_pack_dev(None, some, 16, 4, 8, abi.KV_I4, some) == abi.E_ARG
    assert l.tah_unpack_dev(None, some, 16, 4, 8, abi.KV_I4, some) == abi.E_ARG
    assert l.tah_unpack(None, None, 16, 4, 8, abi.KV_I4, None) == abi.E_ARG


# ---- the card ------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def gpu():
    g = hip.Gpu(0)
    yield g
    g.close()


def network(heads, layers=1, width=64):
    """A network of in-context layers of `heads` heads of `width`."""
    e = 128 if heads * width % 128 == 0 else 16
    cfg = dict(M.FULL_CLASSIFIER, col_num_blocks=1, row_num_blocks=1, icl_num_blocks=layers, icl_nhead=heads, embed_dim=e,
               row_num_cls=heads * width // e)
    return M.Model.random(cfg, seed=5)


@pytest.fixture(scope="module")
def eight(gpu):
    m = network(8, 2)
    w = gpu.weights(m)
    yield m, w
    w.free()


def values(rng, rows, d):
    """Keys and values [rows][d] each: a mean of its own per coordinate."""
    mean = rng.standard_normal((2, 1, d)) * 0.3
    return (rng.standard_normal((2, rows, d)) * 0.55 + mean).astype(np.float32)


def special_chunk(rng, d, rc):
    c = (rng.standard_normal((2 * d, rc)) * 3 + rng.standard_normal((2 * d, 1))).astype(np.float32)
    c[0] = 0.0                       # a constant group: no step
    c[1] = 1.0 / 3.0                 # a constant that bfloat16 does not hold: a step for the rest of it
    c[2] *= 1e-38                    # below the smallest step
    c[3] *= 1e30
    c[4] = 1000.0 + 0.001 * c[4]     # a small spread about a large mean
    c[5, ::2] = np.nan
    c[6, : (rc + 1) // 2] = np.inf
    c[7] = np.nan                    # nothing finite
    c[8, 0] = -np.inf
    c[9] = np.round(c[9])            # ties between levels
    c[10] = 3.0e38
    c[11] = np.where(np.arange(rc) % 2, 3.4e38, -3.4e38)
    c[12] = -0.0
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("d,rc", [(16, 1), (16, 2), (16, 48), (32, 63), (16, 64), (16, 65), (512, 256), (64, 1000), (7, 129)])
def test_pack_bit_exact(gpu, d, rc):
    say(f"pack i4 d={d} rc={rc}")
    c = special_chunk(np.random.default_rng(d + rc), d, rc)
    got, want = gpu.pack(c, d, rc, abi.KV_I4), P.pack(c, d, rc)
    assert np.all(np.isfinite(P.unpack(want, d, rc)))
    assert np.array_equal(got, want)
    assert np.array_equal(gpu.unpack(got, d, rc, rc, abi.KV_I4).view(np.uint32), P.unpack(want, d, rc).reshape(-1).view(np.uint32))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [abi.KV_F32, abi.KV_I16, abi.KV_I8, abi.KV_I4])
@pytest.mark.parametrize("d,rows,chunk", [(16, 1, 8), (48, 777, 100), (512, 1000, 256), (64, 130, 1), (128, 300, 1000)])
def test_a_layer_on_the_card(gpu, fmt, d, rows, chunk):
    """tah_pack_dev is tah_pack chunk by chunk; tah_unpack_dev what each record stands for; nothing past the ends."""
    say(f"layer fmt={fmt} d={d} rows={rows} chunk={chunk}")
    rng = np.random.default_rng(rows)
    kv = rng.standard_normal(2 * rows * d).astype(np.float32)
    size = abi.layer_bytes(fmt, rows, chunk, d)
    parts, at, want = [], 0, []
    for r0 in range(0, rows, chunk):
        rc = min(chunk, rows - r0)
        parts.append(gpu.pack(kv[at:at + 2 * d * rc], d, rc, fmt))
        if fmt == abi.KV_I4:
            want.append(P.unpack(parts[-1], d, rc).reshape(-1))
        elif fmt == abi.KV_F32:
            want.append(kv[at:at + 2 * d * rc])
        else:
            codes = parts[-1][8 * d:].view(np.int16 if fmt == abi.KV_I16 else np.int8).astype(np.float32)
            want.append((codes.reshape(2 * d, rc) * parts[-1][:8 * d].view(np.float32)[:, None]).reshape(-1))
        at += 2 * d * rc
    records, want = np.concatenate(parts), np.concatenate(want)
    assert records.size == size
    src, dst = dm.DeviceBuffer.of(kv), dm.DeviceBuffer.of(np.full(size + 64, 0xA5, np.uint8))
    back = dm.DeviceBuffer.of(np.full(kv.size + 16, 7.0, np.float32))
    gpu.pack_dev(src.ptr, d, rows, chunk, fmt, dst.ptr)
    gpu.unpack_dev(dst.ptr, d, rows, chunk, fmt, back.ptr)
    gpu.sync()
    got = dst.download(size + 64, np.uint8)
    assert np.array_equal(got[:size], records) and np.all(got[size:] == 0xA5)
    vals = back.download(kv.size + 16)
    assert np.array_equal(vals[:kv.size], want) and np.all(vals[kv.size:] == 7.0)
    assert np.array_equal(gpu.unpack(records, d, rows, chunk, fmt), want)
    for b in (src, dst, back):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [abi.KV_F32, abi.KV_I16, abi.KV_I8, abi.KV_I4])
def test_a_chunk_longer_than_any_table(gpu, fmt):
    """Chunks of up to 2^31 - 1 rows: a shorter table is one chunk of its own length."""
    d, rows = 48, 77
    kv = np.random.default_rng(5).standard_normal(2 * rows * d).astype(np.float32)
    size = abi.layer_bytes(fmt, rows, rows, d)
    src, dst, back = dm.DeviceBuffer.of(kv), dm.DeviceBuffer(size), dm.DeviceBuffer(kv.nbytes)
    got = []
    for chunk in (rows, 2 ** 31 - 1):
        gpu.pack_dev(src.ptr, d, rows, chunk, fmt, dst.ptr)
        gpu.unpack_dev(dst.ptr, d, rows, chunk, fmt, back.ptr)
        gpu.sync()
        got.append((dst.download(size, np.uint8), back.download(kv.size)))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
    assert np.array_equal(got[0][0], gpu.pack(kv, d, rows, fmt))
    for b in (src, dst, back):
        b.free()


@pytest.mark.gpu
def test_layers_refused(gpu):
    b = dm.DeviceBuffer(4096)
    for d, rows, chunk, fmt, ptr in ((0, 4, 8, abi.KV_I4, b.ptr), (16, -1, 8, abi.KV_I4, b.ptr), (16, 4, 0, abi.KV_I4, b.ptr),
                                     (16, 4, 8, 4, b.ptr), (16, 4, 8, -1, b.ptr), (16, 4, 8, abi.KV_I4, b.ptr + 1),
                                     (16, 0, 8, abi.KV_I4, None), (1, 1 << 24, 1, abi.KV_I4, b.ptr + 2),
                                     (1 << 20, 0, 1 << 20, abi.KV_I4, b.ptr)):
        with pytest.raises(ValueError):
            gpu.pack_dev(ptr, d, rows, chunk, fmt, b.ptr)
        with pytest.raises(ValueError):
            gpu.unpack_dev(b.ptr, d, rows, chunk, fmt, ptr)
    gpu.pack_dev(b.ptr, 16, 0, 8, abi.KV_I4, b.ptr)
    gpu.unpack_dev(b.ptr, 16, 0, 8, abi.KV_I4, b.ptr)
    with pytest.raises(ValueError):
        gpu.unpack(np.zeros(100, np.uint8), 16, 4, 8, abi.KV_I4)
    b.free()


def check_attention(gpu, w, heads, rows, chunk, nq, rng, scale=0.4, kv=None, layers=1):
    d = w.model.d
    k, v = values(rng, rows, d) if kv is None else kv
    rec = P.pack_layer(P.chunk_layout(k, v, chunk), d, rows, chunk) if rows * d < 300000 else \
        layer_records(gpu, k, v, chunk)
    k4, v4 = P.unpack_layer(rec, d, rows, chunk)
    vm = gpu.load(w, abi.KV_I4, rows, chunk, [rec] * layers, np.ones((layers, d), np.float32))
    q = (rng.standard_normal((nq, d)) * scale).astype(np.float32)
    got = gpu.attend_resident(vm, layers - 1, q)
    vm.free()
    want = P.attention(q, k4, v4, heads)
    err, bound = np.abs(got - want).max(), P.attention_bound(q, k4, v4, heads)
    say(f"  worst {err:.2e} of {bound:.2e}")
    assert err < bound
    return got


def layer_records(gpu, k, v, chunk):
    """Records packed on the card (checked against the statement above at other sizes)."""
    rows, d = k.shape
    kv = P.chunk_layout(k, v, chunk)
    parts, at = [], 0
    for r0 in range(0, rows, chunk):
        rc = min(chunk, rows - r0)
        parts.append(gpu.pack(kv[at:at + 2 * d * rc], d, rc, abi.KV_I4))
        at += 2 * d * rc
    return np.concatenate(parts)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,chunk", [(1, 256), (2, 8), (63, 64), (65, 256), (300, 100), (1000, 48), (4100, 1000), (10000, 256)])
@pytest.mark.parametrize("nq", [1, 2, 8, 15, 16, 17, 33, 100])
def test_attention(gpu, eight, rows, chunk, nq):
    say(f"attention i4 rows={rows} chunk={chunk} nq={nq}")
    m, w = eight
    check_attention(gpu, w, 8, rows, chunk, nq, np.random.default_rng(rows + nq), layers=2)


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [129, 600, 769, 2048])
def test_attention_many_queries(gpu, eight, nq):
    say(f"attention i4 nq={nq}")
    m, w = eight
    check_attention(gpu, w, 8, 3000, 256, nq, np.random.default_rng(nq), layers=2)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,width", [(2, 64), (4, 64), (16, 64), (8, 16), (4, 32), (2, 8)])
def test_attention_other_heads(gpu, heads, width):
    say(f"attention i4 heads={heads} of {width}")
    w = gpu.weights(network(heads, width=width))
    for rows, chunk, nq in ((777, 100, 1), (777, 256, 20), (70, 8, 5), (300, 256, 140)):
        check_attention(gpu, w, heads, rows, chunk, nq, np.random.default_rng(rows + heads))
    w.free()


@pytest.mark.gpu
@pytest.mark.parametrize("k_scale,v_scale,q_scale", [(2000.0, 1e-3, 1e-4), (1e-3, 2000.0, 300.0), (1.0, 1.0, 8.0), (1e-30, 1e25, 1e28)])
def test_attention_magnitudes(gpu, eight, k_scale, v_scale, q_scale):
    """Keys and values far from 1, sharp weights, one head's far larger than the others'."""
    m, w = eight
    rng = np.random.default_rng(3)
    k, v = values(rng, 500, m.d)
    k, v = k * np.float32(k_scale), v * np.float32(v_scale)
    k[:, :64] *= 16
    v[:, 64:128] *= 100
    for nq in (1, 20, 200):
        check_attention(gpu, w, 8, 500, 256, nq, rng, q_scale, (k, v), layers=2)


@pytest.mark.gpu
def test_stage_and_prediction_over_four_bits(gpu):
    """The whole path: a fit that stores 4 bits, its bundle, the stage and the prediction over it, which are those over
    the f32 records of the values it stands for."""
    m = M.Model.random(M.FULL_CLASSIFIER, seed=2)
    w = gpu.weights(m)
    rng = np.random.default_rng(8)
    x = rng.standard_normal((700, 9)).astype(np.float32)
    y = rng.integers(0, 4, 700).astype(np.float32)
    xt = rng.standard_normal((70, 9)).astype(np.float32)
    f4 = fit.fit_raw(gpu, w, x, y, 4, chunk=256, kv_format=abi.KV_I4)
    f32 = fit.fit_raw(gpu, w, x, y, 4, chunk=256)
    for a, b in zip(f4.layers[0], f32.layers[0]):
        kv = b.view(np.float32)
        assert np.array_equal(a, P.pack_layer(kv, m.d, 700, 256))
    reopened = C.Cache.open(B.Bundle(f4.write()))
    vm = reopened.load(gpu, w)[0]
    plain = [gpu.unpack(r, m.d, 700, 256, abi.KV_I4) for r in f4.layers[0]]
    vp = gpu.load(w, abi.KV_F32, 700, 256, [p.view(np.uint8) for p in plain], f4.scales[0])
    vp.set_columns(f4.col_kv, 9, 1)
    for n in (1, 5, 70):
        a, b = gpu.predict(w, vm, xt[:n], 4), gpu.predict(w, vp, xt[:n], 4)
        err = np.abs(a - b).max()
        say(f"  {n} rows: worst {err:.2e}")
        assert err < 5e-5
    assert vm.bytes() < vp.bytes()
    vm.free()
    vp.free()
    w.free()
