"""The 4-bit record of include/tah.h (`TAH_KV_I4`) stated in numpy, written apart from the library: `pack` (its float32
steps as the header words them, one group at a time), `unpack` (float64, rounded to eleven bits) and attention in
float64."""
import numpy as np

GROUP = 64


def bf16_nearest(x):
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + np.uint32(0x7FFF) + ((u >> 16) & 1)) & np.uint32(0xFFFF0000)).astype(np.uint32).view(np.float32)


def bf16_up(x):
    return ((np.asarray(x, np.float32).view(np.uint32) + np.uint32(0xFFFF)) & np.uint32(0xFFFF0000)).view(np.float32)


def eleven_bits(x):
    """float64 to eleven significant bits, ties to even."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 2048.0), e - 11)


def step_of(v):
    """(s, z) of one group's values [k], float32."""
    f = np.float32
    fin = v[np.isfinite(v)]
    if fin.size == 0:
        return f(0), f(0)
    lo, hi = np.clip(f([fin.min(), fin.max()]), f(-2.0 ** 126), f(2.0 ** 126))
    z = bf16_nearest(f(lo * f(7.0 / 15.0)) + f(hi * f(8.0 / 15.0)) + f(0))
    s = max(f(f(hi - z) * f(1.0 / 7.0)), f(f(z - lo) * f(0.125)))
    return (f(0) if s < 2.0 ** -100 else f(bf16_up(s))), f(z)


def pack(c, d, rc):
    """One chunk's record from c [2d][rc] float32."""
    c = np.asarray(c, np.float32).reshape(2 * d, rc)
    ng = -(-rc // GROUP)
    steps = np.zeros((2 * d, ng, 2), np.float32)
    codes = np.zeros((2 * d, 2 * ((rc + 1) // 2)), np.uint8)
    for j in range(2 * d):
        for g in range(ng):
            v = c[j, g * GROUP:(g + 1) * GROUP]
            s, z = step_of(v)
            steps[j, g] = s, z
            code = np.zeros(v.size)
            if s > 0:
                with np.errstate(over="ignore", invalid="ignore"):
                    code = np.rint((v - z).astype(np.float64) / np.float64(s))
                code = np.clip(np.where(np.isnan(v), 0, code), -8, 7)
            codes[j, g * GROUP:g * GROUP + v.size] = (code + 8).astype(np.uint8)
    head = (steps.view(np.uint32) >> 16).astype(np.uint16)
    return np.concatenate([head.view(np.uint8).reshape(-1), (codes[:, ::2] | (codes[:, 1::2] << 4)).reshape(-1)])


def pack_layer(kv, d, rows, chunk):
    """A layer's records from its values in chunk layout (flat, 2 * rows * d)."""
    parts, at = [], 0
    for r0 in range(0, rows, chunk):
        rc = min(chunk, rows - r0)
        parts.append(pack(kv[at:at + 2 * d * rc], d, rc))
        at += 2 * d * rc
    return np.concatenate(parts)


def unpack(rec, d, rc):
    """What a record stands for, [2d][rc] float32 (exact)."""
    ng = -(-rc // GROUP)
    head = rec[:8 * d * ng].copy().view(np.uint16).astype(np.uint32) << 16
    steps = head.astype(np.uint32).view(np.float32).astype(np.float64).reshape(2 * d, ng, 2)
    b = rec[8 * d * ng:].reshape(2 * d, -1)
    codes = np.stack([b & 15, b >> 4], 2).reshape(2 * d, -1)[:, :rc].astype(np.float64) - 8
    g = np.arange(rc) // GROUP
    return eleven_bits(steps[:, g, 1] + steps[:, g, 0] * codes).astype(np.float32)


def record(d, rc):
    return 2 * d * (4 * (-(-rc // GROUP)) + (rc + 1) // 2)


def unpack_layer(rec, d, rows, chunk):
    """Keys [rows][d] and values [rows][d] of a layer's records."""
    out, at = [], 0
    for r0 in range(0, rows, chunk):
        rc = min(chunk, rows - r0)
        out.append(unpack(rec[at:at + record(d, rc)], d, rc))
        at += record(d, rc)
    kv = np.concatenate(out, 1).T
    return np.ascontiguousarray(kv[:, :d]), np.ascontiguousarray(kv[:, d:])


def chunk_layout(k, v, chunk):
    """Keys and values [rows][d] as flat f32 records."""
    kv = np.concatenate([k, v], 1).astype(np.float32)
    return np.concatenate([np.ascontiguousarray(kv[r0:r0 + chunk].T).reshape(-1) for r0 in range(0, len(kv), chunk)])


def attention(q, k, v, heads):
    """Softmax attention per head in float64, [n][d]."""
    d = q.shape[1]
    hd = d // heads
    out = np.empty(q.shape)
    for h in range(heads):
        at = slice(h * hd, (h + 1) * hd)
        t = q[:, at].astype(np.float64) @ k[:, at].T.astype(np.float64)
        p = np.exp(t - t.max(1, keepdims=True))
        out[:, at] = (p @ v[:, at].astype(np.float64)) / p.sum(1, keepdims=True)
    return out


def attention_bound(q, k, v, heads):
    """How far a float32 evaluation may be off: a score's sum of hd products, each operand within 2^-22 of its value and
    each addition within 2^-24 of the terms' magnitudes; twice that in a weight against its sum; the weights' exponentials
    and the sums over the rows, whose roundings are independent (four standard deviations)."""
    d, hd = q.shape[1], q.shape[1] // heads
    worst = 0.0
    for h in range(heads):
        at = slice(h * hd, (h + 1) * hd)
        t = (np.abs(q[:, at]).max(0) * np.abs(k[:, at]).max(0)).sum()
        score = t * (2.0 ** -22 + hd * 2.0 ** -24)
        worst = max(worst, np.abs(v[:, at]).max() * (2 * score + (8 + 4 * np.sqrt(len(k))) * 2.0 ** -24))
    return worst
