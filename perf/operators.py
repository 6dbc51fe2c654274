"""Measurement cases of the 4-bit cache and of the class statistics, with their plain forms.

Kinds of case (`op`):

* `attend`: scaled queries over one in-context layer held in 4 bits (`Gpu.attend_resident_dev` over a `TAH_KV_I4` model);
* `store`: a layer's exact keys and values to 4-bit records and back to the values they stand for (`Gpu.pack_dev`,
  `Gpu.unpack_dev`), what a fit stores and what a prediction, or a bundle in another format, then reads;
* `scores`: rows of class scores read as distributions (`Gpu.class_stats_dev`): entropy, log probabilities of given
  classes, the most probable classes, at a softmax temperature; a score of -inf is a class ruled out.

A 4-bit record holds a chunk of rc rows: for each of the 2d coordinates (keys, then values) and each group of 64 rows a
step s and an offset z in bfloat16, then two codes a byte, the even row's in the low bits, each code c in -8..7 stored as
c + 8. It stands for z + s c, rounded to eleven significant bits.

Keys and values are what a layer norm and a projection leave: a mean of its own per coordinate, spread 0.55. Queries are
already scaled. Everything is made from the seed on the card.
"""
import functools
import importlib
import math

import numpy as np
import torch

own = False

GROUP = 64        # rows that share a step and an offset
HEAD = 64         # head width
SMALLEST = 2.0 ** -100  # steps below it are held as 0
TEMPERATURE = 0.9


def listed():
    return [
        # one row answered at once against a small table's cache: latency
        {"name": "attend_1x1000", "op": "attend", "n": 1, "rows": 1000, "chunk": 256, "heads": 8},
        # one row against a long cache: the cache's bytes
        {"name": "attend_1x100000", "op": "attend", "n": 1, "rows": 100000, "chunk": 256, "heads": 8},
        # a serving loop's small batch, chunks that end inside a group, a last chunk of one row
        {"name": "attend_13x20001", "op": "attend", "n": 13, "rows": 20001, "chunk": 100, "heads": 8},
        # a middling batch on a narrower network
        {"name": "attend_100x5003", "op": "attend", "n": 100, "rows": 5003, "chunk": 256, "heads": 4},
        # the benchmark's batch and table
        {"name": "attend_2048x10000", "op": "attend", "n": 2048, "rows": 10000, "chunk": 256, "heads": 8},
        # a long table scored in one call
        {"name": "attend_1000x40000", "op": "attend", "n": 1000, "rows": 40000, "chunk": 256, "heads": 8},
        # a small problem of a class tree, odd chunks
        {"name": "store_333", "op": "store", "rows": 333, "chunk": 101, "d": 512},
        # the benchmark's table, one layer
        {"name": "store_10000", "op": "store", "rows": 10000, "chunk": 256, "d": 512},
        # an ordinary answer: a batch of ten classes, its labels scored, the two best kept
        {"name": "scores_2048x10", "op": "scores", "rows": 2048, "n": 10, "given": 1, "top": 2, "masked": 0.0},
        # a whole table's answers, some classes ruled out beforehand (in a few rows all of them)
        {"name": "scores_200000x7", "op": "scores", "rows": 200000, "n": 7, "given": 1, "top": 3, "masked": 0.2},
        # a class tree's leaves
        {"name": "scores_3000x1001", "op": "scores", "rows": 3000, "n": 1001, "given": 2, "top": 10, "masked": 0.0},
        # few rows of very many classes
        {"name": "scores_64x100000", "op": "scores", "rows": 64, "n": 100000, "given": 1, "top": 20, "masked": 0.0},
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attend", "attend", "attend", "store", "scores", "scores"])
    if op == "attend":
        rows, heads = between(200, 100000), rng.choice([4, 8, 8, 16])
        n = between(1, 2048)
        return {"op": op, "n": max(1, min(n, 20480000 // rows * 8 // heads)), "rows": rows, "chunk": rng.choice([256, 256, 256, 100, 1000]),
                "heads": heads}
    if op == "store":
        d = rng.choice([256, 512, 512, 1024])
        return {"op": op, "rows": min(between(50, 40000), 20480000 // d), "chunk": rng.choice([256, 256, 101, 1000]), "d": d}
    n = between(2, 100000)
    return {"op": op, "rows": between(1, max(1, min(200000, 6400000 // n))), "n": n, "given": rng.randint(0, 3),
            "top": min(n, rng.choice([0, 1, 3, 5, 20])), "masked": rng.choice([0.0, 0.0, 0.3])}


# ---- what a program has in hand ---------------------------------------------------------------------------------------
def generator(*key):
    return torch.Generator(device="cuda").manual_seed(hash(key) & 0x7FFFFFFF)


def layer_values(rows, d, seed):
    """A layer's exact keys and values, [2d][rows]."""
    g = generator(seed, 1)
    mean = torch.randn(2 * d, 1, device="cuda", generator=g) * 0.3
    return torch.randn(2 * d, rows, device="cuda", generator=g) * 0.55 + mean


def chunked(kv, chunk):
    """[2d][rows] in the stored order: whole chunks [chunks][2d][chunk] and the short last one [1][2d][rest] (either may be
    empty)."""
    full = kv.shape[1] // chunk
    head = kv[:, :full * chunk].reshape(kv.shape[0], full, chunk).permute(1, 0, 2).contiguous()
    return head, kv[:, full * chunk:].unsqueeze(0).contiguous()


@functools.lru_cache(maxsize=None)
def card():
    return importlib.import_module("tabicl-anywhere_amd.hip").Gpu(0)


@functools.lru_cache(maxsize=None)
def weights(heads):
    """A network with one in-context layer of this many heads of 64."""
    m = importlib.import_module("tabicl-anywhere_amd.model")
    cfg = dict(m.FULL_CLASSIFIER, col_num_blocks=1, row_num_blocks=1, icl_num_blocks=1, icl_nhead=heads,
               row_num_cls=heads * HEAD // 128)
    return card().weights(m.Model.random(cfg, seed=2))


def prepare(case, seed):
    op = case["op"]
    s = {"case": case}
    if op == "scores":
        g = generator(seed, 2)
        hidden = torch.rand(case["rows"], case["n"], device="cuda", generator=g) < case["masked"]
        spread = torch.rand(case["rows"], 1, device="cuda", generator=g) * 5.0 + 0.5
        s["x"] = torch.randn(case["rows"], case["n"], device="cuda", generator=g) * spread
        s["x"][hidden] = -math.inf
        s["given"] = torch.randint(0, case["n"], (case["rows"], case["given"]), device="cuda", generator=g, dtype=torch.int32)
        s["stats"] = torch.empty(case["rows"], 1 + case["given"] + case["top"], device="cuda")
        s["ids"] = torch.empty(case["rows"], case["top"], device="cuda", dtype=torch.int32)
    elif op == "store":
        s["kv"] = torch.cat([c.reshape(-1) for c in chunked(layer_values(case["rows"], case["d"], seed), case["chunk"])])
        s["records"] = torch.empty(layer_bytes(case["rows"], case["chunk"], case["d"]), device="cuda", dtype=torch.uint8)
        s["out"] = torch.empty_like(s["kv"])
    else:
        d = case["heads"] * HEAD
        s["records"] = plain_pack(chunked(layer_values(case["rows"], d, seed), case["chunk"]))
        s["q"] = torch.randn(case["n"], d, device="cuda", generator=generator(seed, 3)) * 0.4
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["gpu"] = card()
        if op == "attend":
            kv_i4 = importlib.import_module("tabicl-anywhere_amd.abi").KV_I4
            s["model"] = card().load(weights(case["heads"]), kv_i4, case["rows"], case["chunk"], [s["records"].cpu().numpy()],
                                     np.ones((1, d), np.float32))
    torch.cuda.synchronize()
    return s


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        gpu = state["gpu"]
        if op == "attend":
            gpu.attend_resident_dev(state["model"], 0, state["q"].data_ptr(), case["n"], state["out"].data_ptr())
            return state["out"]
        if op == "store":
            kv_i4 = importlib.import_module("tabicl-anywhere_amd.abi").KV_I4
            gpu.pack_dev(state["kv"].data_ptr(), case["d"], case["rows"], case["chunk"], kv_i4, state["records"].data_ptr())
            gpu.unpack_dev(state["records"].data_ptr(), case["d"], case["rows"], case["chunk"], kv_i4, state["out"].data_ptr())
            return state["out"]
        gpu.class_stats_dev(state["x"].data_ptr(), case["rows"], case["n"], state["given"].data_ptr(), case["given"], case["top"],
                            state["stats"].data_ptr(), state["ids"].data_ptr(), temperature=TEMPERATURE)
        return {"stats": state["stats"], "ids": state["ids"]}
    if op == "attend":
        return plain_attend(state["q"], state["records"], case["rows"], case["chunk"], case["heads"])
    if op == "store":
        return plain_unpack(plain_pack(stored_chunks(state["kv"], case["rows"], case["chunk"], case["d"])), case["rows"],
                            case["chunk"], case["d"])
    return plain_scores(state["x"], state["given"], case["top"])


# ---- plain forms ------------------------------------------------------------------------------------------------------
def record_bytes(rc, d):
    return 2 * d * (4 * (-(-rc // GROUP)) + (rc + 1) // 2)


def layer_bytes(rows, chunk, d):
    return rows // chunk * record_bytes(chunk, d) + (record_bytes(rows % chunk, d) if rows % chunk else 0)


def stored_chunks(flat, rows, chunk, d):
    """Values in the stored order as `chunked` gives them."""
    full = rows // chunk
    at = full * chunk * 2 * d
    return flat[:at].view(full, 2 * d, chunk), flat[at:].view(1, 2 * d, rows % chunk)


def eleven_bits(v):
    """v rounded to eleven significant bits, ties to even."""
    u = v.view(torch.int32)
    return ((u + 0xFFF + ((u >> 13) & 1)) & -0x2000).view(torch.float32)


def pack_chunks(c):
    """Chunks [chunks][2d][rc] as records, flat."""
    n, d2, rc = c.shape
    if n == 0 or rc == 0:
        return torch.empty(0, dtype=torch.uint8, device=c.device)
    groups = -(-rc // GROUP)
    pad = groups * GROUP - rc
    # short groups padded with their own last row, which changes no minimum and no maximum
    v = torch.cat([c, c[..., -1:].expand(n, d2, pad)], 2).view(n, d2, groups, GROUP)
    lo, hi = v.amin(3), v.amax(3)
    z = (lo * (7.0 / 15.0) + hi * (8.0 / 15.0)).to(torch.bfloat16)
    zf = z.float()
    s = torch.maximum((hi - zf) * (1.0 / 7.0), (zf - lo) * 0.125)
    s = torch.where(s < SMALLEST, torch.zeros_like(s), s)
    s = ((s.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)  # up to the next bfloat16
    code = torch.round((v - zf[..., None]) / torch.where(s > 0, s, torch.ones_like(s))[..., None]).clamp(-8, 7)
    code = torch.where(s[..., None] > 0, code, torch.zeros_like(code)).to(torch.int32).view(n, d2, -1)[..., :rc] + 8
    code = torch.cat([code, torch.zeros(n, d2, rc % 2, dtype=torch.int32, device=c.device)], 2)
    pairs = (code[..., ::2] | (code[..., 1::2] << 4)).to(torch.uint8)
    steps = torch.stack([s.to(torch.bfloat16), z], 3).view(torch.uint8).reshape(n, -1)
    return torch.cat([steps, pairs.reshape(n, -1)], 1).reshape(-1)


def plain_pack(chunks):
    return torch.cat([pack_chunks(chunks[0]), pack_chunks(chunks[1])])


def unpack_chunks(rec, n, rc, d):
    """n records of rc rows as values [n][2d][rc]."""
    if n == 0 or rc == 0:
        return torch.empty(n, 2 * d, rc, device=rec.device)
    groups = -(-rc // GROUP)
    rec = rec.view(n, record_bytes(rc, d))
    steps = rec[:, :8 * d * groups].contiguous().view(torch.bfloat16).float().view(n, 2 * d, groups, 2)
    pairs = rec[:, 8 * d * groups:].contiguous().view(n, 2 * d, -1)
    code = torch.stack([pairs & 15, pairs >> 4], 3).view(n, 2 * d, -1)[..., :rc].float() - 8.0
    at = torch.arange(rc, device=rec.device) // GROUP
    return eleven_bits(steps[..., 1][..., at] + steps[..., 0][..., at] * code)


def unpacked(records, rows, chunk, d):
    full = rows // chunk
    at = full * record_bytes(chunk, d)
    return unpack_chunks(records[:at], full, chunk, d), unpack_chunks(records[at:], 1, rows % chunk, d)


def plain_unpack(records, rows, chunk, d):
    head, tail = unpacked(records, rows, chunk, d)
    return torch.cat([head.reshape(-1), tail.reshape(-1)])


def plain_attend(q, records, rows, chunk, heads):
    d = heads * HEAD
    head, tail = unpacked(records, rows, chunk, d)
    kv = torch.cat([head.permute(1, 0, 2).reshape(2 * d, -1), tail[0]], 1)
    k, v = kv[:d].view(heads, HEAD, rows), kv[d:].view(heads, HEAD, rows)
    t = torch.matmul(q.view(-1, heads, HEAD).transpose(0, 1).contiguous(), k)
    p = torch.exp(t - t.amax(2, keepdim=True))
    o = torch.matmul(p, v.transpose(1, 2).contiguous()) / p.sum(2, keepdim=True)
    return o.transpose(0, 1).reshape(q.shape)


def plain_scores(x, given, top):
    order, ids = torch.sort(x, dim=1, descending=True, stable=True)
    # a row without a class left: every log probability -inf, entropy 0
    best = torch.where(order[:, :1] == -math.inf, torch.zeros_like(order[:, :1]), order[:, :1])
    t = (x - best) * (1.0 / TEMPERATURE)
    e = torch.exp(t)
    total = e.sum(1, keepdim=True)
    logs = torch.log(torch.where(total > 0, total, torch.ones_like(total)))
    entropy = logs - torch.where(e > 0, e * t, torch.zeros_like(t)).sum(1, keepdim=True) / total.clamp(min=1.0)
    logp = t - logs
    return {"stats": torch.cat([entropy, torch.gather(logp, 1, given.long()), torch.gather(logp, 1, ids[:, :top])], 1),
            "ids": ids[:, :top].to(torch.int32)}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    op, rows = case["op"], case["rows"]
    if op == "attend":
        d = case["heads"] * HEAD
        return {"bytes": layer_bytes(rows, case["chunk"], d) + 8.0 * case["n"] * d, "flops": 4.0 * case["n"] * rows * d}
    if op == "store":
        # the values in, the records out, the records in and the values out; subtract, divide, round a value and one
        # multiply-add back, and its part of the minimum and maximum
        d = case["d"]
        return {"bytes": 16.0 * rows * d + 2.0 * layer_bytes(rows, case["chunk"], d), "flops": 14.0 * rows * d}
    # a score's difference, exponential, two sums and a product
    return {"bytes": 4.0 * rows * (case["n"] + 1 + 2 * case["given"] + 2 * case["top"]), "flops": 5.0 * rows * case["n"]}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def exact_values(raw, rows, chunk, d):
    """What records (bytes in host memory) stand for, [2d][rows] float64."""
    out, at = np.empty((2 * d, rows)), 0
    for r0 in range(0, rows, chunk):
        rc = min(chunk, rows - r0)
        groups = -(-rc // GROUP)
        steps = (raw[at:at + 8 * d * groups].view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        steps = steps.reshape(2 * d, groups, 2)
        at += 8 * d * groups
        pairs = raw[at:at + d * 2 * ((rc + 1) // 2)].reshape(2 * d, -1)
        at += pairs.size
        for r in range(rc):
            c = ((pairs[:, r // 2] >> (4 * (r & 1))) & 15).astype(np.float64) - 8.0
            out[:, r0 + r] = steps[:, r // GROUP, 1] + steps[:, r // GROUP, 0] * c
    m, e = np.frexp(out)
    return np.ldexp(np.round(m * 2048.0), e - 11)


def exact_store(kv, rows, chunk, d):
    """Values [2d][rows] (float32, host) to what their records stand for, in the stored order."""
    f = np.float32
    parts = []
    for r0 in range(0, rows, chunk):
        c = kv[:, r0:min(r0 + chunk, rows)]
        got = np.empty(c.shape)
        for g in range(0, c.shape[1], GROUP):
            v = c[:, g:g + GROUP]
            lo, hi = v.min(1), v.max(1)
            # the offset and the step are defined by these float32 operations
            z = lo * f(7.0 / 15.0) + hi * f(8.0 / 15.0)
            u = z.view(np.uint32)
            z = ((u + 0x7FFF + ((u >> 16) & 1)) & np.uint32(0xFFFF0000)).view(f)
            s = np.maximum((hi - z) * f(1.0 / 7.0), (z - lo) * f(0.125))
            s[s < SMALLEST] = 0.0
            s = ((s.view(np.uint32) + np.uint32(0xFFFF)) & np.uint32(0xFFFF0000)).view(f)
            r = (v - z[:, None]).astype(np.float64)
            wide = s[:, None].astype(np.float64)
            code = np.clip(np.rint(np.divide(r, wide, out=np.zeros_like(r), where=wide > 0)), -8, 7)
            m, e = np.frexp(z[:, None].astype(np.float64) + wide * code)
            got[:, g:g + GROUP] = np.ldexp(np.round(m * 2048.0), e - 11)
        parts.append(got.reshape(-1))
    return np.concatenate(parts)


def exact_attention(q, kv, heads):
    """Softmax attention of q [n][d] over kv [2d][rows], float64 on the card, a head at a time."""
    d = q.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for h in range(heads):
        at = slice(h * HEAD, (h + 1) * HEAD)
        p = torch.softmax(q[:, at].double() @ kv[:d][at], 1)
        out[:, at] = p @ kv[d:][at].T.contiguous()
    return out


def exact_scores(x, given, top):
    x = x.double()
    logp = torch.log_softmax(x / TEMPERATURE, 1)
    logp = torch.where((x == -math.inf).all(1, keepdim=True), x, logp)
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1, keepdim=True)
    ids = torch.argsort(x, dim=1, descending=True, stable=True)[:, :top]
    return {"stats": torch.cat([entropy, logp.gather(1, given.long()), logp.gather(1, ids)], 1), "ids": ids.to(torch.int32)}


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "attend":
        d = case["heads"] * HEAD
        kv = torch.from_numpy(exact_values(s["records"].cpu().numpy(), case["rows"], case["chunk"], d)).cuda()
        return exact_attention(s["q"], kv, case["heads"])
    if op == "store":
        kv = layer_values(case["rows"], case["d"], seed).cpu().numpy()
        return torch.from_numpy(exact_store(kv, case["rows"], case["chunk"], case["d"])).cuda()
    return exact_scores(s["x"], s["given"], case["top"])
