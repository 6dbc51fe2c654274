"""Measurement cases of the operators over many tables at once, with their plain forms.

Kinds of case (`op`):

* `store`: new rows' exact keys and values, of many tables, into pages of a pool and back to the values that the pages then
  stand for (`Gpu.pages_write_dev`, `Gpu.pages_read_dev`);
* `attend`: scaled queries of many tables, one or a few new rows each, over the tables' pages (`Gpu.pages_attend_dev`);
* `packed`: scaled queries of whole tables that lie one after the other, each over its own table's rows in full precision
  (`Gpu.attend_packed_dev`).

A page holds `page` rows of one layer. Per key/value head: the rows' keys [page][hd], then their values [hd][page], as f32,
int16 or int8; after int16 and int8 the rows' key steps [page], then their value steps [page], in f32. An int stands for
itself times its row's step. A row's step is its largest magnitude over 32767 or 127, an int the row's number over it, rounded
to the nearest, ties to even. A table's pages are listed in order, -1 where there is none.

Keys and values are what a layer norm and a projection leave: a mean of its own per coordinate, spread 0.55. Queries are
already scaled. Everything is made from the seed on the card; the lengths are the case's own.
"""
import functools
import importlib
import math

import numpy as np
import torch

own = False

WIDTH = {"f32": 4, "i16": 2, "i8": 1}
TOP = {"i16": 32767.0, "i8": 127.0}
SMALLEST = 2.0 ** -126  # steps below it are held as 0


def listed():
    return [
        # a row more in each of 64 tables that are served together: latency
        {"name": "store_64x1", "op": "store", "tables": 64, "least": 1, "most": 1, "kv_heads": 8, "hd": 64, "fmt": "i8", "page": 64},
        # the benchmark's table put into pages, one layer
        {"name": "store_10000", "op": "store", "tables": 1, "least": 10000, "most": 10000, "kv_heads": 8, "hd": 64, "fmt": "i8",
         "page": 64},
        # tables of all lengths in small pages, wide grouped heads, two bytes a number
        {"name": "store_40x1500", "op": "store", "tables": 40, "least": 1, "most": 1500, "kv_heads": 4, "hd": 128, "fmt": "i16",
         "page": 16},
        # one row answered from a small table: latency
        {"name": "attend_1x1000", "op": "attend", "tables": 1, "least": 1000, "most": 1000, "new": 1, "causal": False, "heads": 8,
         "kv_heads": 8, "hd": 64, "fmt": "i8", "page": 64},
        # one row against a long table: its bytes
        {"name": "attend_1x100000", "op": "attend", "tables": 1, "least": 100000, "most": 100000, "new": 1, "causal": False,
         "heads": 8, "kv_heads": 8, "hd": 64, "fmt": "i8", "page": 64},
        # a row for each of many tables of very different lengths, some of them empty
        {"name": "attend_64x20000", "op": "attend", "tables": 64, "least": 0, "most": 20000, "new": 1, "causal": False, "heads": 8,
         "kv_heads": 8, "hd": 64, "fmt": "i8", "page": 64},
        # a few new rows a table that see those before them, grouped heads, small pages, two bytes a number
        {"name": "attend_24x6001", "op": "attend", "tables": 24, "least": 5, "most": 6001, "new": 9, "causal": True, "heads": 16,
         "kv_heads": 4, "hd": 128, "fmt": "i16", "page": 16},
        # exact pages, a narrower network
        {"name": "attend_7x9000", "op": "attend", "tables": 7, "least": 800, "most": 9000, "new": 3, "causal": False, "heads": 4,
         "kv_heads": 4, "hd": 64, "fmt": "f32", "page": 128},
        # the small problems of a class tree, fitted together
        {"name": "packed_32x300", "op": "packed", "tables": 32, "least": 11, "most": 300, "causal": False, "heads": 8, "kv_heads": 8,
         "hd": 64},
        # the benchmark's table, every row over all rows
        {"name": "packed_1x10000", "op": "packed", "tables": 1, "least": 10000, "most": 10000, "causal": False, "heads": 8,
         "kv_heads": 8, "hd": 64},
        # tables in order, each row over those before it, grouped heads
        {"name": "packed_5x6007", "op": "packed", "tables": 5, "least": 500, "most": 6007, "causal": True, "heads": 16, "kv_heads": 4,
         "hd": 64},
        # wide heads
        {"name": "packed_3x2500", "op": "packed", "tables": 3, "least": 900, "most": 2500, "causal": True, "heads": 8, "kv_heads": 2,
         "hd": 128},
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["store", "attend", "attend", "attend", "packed", "packed"])
    kv_heads, group = rng.choice([(8, 1), (8, 1), (4, 4), (2, 4), (4, 1), (1, 8)])
    hd = rng.choice([64, 64, 64, 128, 32])
    tables = between(1, 200)
    case = {"op": op, "tables": tables, "least": 0, "most": 0}
    if op == "packed":
        # at most the products of the largest listed case
        most = max(3, int(math.sqrt(between(4000, 100_000_000) * 64 * 8 / (hd * kv_heads * group * tables))))
        return dict(case, least=rng.choice([1, most // 2, most]), most=most, causal=rng.choice([True, False]),
                    heads=kv_heads * group, kv_heads=kv_heads, hd=hd)
    fmt = rng.choice(["i8", "i8", "i16", "f32"])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    if op == "store":
        most = between(1, max(1, 5_120_000 // (tables * kv_heads * hd)))
        return dict(case, least=rng.choice([1, most]), most=most, kv_heads=kv_heads, hd=hd, fmt=fmt, page=page)
    most = between(30, max(31, min(120_000, 330_000_000 // (tables * kv_heads * hd * WIDTH[fmt]))))
    return dict(case, least=rng.choice([0, 1, most // 2]), most=most, new=rng.choice([1, 1, 1, 2, 5, 16]),
                causal=rng.choice([True, False]), heads=kv_heads * group, kv_heads=kv_heads, hd=hd, fmt=fmt, page=page)


# ---- what a program has in hand ---------------------------------------------------------------------------------------
def lengths(case):
    """The tables' row counts: the most for the first, the others spread over the range, the least for the second."""
    n, lo, hi = case["tables"], case["least"], case["most"]
    return [hi if i == 0 else lo if i == 1 else lo + int((hi - lo) * (i * 0.6180339887 % 1.0)) for i in range(n)]


def new_rows(case):
    """The tables' new rows (`attend`): up to `new`, not the same for all."""
    return [max(1, case["new"] - i % 3) for i in range(case["tables"])]


def starts(case):
    """Where the tables' new rows begin (`store`): anywhere in a page."""
    return [(37 * i) % 101 if case["tables"] > 1 else 0 for i in range(case["tables"])]


def head_bytes(case):
    w = WIDTH[case["fmt"]]
    return case["page"] * (2 * case["hd"] * w + (8 if w < 4 else 0))


def generator(*key):
    return torch.Generator(device="cuda").manual_seed(hash(key) & 0x7FFFFFFF)


def layer_values(rows, kv_heads, hd, seed, which):
    """Exact keys (which 1) or values (2) of rows, [rows][kv_heads][hd]."""
    g = generator(seed, which)
    mean = torch.randn(kv_heads, hd, device="cuda", generator=g) * 0.3
    return torch.randn(rows, kv_heads, hd, device="cuda", generator=g) * 0.55 + mean


def whole(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets(counts):
    return whole(np.concatenate([[0], np.cumsum(counts)]).tolist())


def page_table(case, most_rows, seed):
    """(table [tables][ld], pages of the pool): tables of up to most_rows[i] rows, their pages anywhere in the pool."""
    need = [-(-r // case["page"]) for r in most_rows]
    ld, total = max(1, max(need)), sum(need) + 3
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).numpy()
    table = np.full((case["tables"], ld), -1, np.int32)
    table[np.arange(ld)[None, :] < np.array(need)[:, None]] = order[:sum(need)]
    return torch.from_numpy(table).cuda(), total


@functools.lru_cache(maxsize=None)
def card():
    return importlib.import_module("tabicl-anywhere_amd.hip").Gpu(0)


def prepare(case, seed):
    op, hkv, hd = case["op"], case["kv_heads"], case["hd"]
    s = {"case": case, "counts": lengths(case)}
    if op == "packed":
        rows = sum(s["counts"])
        s["k"], s["v"] = layer_values(rows, hkv, hd, seed, 1), layer_values(rows, hkv, hd, seed, 2)
        s["q"] = torch.randn(rows, case["heads"], hd, device="cuda", generator=generator(seed, 3)) * 0.4
        s["offsets"] = offsets(s["counts"])
        s["out"] = torch.empty_like(s["q"])
    elif op == "store":
        s["starts"], s["offsets"] = whole(starts(case)), offsets(s["counts"])
        s["table"], s["pages"] = page_table(case, [a + n for a, n in zip(starts(case), s["counts"])], seed)
        s["pool"] = torch.zeros(s["pages"] * hkv * head_bytes(case), dtype=torch.uint8, device="cuda")
        rows = sum(s["counts"])
        s["k"], s["v"] = layer_values(rows, hkv, hd, seed, 1), layer_values(rows, hkv, hd, seed, 2)
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    else:
        s["table"], s["pages"] = page_table(case, s["counts"], seed)
        s["pool"] = torch.zeros(s["pages"] * hkv * head_bytes(case), dtype=torch.uint8, device="cuda")
        # every row of every page, those behind a table's end too
        at = torch.arange(s["pages"] * case["page"], device="cuda")
        rows = at.numel()
        plain_write(s["pool"], case, at // case["page"], at % case["page"], layer_values(rows, hkv, hd, seed, 1),
                    layer_values(rows, hkv, hd, seed, 2))
        s["new"] = new_rows(case)
        s["q"] = torch.randn(sum(s["new"]), case["heads"], hd, device="cuda", generator=generator(seed, 3)) * 0.4
        s["offsets"], s["lengths"] = offsets(s["new"]), whole(s["counts"])
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["gpu"] = card()
        if op != "packed":
            s["described"] = described(s)
    torch.cuda.synchronize()
    return s


def described(state):
    """The pages as the framework takes them."""
    case, abi = state["case"], importlib.import_module("tabicl-anywhere_amd.abi")
    return abi.Pages(pool=state["pool"].data_ptr(), table=state["table"].data_ptr(), kv_format=abi.KV_NAMES[case["fmt"]],
                     kv_heads=case["kv_heads"], hd=case["hd"], page_rows=case["page"], pages=state["pages"],
                     tables=case["tables"], ld=state["table"].shape[1])


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        gpu = state["gpu"]
        if op == "packed":
            at = state["offsets"].data_ptr()
            rows = state["q"].shape[0]
            gpu.attend_packed_dev(state["q"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(), at, at, case["tables"], rows,
                                  rows, case["heads"], case["kv_heads"], case["hd"], state["out"].data_ptr(),
                                  causal=case["causal"])
            return state["out"]
        pages = state["described"]
        if op == "store":
            rows = state["k"].shape[0]
            gpu.pages_write_dev(pages, state["starts"].data_ptr(), state["offsets"].data_ptr(), state["k"].data_ptr(),
                                state["v"].data_ptr(), rows)
            gpu.pages_read_dev(pages, state["starts"].data_ptr(), state["offsets"].data_ptr(), state["k_out"].data_ptr(),
                               state["v_out"].data_ptr(), rows)
            return state["k_out"], state["v_out"]
        gpu.pages_attend_dev(pages, state["lengths"].data_ptr(), state["q"].data_ptr(), state["offsets"].data_ptr(),
                             state["q"].shape[0], case["heads"], state["out"].data_ptr(), causal=case["causal"])
        return state["out"]
    if op == "packed":
        return plain_packed(state["q"], state["k"], state["v"], state["offsets"], max(state["counts"]), case["causal"])
    if op == "store":
        page, slot = plain_places(case, state["table"], state["starts"], state["offsets"], state["k"].shape[0])
        plain_write(state["pool"], case, page, slot, state["k"], state["v"])
        return plain_read(state["pool"], case, page, slot)
    return plain_attend(state["pool"], case, state["table"], state["lengths"], state["q"], state["offsets"], max(state["new"]))


# ---- plain forms ------------------------------------------------------------------------------------------------------
def sections(pool, case):
    """Views of a pool: keys [pages][heads][page][hd], values [pages][heads][hd][page], steps [pages][heads][2][page]."""
    p, hd, w = case["page"], case["hd"], WIDTH[case["fmt"]]
    heads = pool.view(-1, case["kv_heads"], head_bytes(case))
    number = {4: torch.float32, 2: torch.int16, 1: torch.int8}[w]
    keys = heads[:, :, :p * hd * w].view(number).unflatten(2, (p, hd))
    values = heads[:, :, p * hd * w:2 * p * hd * w].view(number).unflatten(2, (hd, p))
    steps = heads[:, :, 2 * p * hd * w:].view(torch.float32).unflatten(2, (2, p)) if w < 4 else None
    return keys, values, steps


def plain_places(case, table, start, offset, rows):
    """The page and the row within it of each row of a call."""
    r = torch.arange(rows, device="cuda")
    t = torch.searchsorted(offset.long(), r, right=True) - 1
    at = start.long()[t] + r - offset.long()[t]
    return table.long()[t, at // case["page"]], at % case["page"]


def quantised(x, top, number):
    """Rows of numbers as ints, and their steps."""
    s = (x.abs().amax(2).double() / top).float()  # the float32 quotient, rounded once
    s = torch.where(s < SMALLEST, torch.zeros_like(s), s)
    # the quotient in 64 bits, so that none is rounded onto a tie
    c = torch.round(x.double() / torch.where(s > 0, s, torch.ones_like(s)).double()[:, :, None]).clamp(-top, top)
    return torch.where(s[:, :, None] > 0, c, torch.zeros_like(c)).to(number), s


def plain_write(pool, case, page, slot, k, v):
    keys, values, steps = sections(pool, case)
    if steps is not None:
        k, sk = quantised(k, TOP[case["fmt"]], keys.dtype)
        v, sv = quantised(v, TOP[case["fmt"]], keys.dtype)
        steps[page, :, 0, slot] = sk
        steps[page, :, 1, slot] = sv
    keys[page, :, slot] = k
    values[page, :, :, slot] = v


def plain_read(pool, case, page, slot):
    keys, values, steps = sections(pool, case)
    k, v = keys[page, :, slot].float(), values[page, :, :, slot].float()
    if steps is None:
        return k, v
    return k * steps[page, :, 0, slot][:, :, None], v * steps[page, :, 1, slot][:, :, None]


def padded(x, offset, most):
    """Rows of tables one after the other as [tables][most][..] (a table's end filled with whatever), and their counts."""
    at = torch.arange(most, device="cuda")[None, :] + offset.long()[:-1, None]
    return x[at.clamp(max=max(0, x.shape[0] - 1))], (offset[1:] - offset[:-1]).long()


def softmax_attention(q, k, v, seen):
    """q [..][queries][hd] over k, v [..][keys][hd], where seen says which keys; nothing seen gives 0."""
    t = torch.matmul(q, k.transpose(-1, -2).contiguous())
    t = torch.where(seen, t, torch.full_like(t, -math.inf))
    m = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def unpadded(o, counts):
    """[tables][most][heads][hd] to the tables' rows one after the other."""
    return o[torch.arange(o.shape[1], device="cuda")[None, :] < counts[:, None]]


def plain_attend(pool, case, table, length, q, offset, most):
    keys, values, steps = sections(pool, case)
    hkv, hd, ids = case["kv_heads"], case["hd"], table.long().clamp(min=0)
    k = keys[ids].float()    # [tables][ld][heads][page][hd]
    v = values[ids].float()  # [tables][ld][heads][hd][page]
    if steps is not None:
        k = k * steps[ids][:, :, :, 0, :, None]
        v = v * steps[ids][:, :, :, 1, None, :]
    k = k.permute(0, 2, 1, 3, 4).reshape(case["tables"], hkv, -1, hd)
    v = v.permute(0, 2, 1, 4, 3).reshape(case["tables"], hkv, -1, hd)
    qp, new = padded(q, offset, most)  # [tables][most][heads][hd]
    i, j = torch.arange(most, device="cuda"), torch.arange(k.shape[2], device="cuda")
    last = length.long()[:, None] - 1 + ((i[None, :] + 1 - new[:, None]) if case["causal"] else 0 * i[None, :])
    seen = j[None, None, :] <= last[:, :, None]  # [tables][most][keys]
    group = case["heads"] // hkv
    qg = qp.reshape(-1, most, hkv, group, hd).permute(0, 2, 1, 3, 4).reshape(-1, hkv, most * group, hd)
    o = softmax_attention(qg, k, v, seen[:, None, :, None, :].expand(-1, hkv, -1, group, -1).reshape(-1, hkv, most * group, j.numel()))
    o = o.view(-1, hkv, most, group, hd).permute(0, 2, 1, 3, 4).reshape(-1, most, case["heads"], hd)
    return unpadded(o, new)


def plain_packed(q, k, v, offset, most, causal):
    group = q.shape[1] // k.shape[1]
    qp, counts = padded(q, offset, most)
    kp, vp = padded(k, offset, most)[0], padded(v, offset, most)[0]
    i = torch.arange(most, device="cuda")
    seen = (i[None, None, :] < counts[:, None, None]) & ((i[:, None] >= i[None, :])[None] if causal else True)
    kp, vp = (x.transpose(1, 2).repeat_interleave(group, 1) for x in (kp, vp))
    return unpadded(softmax_attention(qp.transpose(1, 2), kp, vp, seen[:, None]).transpose(1, 2), counts)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def pairs(case):
    """(query, key) pairs of a head."""
    if case["op"] == "packed":
        return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths(case))
    return sum(sum(max(0, n - new + 1 + i if case["causal"] else n) for i in range(new)) for n, new in zip(lengths(case), new_rows(case)))


def work(case):
    rows, hkv, hd = sum(lengths(case)), case["kv_heads"], case["hd"]
    if case["op"] == "packed":
        return {"bytes": 8.0 * rows * hd * (case["heads"] + hkv), "flops": 4.0 * hd * case["heads"] * pairs(case)}
    held = 2.0 * rows * hkv * (hd * WIDTH[case["fmt"]] + (4 if case["fmt"] != "f32" else 0))
    if case["op"] == "store":
        # the values in, the pages out, the pages in and the values out; magnitude and maximum, a quotient rounded, a product back
        return {"bytes": 2.0 * held + 16.0 * rows * hkv * hd, "flops": 10.0 * rows * hkv * hd}
    return {"bytes": held + 8.0 * sum(new_rows(case)) * case["heads"] * hd, "flops": 4.0 * hd * case["heads"] * pairs(case)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def exact_values(x, fmt):
    """What rows [rows][heads][hd] (float32, host) stand for once stored."""
    if fmt == "f32":
        return x.astype(np.float64)
    # the step is defined by this float32 quotient
    s = np.abs(x).max(2, keepdims=True) / np.float32(TOP[fmt])
    s = np.where(s < np.float32(SMALLEST), np.float32(0.0), s).astype(np.float64)
    c = np.rint(np.divide(x.astype(np.float64), s, out=np.zeros(x.shape), where=s > 0))
    return np.clip(c, -TOP[fmt], TOP[fmt]) * s


def exact_rows(raw, case, ids, rows, head):
    """Keys and values [rows][hd] of one head of a table with these pages, from the pool's bytes, float64 on the card."""
    p, hd, w = case["page"], case["hd"], WIDTH[case["fmt"]]
    j = torch.arange(rows, device="cuda")
    base = (ids.long()[j // p] * case["kv_heads"] + head) * head_bytes(case)
    slot, dim = j % p, torch.arange(hd, device="cuda")

    def numbers(at, kind, width):
        byte = at[..., None] + torch.arange(width, device="cuda")
        return raw[byte].view(kind).squeeze(-1).double()

    kind = {4: torch.float32, 2: torch.int16, 1: torch.int8}[w]
    k = numbers(base[:, None] + (slot[:, None] * hd + dim[None, :]) * w, kind, w)
    v = numbers(base[:, None] + (p * hd + dim[None, :] * p + slot[:, None]) * w, kind, w)
    if w < 4:
        k = k * numbers(base + 2 * p * hd * w + 4 * slot, torch.float32, 4)[:, None]
        v = v * numbers(base + 2 * p * hd * w + 4 * (p + slot), torch.float32, 4)[:, None]
    return k, v


def exact_head(q, k, v, first):
    """Softmax attention in float64 of q [n][hd] over k, v [m][hd]; query i sees the first first + i keys (first None: all)."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    t = q @ k.T
    if first is not None:
        sees = torch.arange(q.shape[0], device="cuda")[:, None] + first
        t = t.masked_fill(torch.arange(k.shape[0], device="cuda")[None, :] >= sees, -math.inf)
        return torch.nan_to_num(torch.softmax(t, 1)) @ v
    return torch.softmax(t, 1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return tuple(torch.from_numpy(exact_values(s[x].cpu().numpy(), case["fmt"])).cuda() for x in ("k", "v"))
    out, group = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), case["heads"] // case["kv_heads"]
    at = s["offsets"].tolist()
    for t, n in enumerate(s["counts"]):
        a, b = at[t], at[t + 1]
        for h in range(case["kv_heads"]):
            if case["op"] == "packed":
                k, v, first = s["k"][a:b, h].double(), s["v"][a:b, h].double(), 1
            else:
                k, v = exact_rows(s["pool"], case, s["table"][t], n, h)
                first = n - (b - a) + 1
            for g in range(h * group, (h + 1) * group):
                out[a:b, g] = exact_head(s["q"][a:b, g].double(), k, v, first if case["causal"] else None)
    return out
