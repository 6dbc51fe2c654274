"""Pages (`tah_pages`) stated in numpy: a pool's bytes, what a row is stored as, and attention in 64 bits with the error that the
kernels' roundings can come to."""
import numpy as np

from conftest import pkg

abi = pkg("abi")
TOP = {abi.KV_I16: 32767, abi.KV_I8: 127}
TYPE = {abi.KV_F32: np.float32, abi.KV_I16: np.int16, abi.KV_I8: np.int8}


class Pool:
    """A pool on the host: `bytes` and views of it, keys [pages][heads][rows][hd], values [pages][heads][hd][rows], steps
    [pages][heads][2][rows]."""

    def __init__(self, fmt, heads, hd, rows, pages, fill=0):
        self.fmt, self.heads, self.hd, self.rows, self.pages = fmt, heads, hd, rows, pages
        self.bytes = np.full(pages * abi.page_bytes(fmt, heads, hd, rows), fill, np.uint8)

    def _part(self, head, at, count, dtype):
        """`count` numbers of every page's head from byte `at` of it, as a view."""
        b = self.bytes.reshape(self.pages, self.heads, -1)
        w = np.dtype(dtype).itemsize
        return np.lib.stride_tricks.as_strided(b[:, :, at:].view(np.uint8)[:, :, :w].view(dtype)[..., 0], (self.pages, self.heads, count),
                                               (b.strides[0], b.strides[1], w))

    @property
    def keys(self):
        return self._part(None, 0, self.rows * self.hd, TYPE[self.fmt]).reshape(self.pages, self.heads, self.rows, self.hd, copy=False)

    @property
    def values(self):
        w = np.dtype(TYPE[self.fmt]).itemsize
        return self._part(None, self.rows * self.hd * w, self.rows * self.hd, TYPE[self.fmt]).reshape(
            self.pages, self.heads, self.hd, self.rows, copy=False)

    @property
    def steps(self):
        w = np.dtype(TYPE[self.fmt]).itemsize
        return self._part(None, 2 * self.rows * self.hd * w, 2 * self.rows, np.float32).reshape(self.pages, self.heads, 2, self.rows,
                                                                                               copy=False)

    def write(self, page, slot, k, v):
        """Row k, v [heads][hd] at slot `slot` of page `page`."""
        if self.fmt == abi.KV_F32:
            self.keys[page, :, slot], self.values[page, :, :, slot] = k, v
            return
        for which, x in ((0, k), (1, v)):
            c, s = quantised(x, TOP[self.fmt])
            self.steps[page, :, which, slot] = s
            if which:
                self.values[page, :, :, slot] = c
            else:
                self.keys[page, :, slot] = c

    def read(self, page, slot):
        """What the row stands for, in 64 bits."""
        k, v = self.keys[page, :, slot].astype(np.float64), self.values[page, :, :, slot].astype(np.float64)
        if self.fmt == abi.KV_F32:
            return k, v
        s = self.steps[page, :, :, slot].astype(np.float64)
        return k * s[:, 0, None], v * s[:, 1, None]

    def rows_of(self, table, n):
        """Keys and values [n][heads][hd] of a table's first n rows."""
        at = np.arange(n)
        page, slot = np.asarray(table)[at // self.rows], at % self.rows
        k, v = self.keys[page, :, slot].astype(np.float64), self.values[page, :, :, slot].astype(np.float64)
        if self.fmt != abi.KV_F32:
            s = self.steps[page, :, :, slot].astype(np.float64)
            k, v = k * s[:, :, 0, None], v * s[:, :, 1, None]
        return k, v


def quantised(x, top):
    """Rows x [..][hd] (float32) as ints and steps, as the header states them."""
    x = np.asarray(x, np.float32)
    finite = np.where(np.isfinite(x), np.abs(x), np.float32(0))
    s = (finite.max(-1) / np.float32(top)).astype(np.float32)
    s = np.where(s < np.float32(2.0**-126), np.float32(0), s)
    wide = np.where(s > 0, s, np.float32(1)).astype(np.float64)[..., None]
    c = np.clip(np.rint(np.where(np.isfinite(x), x, 0).astype(np.float64) / wide), -top, top)
    c = np.where(np.isposinf(x), top, np.where(np.isneginf(x), -top, c))
    return np.where(s[..., None] > 0, c, 0).astype(np.int64), s


def attention(q, k, v, limits):
    """q [n][heads][hd] over k, v [m][kv_heads][hd] in 64 bits, query i over its first limits[i] rows; and how far a kernel may
    be off, per output.

    The error, with u = 2^-24: a score is a sum of products of operands held in two halves of 11 bits (2^-22 of a term at worst
    for the three dropped or rounded parts of either, 2^-38 of the largest terms where a half is below fp16's normal numbers)
    added in f32 (hd + 4 additions), times a step and log2 e, in an exponent (three roundings of the score's, one of an
    argument of up to the score's distance from the maximum and 15): `ds`. A weight is off by as much of itself, 2^-22 for exp2
    and 2^-22 for its halves and its value's step; values' halves 2^-22 more; both sums are of f32 over the rows, a block of 64 at
    a time, scaled again for each new maximum, joined over at most 64 states. Weights below fp16's normal numbers, 2^-26 of the
    largest, are off by 2^-37 of it each."""
    n, heads, hd = q.shape
    group = heads // k.shape[1]
    out, off = np.zeros(q.shape), np.zeros(q.shape)
    q, k, v, u = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64), 2.0**-24
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        for i in range(n):
            m = int(limits[i])
            if m <= 0:
                continue
            t = kh[:m] @ q[i, h]
            w = np.exp(t - t.max())
            out[i, h] = (w @ vh[:m]) / w.sum()
            ds = ((3 * 2.0**-22 + (hd + 4) * u) * (np.abs(kh[:m]) @ np.abs(q[i, h])) + 4 * u * np.abs(t) +
                  2.0**-38 * hd * np.abs(q[i, h]).max() * np.abs(kh[:m]).max())
            dw = ds + ds.max() + u * (np.abs(t - t.max()) + 20.0) + 4 * 2.0**-22 + (m / 64 + 80) * 2 * u
            off[i, h] = (w * dw) @ (np.abs(vh[:m]) + np.abs(out[i, h])) / w.sum() + m * 2.0**-37 * np.abs(vh[:m]).max()
    return out, off


def limits_of(length, n, causal):
    return [max(0, length - (n - 1 - i)) if causal else length for i in range(n)]
