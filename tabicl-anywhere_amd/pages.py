"""Fitted problems in pages of one pool on the card, so that many are served together and (where rows see only those before them)
grow a row at a time.

`PagePool` is the host side of `Gpu.pages_write`, `pages_read` and `pages_attend` (`tah_pages` in tah.h): which pages are whose. A
problem is held by `(prefix, node)` as `hip.CardAttend` holds models, from exact keys and values or from a bundle's stored
records; `attend` has the form of `predict::AttendCached::attend` (`src/predict.rs:63-79`) and returns `None` for a problem the
pool does not hold; `attend_many` answers rows of many problems in one call a layer. A problem's layers lie in the same pages of
the layers' pools, and what a problem gives up the next one takes: the pool never grows. Calls take arrays in host memory, and
borrow room for them on the card from the handle's working memory, whose budget they can exceed (`hip.BudgetError`).
"""
from __future__ import annotations

import threading

import numpy as np

from . import abi, devmem, hip


class PagePool:
    def __init__(self, gpu: "hip.Gpu", layers: int, heads: int, hd: int, pages: int, kv_format: int = abi.KV_I8, page_rows: int = 64):
        if layers <= 0 or pages <= 0 or abi.lib().tah_page_bytes(kv_format, heads, hd, page_rows) == 0:
            raise ValueError("PagePool: bad size or format")
        self.gpu, self.layers, self.heads, self.hd, self.pages = gpu, int(layers), int(heads), int(hd), int(pages)
        self.kv_format, self.page_rows = int(kv_format), int(page_rows)
        self.layer_bytes = pages * abi.page_bytes(kv_format, heads, hd, page_rows)
        # on the handle's card, whichever the calling thread's current one is
        try:
            with devmem.on_card(getattr(gpu, "ordinal", None)):
                self._memory = devmem.DeviceBuffer(self.layers * self.layer_bytes)
        except devmem.HipError as e:
            raise (hip.BudgetError if e.status == devmem.OUT_OF_MEMORY else hip.CardError)(str(e)) from e
        self._free = list(range(self.pages - 1, -1, -1))
        self._held: dict = {}  # (prefix, node): [rows, pages]
        self._lock = threading.RLock()

    @property
    def d(self) -> int:
        return self.heads * self.hd

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def bytes(self) -> int:
        """Card bytes of the pool."""
        return self.layers * self.layer_bytes

    def rows(self, prefix: str, node: int) -> int:
        """Rows held of a problem (0: none)."""
        with self._lock:
            return self._held.get((prefix, node), (0, ()))[0]

    def free(self) -> None:
        with self._lock:
            self._memory.free()
            self._held.clear()
            self._free = []

    # ---- what is held ---------------------------------------------------------------------------------------------
    def hold(self, prefix: str, node: int, layers) -> None:
        """Hold a problem: `layers` its layers' keys and values, (k, v) of [rows][heads * hd] each. In place of what was held by
        that name; if there are too few pages (`hip.BudgetError`) nothing changes. The rows are written into free pages, and
        what was held is given up when they are there; only where that leaves too few pages are its own taken, and it is gone
        if the writing then fails."""
        with self._lock:
            layers, rows = self._checked(layers)
            old = self._held.get((prefix, node), [0, []])
            need = -(-rows // self.page_rows)
            if need > len(self._free) + len(old[1]):
                raise hip.BudgetError(f"graphics card: {need} pages wanted, {len(self._free) + len(old[1])} free")
            if need > len(self._free):
                self.drop(prefix, node)
            new = [0, []]
            self._append(new, layers, rows)
            self.drop(prefix, node)
            self._held[(prefix, node)] = new

    def hold_records(self, prefix: str, node: int, kv_format: int, rows: int, chunk: int, records) -> None:
        """`hold` from a bundle's stored records (`n{j}_kv{l}`), what they stand for."""
        layers = []
        for rec in records:
            kv = self.gpu.unpack(rec, self.d, rows, chunk, kv_format)
            parts = [kv[2 * self.d * a:2 * self.d * min(a + chunk, rows)].reshape(2, self.d, -1) for a in range(0, rows, chunk)]
            both = np.concatenate(parts, axis=2) if parts else np.zeros((2, self.d, 0), np.float32)
            layers.append((both[0].T, both[1].T))
        self.hold(prefix, node, layers)

    def grow(self, prefix: str, node: int, layers) -> None:
        """More rows of a problem that is held (`LookupError` if it is not), as `hold` takes them, behind those it has. What a fit of
        all the rows would give only where rows see those before them and no others: a network whose rows all see each other has
        other keys and values for the rows that were there, and the problem is held anew."""
        with self._lock:
            if (prefix, node) not in self._held:
                raise LookupError(f"no problem {prefix!r}, {node} in the pool")
            held = self._held[(prefix, node)]
            self._append(held, *self._checked(layers, held[0]))

    def drop(self, prefix: str, node: int) -> bool:
        """Give a problem's pages back; whether it was held."""
        with self._lock:
            rows_pages = self._held.pop((prefix, node), None)
            if rows_pages is not None:
                self._free.extend(reversed(rows_pages[1]))
            return rows_pages is not None

    def _checked(self, layers, have: int = 0):
        layers = [tuple(hip._rows_of(a, self.d, "PagePool") for a in kv) for kv in layers]
        if len(layers) != self.layers or any(len(kv) != 2 or kv[0].shape != layers[0][0].shape or kv[1].shape != layers[0][0].shape
                                             for kv in layers):
            raise ValueError(f"PagePool: expected keys and values of {self.layers} layers, all of as many rows")
        rows = layers[0][0].shape[0]
        if have + rows > 2**31 - 1024:
            raise ValueError("PagePool: at most 2^31 - 1024 rows")
        return layers, rows

    def _append(self, held: list, layers, rows: int) -> None:
        """Rows behind those of `held` ([rows, pages]), which stays as it was if that fails."""
        have, pages = held
        need = -(-(have + rows) // self.page_rows) - len(pages)
        if need > len(self._free):
            raise hip.BudgetError(f"graphics card: {need} pages wanted, {len(self._free)} free")
        if rows == 0:
            return
        taken = [self._free.pop() for _ in range(need)]
        try:
            table = np.array([pages + taken], np.int32)
            for l, (k, v) in enumerate(layers):
                self.gpu.pages_write(self._pages(l, table), table, [have], [0, rows], k, v)
        except BaseException:
            self._free.extend(reversed(taken))  # the rows it has are as they were
            raise
        pages.extend(taken)
        held[0] = have + rows

    def _pages(self, layer: int, table: np.ndarray) -> abi.Pages:
        return abi.Pages(pool=self._memory.ptr + layer * self.layer_bytes, kv_format=self.kv_format, kv_heads=self.heads, hd=self.hd,
                         page_rows=self.page_rows, pages=self.pages, tables=table.shape[0], ld=table.shape[1])

    # ---- answers --------------------------------------------------------------------------------------------------
    def attend(self, prefix: str, node: int, layer: int, q, d: int, heads: int):
        """Attention outputs [nq][d] of scaled queries over one layer of a problem; `None` if the pool does not hold it."""
        with self._lock:
            if (prefix, node) not in self._held or d != heads * self.hd or heads % self.heads or not 0 <= layer < self.layers:
                return None
            return self.attend_many(layer, [(prefix, node, q)], heads)[0]

    def attend_many(self, layer: int, asked, heads: int, causal: bool = False) -> list:
        """`attend` of many problems in one call: `asked` a list of (prefix, node, q [nq][heads * hd]); the outputs in order.
        With causal a problem's queries are its last rows, and each sees the rows before it and its own."""
        with self._lock:
            if not 0 <= layer < self.layers:
                raise ValueError(f"PagePool: no layer {layer}")
            held = []
            for prefix, node, _ in asked:
                if (prefix, node) not in self._held:
                    raise LookupError(f"no problem {prefix!r}, {node} in the pool")
                held.append(self._held[(prefix, node)])
            if not held:
                return []
            q = [hip._rows_of(a, heads * self.hd, "PagePool") for _, _, a in asked]
            offsets = np.concatenate([[0], np.cumsum([a.shape[0] for a in q])])
            table = np.full((len(held), max(1, max(len(pages) for _, pages in held))), -1, np.int32)
            for t, (_, pages) in enumerate(held):
                table[t, :len(pages)] = pages
            out = self.gpu.pages_attend(self._pages(layer, table), table, [rows for rows, _ in held], np.concatenate(q), offsets, heads,
                                        causal)
            return [out[a:b] for a, b in zip(offsets[:-1], offsets[1:])]

    def read(self, prefix: str, node: int, layer: int) -> tuple:
        """What a problem's rows of a layer stand for, (k, v) of [rows][heads * hd]."""
        with self._lock:
            if (prefix, node) not in self._held:
                raise LookupError(f"no problem {prefix!r}, {node} in the pool")
            if not 0 <= layer < self.layers:
                raise ValueError(f"PagePool: no layer {layer}")
            rows, pages = self._held[(prefix, node)]
            table = np.array([pages or [-1]], np.int32)
            return self.gpu.pages_read(self._pages(layer, table), table, [0], [0, rows])
