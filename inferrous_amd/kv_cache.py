"""A paged 8-bit cache of keys and values: its memory, and which page belongs to whom.

``KvCache`` is the device memory of every layer's pages, in the layout of
include/inferrous_w8a8.h.  ``PagePool`` is the host's bookkeeping: it hands out,
shares, copies on write, frees and compacts page numbers, which are the same in
every layer.  It touches no device memory: what has to be copied it returns as
(source, destination) pairs for ``LoadedModule.copy_pages``.  The reference keeps
one request's cache as two plain buffers per layer (crates/inferrous-qwen3/src/gpu.rs:90-121).
"""
from __future__ import annotations

import numpy as np

from ._lib import PAGE_TOKENS
from .runtime import DeviceBuffer

_U8, _F32 = np.dtype(np.uint8), np.dtype(np.float32)


class KvCache:
    """``layers`` caches of ``pages`` pages of 64 tokens, ``kv_heads`` heads of
    ``head_dim`` (64 or 128): ``codes`` (uint8 [layers, pages, kv_heads, 2, 64 *
    head_dim], e4m3) and ``scales`` (float32 [layers, pages, kv_heads, 2])."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int):
        self._take(layers, pages, kv_heads, head_dim)
        self._hold(DeviceBuffer(self.values, _U8), DeviceBuffer(self.blocks, _F32))

    @classmethod
    def over(cls, codes, scales, layers: int, pages: int, kv_heads: int, head_dim: int) -> "KvCache":
        """The same over buffers that the caller holds."""
        c = cls.__new__(cls)
        c._take(layers, pages, kv_heads, head_dim)
        if codes.dtype != _U8 or scales.dtype != _F32:
            raise TypeError("codes must be uint8 and scales float32")
        if len(codes) < c.values or len(scales) < c.blocks:
            raise ValueError(f"codes and scales hold {len(codes)} and {len(scales)} values, "
                             f"need {c.values} and {c.blocks}")
        c._hold(codes, scales)
        return c

    def _take(self, layers, pages, kv_heads, head_dim):
        if min(layers, pages, kv_heads) < 1 or head_dim not in (64, 128):
            raise ValueError("a cache has layers, pages and heads, of 64 or 128 values")
        self.layers, self.pages, self.kv_heads, self.head_dim = layers, pages, kv_heads, head_dim
        self.blocks = layers * pages * kv_heads * 2
        self.values = self.blocks * PAGE_TOKENS * head_dim

    def _hold(self, codes, scales):
        self.codes, self.scales = codes, scales
        step, part = self.values // self.layers, 4 * (self.blocks // self.layers)
        self.at = [(codes.ptr + i * step, scales.ptr + i * part) for i in range(self.layers)]

    def layer(self, i: int) -> tuple[int, int]:
        """Addresses of a layer's codes and scales."""
        if not 0 <= i < self.layers:
            raise ValueError(f"layer {i} of {self.layers}")
        return self.at[i]


class PagePool:
    """Page numbers 0 .. pages - 1 of a cache, and the sequences that hold them.

    Full pages may be shared by forked sequences; a page that a sequence still
    writes to (its last, while it is not full) is its own: ``extend`` copies a shared
    one first.  Nothing changes where a call raises.

    The pairs that ``extend`` and ``compact`` return are copied before any sequence's
    rows are written.  Those of several calls of ``extend`` may be one copy; before a
    ``fork``, ``free``, ``shorten`` or ``compact`` they are made, since these can let a
    page that is copied to be copied from, or to again."""

    def __init__(self, pages: int):
        if pages < 1:
            raise ValueError("a pool has pages")
        self.pages = pages
        self._free = list(range(pages - 1, -1, -1))   # the lowest number is handed out first
        self._users = [0] * pages
        self._of: dict[int, list[int]] = {}
        self._tokens: dict[int, int] = {}
        self._next = 0

    def __len__(self) -> int:
        """Sequences."""
        return len(self._of)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A new sequence without tokens."""
        seq, self._next = self._next, self._next + 1
        self._of[seq], self._tokens[seq] = [], 0
        return seq

    def length(self, seq: int) -> int:
        return self._tokens[seq]

    def extend(self, seq: int, tokens: int) -> list[tuple[int, int]]:
        """Room for ``tokens`` more tokens.  Returns the copies to make before
        they are written: the last page, if it is shared and not full."""
        if tokens < 0:
            raise ValueError("tokens must not be negative")
        held, have = self._of[seq], self._tokens[seq]
        if tokens == 0:
            return []
        copy = have % PAGE_TOKENS != 0 and self._users[held[-1]] > 1
        more = -(-(have + tokens) // PAGE_TOKENS) - len(held)
        if more + copy > len(self._free):
            raise MemoryError(f"{more + copy} pages needed, {len(self._free)} free")
        pairs = []
        if copy:
            old, new = held[-1], self._take()
            self._users[old] -= 1
            held[-1] = new
            pairs.append((old, new))
        held.extend(self._take() for _ in range(more))
        self._tokens[seq] = have + tokens
        return pairs

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens, on the same pages."""
        new, held = None, self._of[seq]
        new = self.add()
        self._of[new], self._tokens[new] = list(held), self._tokens[seq]
        for page in held:
            self._users[page] += 1
        return new

    def shorten(self, seq: int, tokens: int) -> None:
        """The sequence keeps its first ``tokens`` tokens (drafts that were not taken
        are gone); pages behind them that nobody else holds are free again."""
        held, have = self._of[seq], self._tokens[seq]
        if not 0 <= tokens <= have:
            raise ValueError(f"a sequence of {have} tokens cannot keep {tokens}")
        keep = -(-tokens // PAGE_TOKENS)
        for page in reversed(held[keep:]):
            self._drop(page)
        del held[keep:]
        self._tokens[seq] = tokens

    def free(self, seq: int) -> None:
        """The sequence ends; pages that nobody else holds are free again."""
        for page in self._of.pop(seq):
            self._drop(page)
        del self._tokens[seq]

    def compact(self) -> list[tuple[int, int]]:
        """Brings the pages in use to the lowest numbers.  Returns the copies to
        make: no page is a source and a destination."""
        used = sum(n > 0 for n in self._users)
        holes = iter([p for p in range(used) if not self._users[p]])
        to = {p: next(holes) for p in range(used, self.pages) if self._users[p]}
        for held in self._of.values():
            held[:] = [to.get(p, p) for p in held]
        for old, new in to.items():
            self._users[new], self._users[old] = self._users[old], 0
        self._free = list(range(self.pages - 1, used - 1, -1))
        return list(to.items())

    def table(self, seqs, width: int | None = None) -> np.ndarray:
        """int32 [len(seqs), width] for the operators; -1 behind a sequence's pages."""
        held = [self._of[s] for s in seqs]
        need = max([1, *map(len, held)])
        if width is None:
            width = need
        if width < need:
            raise ValueError(f"a sequence has {need} pages, the table {width}")
        out = np.full((len(held), width), -1, np.int32)
        for row, pages in zip(out, held):
            row[:len(pages)] = pages
        return out

    def _take(self) -> int:
        page = self._free.pop()
        self._users[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if not self._users[page]:
            self._free.append(page)
