"""States whose keys and values lie in 4 bits in pages: the bookkeeping around ``kernels.kv4``.

``PagePool`` hands out page numbers with reference counts (host only, thread-safe): ``allocate``,
``share``, ``release``, ``fork`` (the full pages of a sequence shared, its last partly filled one
to be copied) and ``compact`` (which pages move where so that the live ones are the lowest).

``Kv4States`` joins a pool, a ``Kv4Cache`` for the full-attention layers and one device tensor of
page tables. ``store(snapshot)`` quantises the K/V of a state pass's snapshot into pages and gives a
``Kv4Snapshot``: the same list with a ``Kv4Entry`` in the place of every ``AttentionEntry``, which
``D3Backbone.questions`` reads and ``StateCache`` keeps (``tensor_bytes`` counts its pages).
``fork``, ``extend`` and ``compact`` copy and move pages on the device.

Lifetime: a state's pages go back to the pool when the last snapshot, copy of its list or entry of it
is dropped. Work queued before then on the current stream may still read them; what is queued later on
that stream comes after it. Readers on other streams must be ordered by the caller, as for any tensor.
``compact`` rewrites the tables in place: a captured graph that reads them stays right.
"""

from __future__ import annotations

import collections
import dataclasses
import heapq
import threading
from dataclasses import dataclass, field
from typing import Any, Callable, Sequence

import torch

from ..kernels.kv4 import Kv4Cache, page_bytes
from .snapshot import AttentionEntry


class PagePool:
    """Page numbers 0 .. ``pages`` with reference counts; the lowest free ones go first."""

    def __init__(self, pages: int):
        if pages < 0:
            raise ValueError("pages must be >= 0")
        self.pages = int(pages)
        self._count = [0] * self.pages
        self._free = list(range(self.pages))  # a heap: ascending is one
        self._lock = threading.RLock()

    @property
    def free(self) -> int:
        return len(self._free)

    @property
    def used(self) -> int:
        return self.pages - len(self._free)

    def references(self, page: int) -> int:
        return self._count[page]

    def _live(self, pages: Sequence[int]) -> None:
        for p in pages:
            if not 0 <= p < self.pages or self._count[p] == 0:
                raise ValueError(f"page {p} is not in use")

    def allocate(self, n: int) -> list[int] | None:
        """``n`` pages with one reference each, or None where fewer are free."""
        if n < 0:
            raise ValueError("n must be >= 0")
        with self._lock:
            if n > len(self._free):
                return None
            got = [heapq.heappop(self._free) for _ in range(n)]
            for p in got:
                self._count[p] = 1
            return got

    def share(self, pages: Sequence[int]) -> None:
        """One more reference to each of ``pages``."""
        with self._lock:
            self._live(pages)
            for p in pages:
                self._count[p] += 1

    def release(self, pages: Sequence[int]) -> None:
        """One reference less to each; pages without one are free again."""
        with self._lock:
            self._live(pages)
            for p, n in collections.Counter(pages).items():
                if self._count[p] < n:
                    raise ValueError(f"page {p} has {self._count[p]} references")
            for p in pages:
                self._count[p] -= 1
                if self._count[p] == 0:
                    heapq.heappush(self._free, p)

    def fork(self, pages: Sequence[int], tokens: int, page_tokens: int) -> tuple[list[int], list[int], list[int]] | None:
        """(pages, src, dst) of a copy of a sequence of ``tokens`` tokens that can grow by itself: full
        pages are shared, a partly filled last page is to be copied from src to dst. None where no page
        is free for it."""
        full, rest = divmod(int(tokens), int(page_tokens))
        if tokens < 0 or full + bool(rest) > len(pages):
            raise ValueError(f"{tokens} tokens in {len(pages)} pages of {page_tokens}")
        with self._lock:
            self._live(pages[:full + bool(rest)])
            own = self.allocate(1 if rest else 0)
            if own is None:
                return None
            self.share(pages[:full])
            return list(pages[:full]) + own, list(pages[full:full + 1]) if rest else [], own

    def compact(self, move: Callable[[list[int], list[int]], None] | None = None) -> tuple[list[int], list[int]]:
        """(src ascending, dst): the moves after which the used pages are 0 .. used. The counts move with
        them; whoever holds page numbers has to replace src[i] by dst[i]. ``move(src, dst)`` is called first
        where there is something to move: what it raises leaves the pool as it was."""
        with self._lock:
            used = self.used
            src = [p for p in range(used, self.pages) if self._count[p]]
            dst = [p for p in range(used) if not self._count[p]]
            if src and move is not None:
                move(src, dst)
            for a, b in zip(src, dst):
                self._count[b], self._count[a] = self._count[a], 0
            self._free = list(range(used, self.pages))
            return src, dst


class Kv4Pages:
    """A state's pages and its row of the tables; given back when nothing refers to them any more."""

    __slots__ = ("states", "row", "pages", "tokens")

    def __init__(self, states: "Kv4States", row: int, pages: list[int], tokens: int):
        self.states, self.row, self.pages, self.tokens = states, row, pages, tokens

    def __del__(self):
        try:
            self.states._drop(self.row)
        except Exception:  # interpreter shutdown, or a constructor that failed
            pass


@dataclass(slots=True, eq=False)
class Kv4Entry:
    """A full-attention layer's state keys and values in pages (``AttentionEntry`` in 4 bits)."""

    cache: Kv4Cache
    layer: int  # of the cache
    table: torch.Tensor  # [pages] int32, a row of the states' tables
    tokens: int
    held: Kv4Pages | None = field(default=None, repr=False)  # keeps the pages

    @property
    def held_bytes(self) -> int:
        """Bytes of the layer's pages; those that a fork shares count for each state that does."""
        return self.table.numel() * self.cache.pool.shape[2]


class Kv4Snapshot(list):
    """A snapshot with ``Kv4Entry`` entries; its pages live as long as this list or an entry of it."""

    packable = False  # not tensors: a state cache keeps it as it is

    def __init__(self, entries: Sequence[Any], held: Kv4Pages):
        super().__init__(entries)
        self.held, self.tokens = held, held.tokens

    @property
    def states(self) -> "Kv4States":
        return self.held.states

    @property
    def row(self) -> int:
        return self.held.row

    @property
    def pages(self) -> list[int]:
        return self.held.pages


class Kv4States:
    """Snapshots in 4 bits: one cache for all full-attention layers, its pages and its tables.

    ``max_tokens`` bounds a state's length, ``max_states`` how many are held at a time."""

    def __init__(self, layers: int, pages: int, *, kv_heads: int, head_dim: int, page_tokens: int = 64,
                 max_tokens: int = 16384, max_states: int = 64, device: torch.device | str | int | None = None):
        self.cache = Kv4Cache(layers, pages, kv_heads=kv_heads, head_dim=head_dim, page_tokens=page_tokens, device=device)
        self.pool = PagePool(pages)
        width = -(-int(max_tokens) // page_tokens)
        if max_states < 1 or width < 1:
            raise ValueError("max_states and max_tokens must be positive")
        self.tables = torch.full((max_states, width), -1, dtype=torch.int32, device=self.cache.device)
        self._rows = list(range(max_states))
        self._held: dict[int, list[int]] = {}  # the pages of the states, by row; the snapshots share the lists
        self._lock = threading.RLock()
        self._moving = False
        self._dropped: list[int] = []  # rows whose snapshot went while the pages moved

    @staticmethod
    def pages_for(tokens: int, page_tokens: int = 64) -> int:
        return -(-int(tokens) // page_tokens)

    def stats(self) -> dict[str, int]:
        size = page_bytes(self.cache.kv_heads, self.cache.head_dim, self.cache.page_tokens) * self.cache.layers
        return {"pages": self.pool.pages, "used_pages": self.pool.used, "used_bytes": self.pool.used * size,
                "states": len(self._held)}

    def _drop(self, row: int) -> None:
        with self._lock:
            if self._moving:  # a finaliser that ran inside compact(): this thread holds the lock already
                self._dropped.append(row)
                return
            self.pool.release(self._held.pop(row))
            heapq.heappush(self._rows, row)

    def _snapshot(self, entries: Sequence[Any], pages: list[int], tokens: int, write: int) -> Kv4Snapshot:
        """A snapshot over ``pages`` (already counted for it); tables from page ``write`` on are set."""
        row = heapq.heappop(self._rows)
        self._held[row] = pages
        snap = Kv4Snapshot([], Kv4Pages(self, row, pages, tokens))
        self._fill(snap, write)
        layer = 0
        for e in entries:
            if isinstance(e, (AttentionEntry, Kv4Entry)):
                e = Kv4Entry(self.cache, layer, self.tables[row, :len(pages)], tokens, snap.held)
                layer += 1
            snap.append(e)
        return snap

    def _fill(self, snap: Kv4Snapshot, first: int) -> None:
        if first < len(snap.pages):
            self.tables[snap.row, first:len(snap.pages)] = torch.tensor(snap.pages[first:], dtype=torch.int32).to(
                self.tables.device)

    def store(self, snapshot: Sequence[Any]) -> Kv4Snapshot | None:
        """The snapshot with its K/V quantised into pages; None where no pages or no row are free. Other
        entries (the GDN layers') are kept as they are."""
        entries = [e for e in snapshot if isinstance(e, AttentionEntry)]
        if len(entries) != self.cache.layers:
            raise RuntimeError(f"a snapshot with {len(entries)} attention entries for a cache of {self.cache.layers} layers")
        shapes = {(tuple(e.keys.shape), tuple(e.values.shape)) for e in entries}
        if entries and (len(shapes) != 1 or entries[0].keys.dim() != 4 or entries[0].keys.shape[0] != 1):
            raise RuntimeError(f"attention entries must be [1, H_kv, S, D] alike, got {shapes}")
        tokens = entries[0].keys.shape[2] if entries else 0
        with self._lock:
            need = self.pages_for(tokens, self.cache.page_tokens)
            if need > self.tables.shape[1]:
                raise RuntimeError(f"a state of {tokens} tokens, tables hold {self.tables.shape[1] * self.cache.page_tokens}")
            pages = self.pool.allocate(need) if self._rows else None
            if pages is None:
                return None
            snap = self._snapshot(snapshot, pages, tokens, 0)
            if tokens:
                slots = self.cache.slots(snap_table(snap), 0, tokens)
                for layer, e in enumerate(entries):
                    self.cache.append(layer, e.keys[0].transpose(0, 1), e.values[0].transpose(0, 1), slots)
            return snap

    def _own(self, snap: Kv4Snapshot) -> None:
        if not isinstance(snap, Kv4Snapshot) or snap.states is not self:
            raise RuntimeError("not a snapshot that these states hold")

    def fork(self, snap: Kv4Snapshot) -> Kv4Snapshot | None:
        """A snapshot of the same state that can be extended by itself: its full pages are shared, a partly
        filled last one is copied in every layer. None where no page or row is free."""
        self._own(snap)
        with self._lock:
            if not self._rows:
                return None
            got = self.pool.fork(snap.pages, snap.tokens, self.cache.page_tokens)
            if got is None:
                return None
            pages, src, dst = got
            new = self._snapshot(snap, pages, snap.tokens, 0)
            self.cache.copy_pages(src, dst)
            return new

    def extend(self, snap: Kv4Snapshot, count: int) -> torch.Tensor | None:
        """int64 slots of ``count`` new tokens of ``snap``, to append K/V to in every layer; its entries then
        have them. Only for a snapshot whose last page is its own (a stored one that was not forked since,
        or a fork). None where no pages are free. The slots are places in the pool: append before the next
        ``compact``. A ``StateCache`` counts the pages that a snapshot had when it was put: put it again."""
        self._own(snap)
        with self._lock:
            page = self.cache.page_tokens
            if snap.tokens != snap.held.tokens:
                raise RuntimeError("a copy of this snapshot was extended already: extend a fork")
            need = self.pages_for(snap.tokens + count, page)
            if count < 0 or need > self.tables.shape[1]:
                raise RuntimeError(f"{snap.tokens} + {count} tokens, tables hold {self.tables.shape[1] * page}")
            if count and snap.tokens % page and self.pool.references(snap.pages[-1]) > 1:
                raise RuntimeError("the last page is shared: extend a fork")
            more = self.pool.allocate(need - len(snap.pages))
            if more is None:
                return None
            first = len(snap.pages)
            snap.pages.extend(more)
            self._fill(snap, first)
            slots = self.cache.slots(snap_table(snap), snap.tokens, count)
            snap.tokens = snap.held.tokens = snap.tokens + count
            for i, e in enumerate(snap):
                if isinstance(e, Kv4Entry):
                    snap[i] = dataclasses.replace(e, table=snap_table(snap), tokens=snap.tokens)
            return slots

    def compact(self) -> int:
        """Move the used pages to the front of the pool, in every layer and table, in one launch; how many
        moved."""
        with self._lock:
            self._moving = True
            try:
                src, dst = self.pool.compact(lambda src, dst: self.cache.move_pages(src, dst, self.tables))
                to = dict(zip(src, dst))
                for pages in self._held.values():
                    pages[:] = [to.get(p, p) for p in pages]
            finally:
                self._moving = False
                while self._dropped:
                    self._drop(self._dropped.pop())
            return len(src)


def snap_table(snap: Kv4Snapshot) -> torch.Tensor:
    """The snapshot's page table [pages] int32."""
    return snap.states.tables[snap.row, :len(snap.pages)]


__all__ = ["Kv4Entry", "Kv4Snapshot", "Kv4States", "PagePool"]
