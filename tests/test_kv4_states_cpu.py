"""The bookkeeping of states in 4-bit pages over a cache that only notes what it is asked for."""

from __future__ import annotations

import copy
import gc

import pytest
import torch

from conftest import ROOT  # noqa: F401  (puts the repository on sys.path)

from d3_turbo_trt_b200.kernels import kv4
from d3_turbo_trt_b200.model import pages
from d3_turbo_trt_b200.model.cache import StateCache
from d3_turbo_trt_b200.model.snapshot import AttentionEntry


class NotingCache:
    """The parts of a ``Kv4Cache`` that states use, on the CPU."""

    def __init__(self, layers, count, *, kv_heads, head_dim, page_tokens, device=None):
        self.layers, self.pages, self.kv_heads, self.head_dim, self.page_tokens = layers, count, kv_heads, head_dim, page_tokens
        self.device, self.calls = torch.device("cpu"), []
        self.pool = torch.zeros(layers, count, kv4.page_bytes(kv_heads, head_dim, page_tokens), dtype=torch.uint8)

    slots = kv4.Kv4Cache.slots

    def append(self, layer, k, v, slots):
        self.calls.append(("append", layer, slots.tolist()))

    def copy_pages(self, src, dst):
        self.calls.append(("copy", list(src), list(dst)))

    def move_pages(self, src, dst, tables):
        self.calls.append(("move", list(src), list(dst)))
        to = dict(zip(src, dst))
        tables.copy_(torch.tensor([[to.get(p, p) for p in row] for row in tables.tolist()], dtype=torch.int32))


@pytest.fixture
def states(monkeypatch):
    monkeypatch.setattr(pages, "Kv4Cache", NotingCache)
    return pages.Kv4States(1, 12, kv_heads=1, head_dim=64, page_tokens=16, max_tokens=96, max_states=5)


def snapshot(tokens):
    x = torch.zeros(1, 1, tokens, 64)
    return [AttentionEntry(x, x)]


def test_pages_live_as_long_as_an_entry(states):
    """A plain list of the entries, a slice, one entry or a copy keeps the pages; the row is not given out again."""
    for keep in (lambda s: list(s), lambda s: s[:1], lambda s: s[0], copy.copy, lambda s: s + []):
        snap = states.store(snapshot(40))
        kept, mine = keep(snap), list(snap.pages)
        del snap
        gc.collect()
        assert states.pool.used == 3 and states.stats()["states"] == 1
        other = states.store(snapshot(16))
        entry = kept if isinstance(kept, pages.Kv4Entry) else kept[0]
        assert entry.table.tolist() == mine and not set(mine) & set(other.pages)
        del other, entry, kept
        gc.collect()
        assert states.pool.used == 0 and states.stats()["states"] == 0


def test_a_copy_dropped_leaves_the_other(states):
    snap = states.store(snapshot(40))
    twin = copy.copy(snap)
    assert twin.pages == snap.pages and twin.tokens == 40 and twin.states is states
    del snap
    gc.collect()
    again = states.store(snapshot(40))
    del twin
    gc.collect()
    assert states.pool.used == 3 and [states.pool.references(p) for p in again.pages] == [1, 1, 1]


def test_only_one_copy_is_extended(states):
    snap = states.store(snapshot(20))
    twin = copy.copy(snap)
    assert states.extend(snap, 10).tolist() == [p * 16 + i for p, i in [(snap.pages[1], i) for i in range(4, 14)]]
    with pytest.raises(RuntimeError, match="extended already"):
        states.extend(twin, 3)
    assert twin.tokens == 20 and twin[0].tokens == 20 and snap.tokens == 30 and snap[0].tokens == 30
    assert states.extend(snap, 3) is not None
    fork = states.fork(twin)  # of the 20 tokens that it knows
    assert fork.tokens == 20 and len(fork.pages) == 2 and states.extend(fork, 1) is not None


def test_a_compaction_whose_move_fails(states, monkeypatch):
    """An error of the launch leaves counts, free pages, tables and states as they were; the next one moves them."""
    hole = states.store(snapshot(33))
    base = states.store(snapshot(40))
    fork = states.fork(base)
    del hole
    gc.collect()
    before = ([states.pool.references(p) for p in range(12)], states.pool.free, states.tables.tolist(), list(base.pages), list(fork.pages))

    def fails(src, dst, tables):
        raise RuntimeError("no launch")

    monkeypatch.setattr(states.cache, "move_pages", fails, raising=False)
    with pytest.raises(RuntimeError, match="no launch"):
        states.compact()
    assert before == ([states.pool.references(p) for p in range(12)], states.pool.free, states.tables.tolist(), base.pages, fork.pages)
    got = states.pool.allocate(states.pool.free)
    assert not set(got) & (set(base.pages) | set(fork.pages))
    states.pool.release(got)
    monkeypatch.undo()
    assert states.compact() == 3
    assert sorted(set(base.pages) | set(fork.pages)) == [0, 1, 2, 3] and base[0].table.tolist() == base.pages
    del base, fork
    gc.collect()
    assert states.pool.used == 0


def test_snapshots_of_others_are_refused(states, monkeypatch):
    """Another pool's page numbers mean nothing here."""
    mine = states.store(snapshot(20))
    monkeypatch.setattr(pages, "Kv4Cache", NotingCache)
    other = pages.Kv4States(1, 12, kv_heads=1, head_dim=64, page_tokens=16, max_tokens=96, max_states=5)
    theirs = other.store(snapshot(20))
    for bad in (theirs, list(mine), snapshot(20)):
        with pytest.raises(RuntimeError, match="not a snapshot"):
            states.fork(bad)
        with pytest.raises(RuntimeError, match="not a snapshot"):
            states.extend(bad, 1)
    assert states.pool.used == other.pool.used == 2 and len(states.cache.calls) == len(other.cache.calls) == 1


def test_a_state_cache_counts_a_snapshot_put_again(states):
    held = StateCache(10**6)
    snap = states.store(snapshot(20))
    first = held.put("a", snap, 20).nbytes
    assert states.extend(snap, 30) is not None
    assert held.put("a", snap, 50).nbytes == 2 * first == held.bytes and held.count == 1
    del snap
    gc.collect()
    assert states.pool.used == 4
    held.clear()
    gc.collect()
    assert states.pool.used == 0
