"""The tables of lengths that calls make of host lists: how long they live."""

from __future__ import annotations

import threading

import pytest
import torch

from conftest import ROOT  # noqa: F401  (puts the repository on sys.path)

from d3_turbo_trt_b200 import _lib
from d3_turbo_trt_b200.kernels import kv4
from d3_turbo_trt_b200.kernels import prefix_bidir as pb


def test_block_offset_table_of_a_captured_call_stays(monkeypatch):
    """A captured call's table outlives any number of others; one that was not made before the capture is refused."""
    monkeypatch.setattr(pb, "_LENGTHS", type(pb._LENGTHS)())
    monkeypatch.setattr(pb, "_LENGTHS_CAPTURED", {})
    device = torch.device("cpu")
    table = pb.block_offsets([5, 6], device)
    capture = lambda on: monkeypatch.setattr(pb, "_stream_now", lambda d: (0, on))  # noqa: E731
    capture(True)
    assert pb.block_offsets([5, 6], device) is table
    with pytest.raises(RuntimeError, match="captured"):
        pb.block_offsets([6, 5], device)
    capture(False)
    for i in range(40):
        pb.block_offsets([i, i + 1, 0], device)
    assert len(pb._LENGTHS) == pb._LENGTHS_MAX
    capture(True)
    assert pb.block_offsets([5, 6], device) is table


def test_block_offset_tables_by_several_threads():
    errors = []

    def work(seed):
        try:
            for i in range(400):
                n = (seed * 7 + i * 13) % 23
                assert pb.block_offsets([n, n + 1], torch.device("cpu")).tolist() == [n, n + 1]
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in range(8)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors and len(pb._LENGTHS) <= pb._LENGTHS_MAX


def others(device, first=100):
    """Twenty more tables and a few blocks of their size with other contents: what was freed is used again."""
    for i in range(20):
        pb.block_offsets([first + i, 0, 0], device)
    return [torch.full((3,), 7, dtype=torch.int32, device=device) for _ in range(64)]


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["question in place", "question widened", "prefix"])
def test_a_captured_call_with_host_lengths(monkeypatch, which):
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: which == "question in place")
    monkeypatch.setattr(pb, "_LENGTHS", type(pb._LENGTHS)())
    monkeypatch.setattr(pb, "_LENGTHS_CAPTURED", {})
    kv4._plans_of.cache_clear()
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    cache, table = kv4.Kv4Cache(1, 4, kv_heads=2, head_dim=128, page_tokens=32), torch.arange(4, dtype=torch.int32, device="cuda")
    cache.append(0, new(100, 2, 128), new(100, 2, 128), cache.slots(table, 0, 100))
    q, k, v = new(3, 8, 9, 128), new(3, 2, 9, 128), new(3, 2, 9, 128)
    ks, vs = cache.read(0, table, 100)

    def ask(lengths):
        if which == "prefix":
            return pb.prefix_bidir_attention(q, ks, vs, k, v, lengths, scale=0.1)
        return kv4.question_attention(q, cache, 0, table, 100, k, v, lengths, scale=0.1)

    want = ask([5, 0, 9])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ask([5, 0, 9])
    kept = others(q.device)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and len(kept) == 64
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0


@pytest.mark.gpu
def test_a_table_used_on_another_stream_outlives_its_work(monkeypatch):
    """Made on one stream, read on another behind a long wait, dropped from the cache meanwhile."""
    monkeypatch.setattr(pb, "_LENGTHS", type(pb._LENGTHS)())
    g = torch.Generator(device="cuda").manual_seed(2)
    new = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    q, k, v, ks, vs = new(3, 4, 9, 64), new(3, 2, 9, 64), new(3, 2, 9, 64), new(2, 70, 64), new(2, 70, 64)
    want = pb.prefix_bidir_attention(q, ks, vs, k, v, [5, 0, 9], scale=0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        got = pb.prefix_bidir_attention(q, ks, vs, k, v, [5, 0, 9], scale=0.1)
    kept = others(q.device)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(kept) == 64 and _lib.device_error() == 0
