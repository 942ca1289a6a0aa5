"""States in 4-bit pages as a user runs them: stored from a state pass, forked, extended, decoded, compacted and
asked questions, and the backbone's request over them."""

from __future__ import annotations

import gc

import numpy as np
import pytest
import torch

import e2e_model as em
from conftest import ROOT  # noqa: F401
from test_kv4_gpu import check_question, decode_bound, half_step, rows

from d3_turbo_trt_b200 import _lib
from d3_turbo_trt_b200.kernels import kv4
from d3_turbo_trt_b200.model import fused
from d3_turbo_trt_b200.model.backbone import BackboneConfig, D3Backbone
from d3_turbo_trt_b200.model.cache import StateCache
from d3_turbo_trt_b200.model.pages import Kv4Entry, Kv4States
from d3_turbo_trt_b200.model.snapshot import AttentionEntry, DeltaEntry
from oracle import kv4 as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make_snapshot(layers, kv_heads, tokens, dim, seed):
    snap, kept = [], []
    for i in range(layers):
        k, v = rows((1, tokens, kv_heads, dim), BF, seed + 2 * i, 0.3), rows((1, tokens, kv_heads, dim), BF, seed + 2 * i + 1, 0.3)
        snap.append(AttentionEntry(k.cuda().transpose(1, 2), v.cuda().transpose(1, 2)))
        snap.append(DeltaEntry(torch.ones(1, 4, 3, device="cuda"), torch.ones(1, 1, 2, 2, device="cuda")))
        kept.append((ref.stored(k[0]).transpose(0, 1), ref.stored(v[0]).transpose(0, 1)))
    return snap, kept


def check_decode_entry(entry, kept, q, scale):
    got = kv4.decode_attention(q.cuda(), entry.cache, entry.layer, entry.table[None],
                               torch.tensor([entry.tokens], dtype=torch.int32, device="cuda"), scale=scale).cpu().double()
    out, mass, top = ref.attention(q[0], kept[0], kept[1], scale)
    n = kept[0].shape[1]
    bound = decode_bound(out, mass, top, n, float(kept[1].abs().max()), q.shape[-1], q.dtype)
    assert bool(((got[0] - out).abs() <= bound).all())


def test_store_fork_extend_compact_question():
    layers, kv_heads, dim, page, tokens = 3, 2, 128, 32, 75
    states = Kv4States(layers, 24, kv_heads=kv_heads, head_dim=dim, page_tokens=page, max_tokens=256, max_states=6)
    snap, kept = make_snapshot(layers, kv_heads, tokens, dim, 1)
    other, _ = make_snapshot(layers, kv_heads, 200, dim, 50)
    first = states.store(other)  # pages 0 .. 6, dropped below: a hole in front
    base = states.store(snap)
    assert [type(e) for e in base] == [Kv4Entry, DeltaEntry] * layers and base[0].tokens == tokens
    q = rows((1, 4, 1, dim), BF, 9, 0.2)
    for i in range(layers):
        check_decode_entry(base[2 * i], kept[i], q, 0.09)
    forks = [states.fork(base) for _ in range(2)]
    assert states.stats()["used_pages"] == 7 + 3 + 2  # two full pages shared, a last one each
    with_new = []
    for f, fork in enumerate(forks):
        slots = states.extend(fork, 30)  # into the copied last page, and a new one
        grown = []
        for i in range(layers):
            k, v = rows((30, kv_heads, dim), BF, 100 + 10 * f + i), rows((30, kv_heads, dim), BF, 200 + 10 * f + i)
            states.cache.append(i, k.cuda(), v.cuda(), slots)
            grown.append((torch.cat([kept[i][0], ref.stored(k).transpose(0, 1)], 1),
                          torch.cat([kept[i][1], ref.stored(v).transpose(0, 1)], 1)))
        with_new.append(grown)
    with pytest.raises(RuntimeError, match="shared|tables"):
        states.extend(base, 1000)
    del first
    gc.collect()
    for round_ in range(2):
        for i in range(layers):
            check_decode_entry(base[2 * i], kept[i], q, 0.09)
            for fork, grown in zip(forks, with_new):
                assert fork[2 * i].tokens == tokens + 30
                check_decode_entry(fork[2 * i], grown[i], q, 0.09)
        if round_ == 0:
            used = states.pool.used
            assert states.compact() > 0
            assert max(p for s in [base, *forks] for p in s.pages) == used - 1
            assert states.compact() == 0
    # a question batch over a fork's state
    B, L = 3, 9
    qs = rows((B, L, 4, dim), BF, 5, 0.2).transpose(1, 2)
    k, v = rows((B, kv_heads, L, dim), BF, 6, 0.2), rows((B, kv_heads, L, dim), BF, 7, 0.2)
    e = forks[1][2]
    got = kv4.question_attention(qs.cuda(), e.cache, e.layer, e.table, e.tokens, k.cuda(), v.cuda(), [9, 0, 4], scale=0.09)
    check_question(got, qs, with_new[1][1], k, v, [9, 0, 4], 0.09, BF)
    del e, base, forks, fork
    gc.collect()
    assert states.pool.used == 0 and states.stats()["states"] == 0
    assert _lib.device_error() == 0


def test_a_snapshot_dropped_while_pages_move(monkeypatch):
    # a finaliser may run inside compact() on the same thread: its pages must be those it has after the move
    states = Kv4States(1, 8, kv_heads=1, head_dim=64, page_tokens=16, max_tokens=64, max_states=4)
    snap, kept = make_snapshot(1, 1, 30, 64, 3)
    held = [states.store(snap) for _ in range(3)]
    held.pop(0)
    gc.collect()
    move = states.cache.move_pages

    def moves(src, dst, tables):
        held.pop()  # the one whose pages lie last
        gc.collect()
        move(src, dst, tables)

    monkeypatch.setattr(states.cache, "move_pages", moves)
    assert states.compact() == 2
    assert states.pool.used == 2 and states.stats()["states"] == 1
    monkeypatch.undo()
    check_decode_entry(held[0][0], kept[0], rows((1, 2, 1, 64), BF, 9, 0.2), 0.1)
    states.compact()
    assert sorted(held[0].pages) == [0, 1]
    check_decode_entry(held[0][0], kept[0], rows((1, 2, 1, 64), BF, 9, 0.2), 0.1)
    assert states.store(snap) is not None and _lib.device_error() == 0


def test_a_captured_step_replayed():
    # rotation, append and attention of one token of two sequences in a graph, run for four tokens, against eager calls
    B, heads, kv_heads, dim, page, steps = 2, 6, 2, 128, 16, 4
    table = torch.arange(8, dtype=torch.int32, device="cuda").flip(0).view(B, 4)
    start = [14, 30]  # the second token of both begins a page
    inv = (10000.0 ** (-torch.arange(32) / 32)).float().cuda()
    axes = fused.rotary_axes([12, 10, 10])
    w = rows((2, dim), BF, 3, 0.1).cuda()
    qs, ks, vs = (rows((steps, B, 1, n, dim), BF, 4 + n, 0.5).cuda() for n in (heads, kv_heads, kv_heads))
    q, k, v = (x[0].clone() for x in (qs, ks, vs))
    lengths = torch.tensor(start, dtype=torch.int32, device="cuda")

    def run(cache):
        at = lengths.to(torch.int64)
        positions = torch.stack([at, at // 2, at // 3]).view(3, B, 1)
        slots = table.gather(1, (at // page)[:, None]).view(B).to(torch.int64) * page + at % page
        rq, rk = fused.qk_norm_mrope(q, k, w[0], w[1], positions, inv, axes, 1e-6)
        cache.append(0, rk[:, 0], v[:, 0], slots)
        return kv4.decode_attention(rq.transpose(1, 2), cache, 0, table, lengths + 1, scale=dim**-0.5)

    def fresh():
        cache = kv4.Kv4Cache(1, 8, kv_heads=kv_heads, head_dim=dim, page_tokens=page)
        for b, n in enumerate(start):
            old = rows((n, kv_heads, dim), BF, 20 + b).cuda()
            cache.append(0, old, old, cache.slots(table[b], 0, n))
        lengths.copy_(torch.tensor(start, dtype=torch.int32))
        return cache

    cache, want = fresh(), []
    for i in range(steps):
        q.copy_(qs[i]), k.copy_(ks[i]), v.copy_(vs[i])
        want.append(run(cache))
        lengths.add_(1)
    cache = fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(cache)
    for i in range(steps):
        q.copy_(qs[i]), k.copy_(ks[i]), v.copy_(vs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        lengths.add_(1)
    assert not torch.equal(want[0], want[1]) and _lib.device_error() == 0


@pytest.mark.parametrize("in_place", [True, False])
def test_a_captured_question_batch(monkeypatch, in_place):
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    kv4._plans_of.cache_clear()
    cache = kv4.Kv4Cache(1, 6, kv_heads=2, head_dim=128, page_tokens=32)
    table, lens = torch.arange(6, dtype=torch.int32, device="cuda"), torch.tensor([5, 0, 9], dtype=torch.int32, device="cuda")
    old = rows((150, 2, 128), BF, 1, 0.5)
    cache.append(0, old.cuda(), old.cuda(), cache.slots(table, 0, 150))
    kept = ref.stored(old).transpose(0, 1)
    q, k, v = (rows((3, 9, n, 128), BF, n + s, 0.5).transpose(1, 2) for n, s in ((8, 1), (2, 2), (2, 3)))
    on = [x.cuda() for x in (q, k, v)]
    ask = lambda: kv4.question_attention(on[0], cache, 0, table, 150, on[1], on[2], lens, scale=128**-0.5)  # noqa: E731
    check_question(ask(), q, (kept, kept), k, v, [5, 0, 9], 128**-0.5, BF)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ask()
    for lengths in ([5, 0, 9], [9, 1, 3]):
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_question(out, q, (kept, kept), k, v, lengths, 128**-0.5, BF)
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("in_place", [True, False])
def test_two_question_graphs_side_by_side(monkeypatch, in_place):
    # captured on one stream, the later one replayed first, then both at once on two streams
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    kv4._plans_of.cache_clear()
    tokens, B, L = 4096, 2, 40
    cache = kv4.Kv4Cache(1, 32, kv_heads=4, head_dim=256, page_tokens=128)
    table, lens = torch.arange(32, dtype=torch.int32, device="cuda"), torch.full((B,), L, dtype=torch.int32, device="cuda")
    assert _lib.lib().d3b_prefix_bidir_workspace_size(B, 24, 4, tokens, L, 256) > 0
    old = rows((tokens, 4, 256), BF, 1, 0.5).cuda()
    cache.append(0, old, old, cache.slots(table, 0, tokens))
    args = [[rows((B, L, n, 256), BF, 10 * g + n, 0.5).cuda().transpose(1, 2) for n in (24, 4, 4)] for g in range(2)]
    ask = lambda g: kv4.question_attention(args[g][0], cache, 0, table, tokens, args[g][1], args[g][2], lens, scale=0.1)  # noqa: E731
    want, graphs, outs, streams = [ask(g) for g in range(2)], [], [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    cap = torch.cuda.Stream()
    for g in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[g], stream=cap):
            outs.append(ask(g))
    for order in ((1,), (0,), *((1, 0), (0, 1)) * 10):
        for g in order:
            with torch.cuda.stream(streams[g]):
                outs[g].fill_(1)
                graphs[g].replay()
        torch.cuda.synchronize()
        for g in order:  # a unit's parts are added in the order in which they end: within their rounding of each other
            assert float((outs[g].float() - want[g].float()).abs().max()) <= 2 * half_step(BF) * float(want[g].abs().max())
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0


def test_no_room_and_shared_last_page():
    # five pages: three of the state, one copied by its fork, one that the fork grows into
    states = Kv4States(1, 5, kv_heads=1, head_dim=64, page_tokens=16, max_tokens=64, max_states=2)
    snap, _ = make_snapshot(1, 1, 33, 64, 3)
    a = states.store(snap)
    assert states.store(snap) is None and states.pool.used == 3  # three pages wanted, two free
    b = states.fork(a)
    assert states.fork(a) is None  # no row
    assert states.extend(b, 31) is not None and b[0].tokens == 64
    with pytest.raises(RuntimeError):
        states.extend(b, 1)  # beyond the tables
    del b
    gc.collect()
    with pytest.raises(RuntimeError):
        states.store([snap[0], snap[0]])
    long, _ = make_snapshot(1, 1, 65, 64, 4)
    with pytest.raises(RuntimeError):
        states.store(long)
    assert states.pool.used == 3


def test_state_cache_evicts_pages():
    states = Kv4States(1, 16, kv_heads=1, head_dim=64, page_tokens=16, max_tokens=64, max_states=16)
    size = 2 * kv4.page_bytes(1, 64, 16)
    held = StateCache(2 * (size + 4 * (12 + 4)))
    for i in range(4):
        snap, _ = make_snapshot(1, 1, 20, 64, i)
        held.put(str(i), states.store(snap), 20)
    del snap
    gc.collect()
    assert held.count == 2 and held.evictions == 2 and states.pool.used == 4


@pytest.fixture(scope="module")
def request_():
    bb = D3Backbone(BackboneConfig(**em.CONFIG, mrope_section=(6, 5, 5)), em.make_weights(), device=torch.device("cuda"), mode="fp8")
    return bb, em.make_request()


def probabilities(bb, snap, request, **kw):
    state, ids, lengths, counts, readout = request
    hidden = bb.questions(snap, ids, lengths, state_len=state.shape[1], **kw)
    return bb.probabilities(hidden, readout.cuda(), counts).cpu().numpy()


def test_backbone_over_a_4_bit_state(request_):
    """The question pass over the pages against the same pass over what the pages read back as: one softmax's
    rounding apart, within the gate of the end-to-end test."""
    bb, request = request_
    states = Kv4States(1, 40, kv_heads=2, head_dim=128, page_tokens=16, max_tokens=1024, max_states=3)
    snap = bb.state(request[0], states=states)
    assert isinstance(snap[3], Kv4Entry) and states.pool.used == 32
    got = probabilities(bb, snap, request)
    plain = list(snap)
    k, v = snap[3].cache.read(0, snap[3].table, snap[3].tokens)
    plain[3] = AttentionEntry(k[None], v[None])
    want = probabilities(bb, plain, request)
    assert np.abs(got - want).max() <= 1e-2 and np.array_equal(got.argmax(1), want.argmax(1))
    held = StateCache(64 << 20)
    held.put("s", snap, 512)
    del snap, plain
    again = probabilities(bb, held.get("s").snapshot, request)
    assert np.array_equal(again, got)
    held.clear()
    gc.collect()
    assert states.pool.used == 0
    small = Kv4States(1, 5, kv_heads=2, head_dim=128, page_tokens=16)
    with pytest.raises(RuntimeError, match="no pages"):
        bb.state(request[0], states=small)


def test_backbone_positions_on_three_axes(request_):
    """Equal positions on the three axes are the text pass; other positions change it."""
    bb, request = request_
    state, ids, *_ = request
    S, (B, W) = state.shape[1], ids.shape
    text = torch.arange(S)[None, None].expand(3, 1, -1)
    after = (S + torch.arange(W))[None, None].expand(3, B, -1)
    want = probabilities(bb, bb.state(state), request)
    got = probabilities(bb, bb.state(state, positions=text), request, positions=after)
    assert np.abs(got - want).max() <= 1e-2 and np.array_equal(got.argmax(1), want.argmax(1))
    moved = text.clone()
    moved[1:, :, S // 2:] += 5
    assert not np.array_equal(probabilities(bb, bb.state(state, positions=moved), request, positions=after), got)
    with pytest.raises(ValueError):
        bb.state(state, positions=text[:2])
    with pytest.raises(ValueError):
        bb.state(state, positions=text[:, :, 1:])


def test_backbone_head_dim_256():
    config = dict(em.CONFIG, head_dim=256, num_attention_heads=6, num_key_value_heads=2)
    bb = D3Backbone(BackboneConfig(**config, mrope_section=(11, 11, 10)), em.make_weights(config), device=torch.device("cuda"), mode="fp8")
    request = em.make_request()
    states = Kv4States(1, 20, kv_heads=2, head_dim=256, page_tokens=32, max_tokens=1024)
    p16, p4 = (probabilities(bb, bb.state(request[0], states=s), request) for s in (None, states))
    assert np.isfinite(p16).all() and np.isfinite(p4).all() and _lib.device_error() == 0
