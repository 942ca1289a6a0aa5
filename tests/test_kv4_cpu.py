"""The 4-bit cache without a GPU: what the C ABI refuses before any launch, the page bookkeeping, the
rotary axes, and the oracle against hand-worked values."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from conftest import ROOT  # noqa: F401

from d3_turbo_trt_b200 import _lib
from d3_turbo_trt_b200.kernels import kv4
from d3_turbo_trt_b200.model import fused
from d3_turbo_trt_b200.model.cache import StateCache, tensor_bytes
from d3_turbo_trt_b200.model.pages import Kv4Entry, PagePool
from oracle import kv4 as ref

P = 4096  # an aligned address that nothing reads


def cache(pool=P, layers=2, pages=10, kv_heads=2, head_dim=64, page_tokens=16):
    return ctypes.byref(_lib.Kv4CacheStruct(pool, layers, pages, kv_heads, head_dim, page_tokens))


def st(*values):
    return _lib.i64_array(values)


def test_page_bytes():
    lib = _lib.lib()
    for dim in kv4.HEAD_DIMS:
        for page in kv4.PAGE_TOKENS:
            assert lib.d3b_kv4_page_bytes(3, dim, page) == kv4.page_bytes(3, dim, page) == 3 * page // 16 * (18 * dim + 32)
            assert ref.granule(torch.zeros(16, dim), torch.zeros(16, dim)).numel() == 18 * dim + 32
    for bad in ((0, 64, 16), (1, 96, 16), (1, 64, 24), (1, 64, 8), (1, 64, 512), (65536, 64, 16)):
        assert lib.d3b_kv4_page_bytes(*bad) == 0
        with pytest.raises(RuntimeError):
            kv4.page_bytes(*bad)


@pytest.mark.parametrize("over,code", [
    (dict(c=cache(head_dim=96)), _lib.EUNSUPPORTED), (dict(c=cache(page_tokens=48)), _lib.EUNSUPPORTED),
    (dict(c=cache(pool=P + 8)), _lib.EALIGN), (dict(c=cache(pool=None)), _lib.EINVAL), (dict(c=None), _lib.EINVAL),
    (dict(layer=2), _lib.EINVAL), (dict(layer=-1), _lib.EINVAL), (dict(n=-1), _lib.EINVAL), (dict(dtype=_lib.F32), _lib.EUNSUPPORTED),
    (dict(k=None), _lib.EINVAL), (dict(k=P + 2), _lib.EALIGN), (dict(ks=st(128, 60)), _lib.EALIGN), (dict(slots=None), _lib.EINVAL),
    (dict(slots=P + 4), _lib.EALIGN), (dict(n=0, k=None), _lib.OK)])
def test_append_refuses(over, code):
    a = dict(c=cache(), layer=0, k=P, ks=st(128, 64), v=P, vs=st(128, 64), slots=P, n=3, dtype=_lib.BF16) | over
    assert _lib.lib().d3b_kv4_append(a["c"], a["layer"], a["k"], a["ks"], a["v"], a["vs"], a["slots"], a["n"], a["dtype"], None) == code


@pytest.mark.parametrize("over,code", [
    (dict(tokens=33), _lib.EINVAL), (dict(tokens=-1), _lib.EINVAL), (dict(table=None), _lib.EINVAL), (dict(table=P + 2), _lib.EALIGN),
    (dict(k=P + 8), _lib.EALIGN), (dict(dtype=_lib.I32), _lib.EUNSUPPORTED), (dict(layer=5), _lib.EINVAL),
    (dict(tokens=0, table=None), _lib.OK)])
def test_read_refuses(over, code):
    a = dict(layer=0, table=P, n=2, tokens=32, k=P, v=P, dtype=_lib.F16) | over
    assert _lib.lib().d3b_kv4_read(cache(), a["layer"], a["table"], a["n"], a["tokens"], a["k"], a["v"], a["dtype"], None) == code


def test_move_pages_refuses():
    move = _lib.lib().d3b_kv4_move_pages
    assert move(cache(), P, P, 11, None, 0, None) == _lib.EINVAL  # more than the pool's pages
    assert move(cache(), P, P, -1, None, 0, None) == _lib.EINVAL
    assert move(cache(), None, P, 2, None, 0, None) == _lib.EINVAL
    assert move(cache(), P, P, 2, None, 4, None) == _lib.EINVAL  # entries without tables
    assert move(cache(), P + 2, P, 2, None, 0, None) == _lib.EALIGN
    assert move(cache(), None, None, 0, None, 0, None) == _lib.OK
    assert move(cache(head_dim=32), P, P, 1, None, 0, None) == _lib.EUNSUPPORTED


@pytest.mark.parametrize("over,code", [
    (dict(H=3), _lib.EINVAL), (dict(H=0), _lib.EINVAL), (dict(B=-1), _lib.EINVAL), (dict(L=-1), _lib.EINVAL), (dict(width=-1), _lib.EINVAL),
    (dict(dtype=_lib.F32), _lib.EUNSUPPORTED), (dict(scale=0.0), _lib.EINVAL), (dict(scale=float("nan")), _lib.EINVAL),
    (dict(scale=float("inf")), _lib.EINVAL), (dict(q=P + 8), _lib.EALIGN), (dict(out=None), _lib.EINVAL),
    (dict(qs=st(256, 64, 63)), _lib.EALIGN), (dict(table=None), _lib.EINVAL), (dict(stride=2), _lib.EINVAL), (dict(lengths=None), _lib.EINVAL),
    (dict(lengths=P + 1), _lib.EALIGN), (dict(work=None), _lib.ENOSPACE), (dict(bytes=64), _lib.ENOSPACE), (dict(work=P + 8), _lib.EALIGN),
    (dict(width=1 << 40), _lib.EINVAL), (dict(L=1 << 29), _lib.EINVAL), (dict(B=0), _lib.OK), (dict(L=0, q=None), _lib.OK),
    (dict(c=cache(page_tokens=17)), _lib.EUNSUPPORTED), (dict(layer=2), _lib.EINVAL)])
def test_decode_refuses(over, code):
    a = dict(c=cache(), layer=0, q=P, qs=st(256, 64, 64), table=P, stride=4, width=4, lengths=P, B=2, H=4, L=1, causal=0,
             dtype=_lib.BF16, scale=0.1, out=P, os=st(256, 64, 64), work=P, bytes=1 << 40) | over
    assert _lib.lib().d3b_kv4_decode(a["c"], a["layer"], a["q"], a["qs"], a["table"], a["stride"], a["width"], a["lengths"], a["B"],
                                     a["H"], a["L"], a["causal"], a["dtype"], a["scale"], a["out"], a["os"], a["work"], a["bytes"],
                                     None) == code


@pytest.mark.parametrize("over,code", [
    (dict(state=65), _lib.EINVAL), (dict(state=-1), _lib.EINVAL), (dict(k=None), _lib.EINVAL), (dict(v=P + 2), _lib.EALIGN),
    (dict(ks=st(64, 64, 4)), _lib.EALIGN), (dict(lengths=None), _lib.EINVAL), (dict(work=None), _lib.ENOSPACE), (dict(B=0), _lib.OK),
    (dict(H=5), _lib.EINVAL)])
def test_question_refuses(over, code):
    a = dict(q=P, qs=st(256, 64, 64), table=P, width=4, state=64, k=P, ks=st(128, 64, 64), v=P, vs=st(128, 64, 64), lengths=P, B=2,
             H=4, L=1, dtype=_lib.BF16, scale=0.1, out=P, os=st(256, 64, 64), work=P, bytes=1 << 40) | over
    assert _lib.lib().d3b_kv4_question(cache(), 0, a["q"], a["qs"], a["table"], a["width"], a["state"], a["k"], a["ks"], a["v"], a["vs"],
                                       a["lengths"], a["B"], a["H"], a["L"], a["dtype"], a["scale"], a["out"], a["os"], a["work"],
                                       a["bytes"], None) == code


@pytest.mark.parametrize("over,code", [
    (dict(D=96), _lib.EUNSUPPORTED), (dict(dtype=_lib.F32), _lib.EUNSUPPORTED), (dict(half=12), _lib.EUNSUPPORTED),
    (dict(half=40), _lib.EUNSUPPORTED), (dict(axes=9), _lib.EUNSUPPORTED), (dict(axes=0), _lib.EUNSUPPORTED),
    (dict(axis=bytes([0, 1, 2, 3] + [0] * 4)), _lib.EINVAL), (dict(q=None), _lib.EINVAL), (dict(q=P + 2), _lib.EALIGN),
    (dict(k=P + 2), _lib.EALIGN), (dict(ks=st(64, 64, 9)), _lib.EALIGN), (dict(pos=None), _lib.EINVAL), (dict(pos=P + 4), _lib.EALIGN),
    (dict(rows=-1), _lib.EINVAL), (dict(rows=0, q=None), _lib.OK), (dict(T=0), _lib.OK)])
def test_mrope_refuses(over, code):
    a = dict(q=P, qs=st(64, 64, 64), k=P, ks=st(64, 64, 64), w=P, pos=P, ps=st(1, 1, 1), freq=P, axis=bytes([0, 1, 2] + [0] * 5),
             axes=3, half=8, rows=1, T=1, D=64, dtype=_lib.BF16) | over
    assert _lib.lib().d3b_qk_norm_mrope(a["q"], a["qs"], 1, a["k"], a["ks"], 1, a["w"], a["w"], a["pos"], a["ps"], a["freq"], a["axis"],
                                        a["axes"], a["half"], P, P, a["rows"], a["T"], a["D"], a["dtype"], 1e-6, None) == code


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv4.Kv4Cache.over(torch.zeros(1, 2, kv4.page_bytes(1, 64, 16), dtype=torch.uint8), kv_heads=1, head_dim=64, page_tokens=16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv4.Kv4Cache(1, 2, kv_heads=1, head_dim=64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        fused.qk_norm_mrope(x, x, torch.zeros(64), torch.zeros(64), torch.zeros(1, 1, 1, dtype=torch.int64), torch.ones(8), [0] * 8, 1e-6)


def test_rotary_axes():
    axes = fused.rotary_axes([11, 11, 10])
    assert [axes.count(a) for a in range(3)] == [11, 11, 10] and axes[:7] == (0, 1, 2, 0, 1, 2, 0) and axes[-2:] == (0, 1)
    assert fused.rotary_axes([2, 1, 1], interleaved=False) == (0, 0, 1, 2)
    assert fused.rotary_axes([4]) == (0, 0, 0, 0)
    assert fused.rotary_axes([3, 0]) == (0, 0, 0)
    for bad in ([], [1, -1], [1, 3]):
        with pytest.raises(ValueError):
            fused.rotary_axes(bad)


# --------------------------------------------------------------------------- pages
def test_pool_against_a_plain_model():
    """Random allocations, shares, releases, forks and compactions; page contents are followed as a compaction moves them."""
    rng = random.Random(4)
    pool, held, content, stamp = PagePool(23), [], {}, 0
    for _ in range(3000):
        op = rng.randrange(5)
        if op == 0:
            n = rng.randrange(0, 5)
            got = pool.allocate(n)
            counts = sum(len(set(h)) for h in held)
            if got is None:
                assert pool.free < n
            else:
                assert len(set(got)) == n
                for p in got:
                    content[p] = stamp = stamp + 1
                held.append(got)
            del counts
        elif op == 1 and held:
            h = rng.choice(held)
            pool.share(h)
            held.append(list(h))
        elif op == 2 and held:
            pool.release(held.pop(rng.randrange(len(held))))
        elif op == 3 and held:
            h = rng.choice(held)
            tokens = rng.randrange(0, 16 * len(h) + 1)
            got = pool.fork(h, tokens, 16)
            if got is None:
                assert tokens % 16 and pool.free == 0
            else:
                pages, src, dst = got
                assert len(pages) == -(-tokens // 16) and pages[:tokens // 16] == h[:tokens // 16]
                assert src == (h[tokens // 16:tokens // 16 + 1] if tokens % 16 else []) and dst == pages[tokens // 16:]
                for a, b in zip(src, dst):
                    content[b] = content[a]
                held.append(pages)
        elif op == 4:
            before = [[content[p] for p in h] for h in held]
            src, dst = pool.compact()
            assert src == sorted(src) and not set(src) & set(dst) and len(set(dst)) == len(dst)
            to = dict(zip(src, dst))
            for a, b in to.items():
                content[b] = content[a]
            held = [[to.get(p, p) for p in h] for h in held]
            assert before == [[content[p] for p in h] for h in held]
            assert all(p < pool.used for h in held for p in h)
        refs = [sum(h.count(p) for h in held) for p in range(23)]
        assert [pool.references(p) for p in range(23)] == refs
        assert pool.used == sum(r > 0 for r in refs) == 23 - pool.free


def test_pool_refuses():
    pool = PagePool(4)
    a = pool.allocate(3)
    assert a == [0, 1, 2] and pool.allocate(2) is None and pool.free == 1
    for call in (lambda: pool.release([3]), lambda: pool.release([0, 0]), lambda: pool.release([-1]), lambda: pool.share([4]),
                 lambda: pool.allocate(-1), lambda: pool.fork(a, 49, 16), lambda: pool.fork([3], 3, 16)):
        with pytest.raises(ValueError):
            call()
    assert [pool.references(p) for p in range(4)] == [1, 1, 1, 0]
    with pytest.raises(ValueError):
        PagePool(-1)


def test_state_cache_counts_pages_and_keeps_them_unpacked():
    class FakeCache:
        pool = torch.zeros(1, 1, 1000, dtype=torch.uint8)

    entry = Kv4Entry(FakeCache(), 0, torch.zeros(3, dtype=torch.int32), 40)
    assert tensor_bytes([entry, torch.zeros(5)]) == 3000 + 20

    class Unpackable(list):
        packable = False

    held = StateCache(10_000, arena=object()).put("a", Unpackable([entry]), 40)
    assert held.nbytes == 3000 and isinstance(held.snapshot, Unpackable)


# --------------------------------------------------------------------------- the oracle itself
def test_oracle_values():
    x = torch.zeros(1, 64)
    x[0, :16] = torch.tensor([6.0, 5.0, -5.01, 4.99, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, 0.26, -0.25, 0.5, 1.0, 2688.0 / 448, 0.0])
    x[0, 16] = 2688.0
    x[0, 32] = 100.0  # scale: nearest e4m3 to 100/6 = 16.67 is 16 (step 2)
    got = ref.stored(x)[0]
    want = [6, 4, -6, 4, 4, 2, 2, 1, 1, 0, 0.5, 0, 0.5, 1, 6, 0]
    assert got[:16].tolist() == want and got[16] == 2688 and got[32] == 96
    assert int(ref.quantise(x)[2][0]) == 127  # 2688 = 6 * 448: exponent 0
    assert int(ref.quantise(x * 1.01)[2][0]) == 128
    assert int(ref.quantise(torch.zeros(1, 64))[2][0]) == 127 - 64
    code, scale, exponent = ref.quantise(torch.full((1, 64), float("inf")))
    assert int(exponent[0]) == 255 and not code.any() and not scale.any()


def test_oracle_granule_round_trip():
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(16, 128, generator=g), torch.randn(16, 128, generator=g)
    parts = ref.parts(ref.granule(k, v), 128)
    assert torch.equal(ref.values(*parts[0]), ref.stored(k)) and torch.equal(ref.values(*parts[1]), ref.stored(v))
