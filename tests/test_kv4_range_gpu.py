"""The 4-bit cache's attention where magnitudes lie far apart: query rows of one tile, V rows of one step, and a
block's own rows, in place and over a widened state. The bounds go by channel."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import ROOT  # noqa: F401  (puts the repository on sys.path)
from test_kv4_gpu import BF, HF, half_step, new_cache, rows

from d3_turbo_trt_b200 import _lib
from d3_turbo_trt_b200.kernels import kv4
from oracle import kv4 as ref

pytestmark = pytest.mark.gpu


def channel_bound(out, mass, spread, top, keys, dim, dtype, widened=False):
    """How far a kernel output may be from ``out``, channel by channel (all float64).

    * the output's rounding: half a step of it, and of the subnormals' spacing;
    * scores: a product is exact, its fp32 sum of dim terms is off by at most dim * 2^-24 of the sum of magnitudes
      (``top`` bounds that), three fp32 factors by 2^-22 more; a score off by d changes a weight by a factor e^(2 d);
    * weights: 2^-11 of each and 2^-25 of the largest one in fp16, so 2^-25 of |V| in this channel at most
      (``spread`` sums it over the keys); ex2 is off by 2^-22, sums of ``keys`` terms by keys * 2^-24;
    * over a widened state, or over its own keys, a weight has the inputs' type: half a step of it, twice.
    """
    weight = 2.0**-11 + 2 * top * (dim + 6) * 2.0**-24 + 2.0**-20 + keys * 2.0**-23
    if widened:
        weight += 2 * half_step(dtype)
    tiny = float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    return out.abs() * half_step(dtype) * (1 + 2.0**-10) + mass * weight + spread * 2.0**-25 + tiny


def check_rows(got, q, k, v, scale, widened=False):
    """got, q [H, n, D]; k, v [Hkv, m, D]: each output row against float64."""
    out, mass, top = ref.attention(q, k, v, scale)
    spread = v.double().abs().sum(1, keepdim=True).repeat_interleave(q.shape[0] // v.shape[0], 0)
    bound = channel_bound(out, mass, spread, top, k.shape[1], q.shape[-1], got.dtype, widened)
    off = (got.cpu().double() - out).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), float(off.max()))


def cache_of(k, v, page, layers_seed=0):
    """(cache, table [pages], K, V as stored [Hkv, n, D]) of rows k, v [n, Hkv, D]."""
    n, kv_heads, dim = k.shape
    pages = max(1, -(-n // page))
    cache = new_cache(pages + 2, kv_heads, dim, page, seed=layers_seed)
    table = torch.randperm(pages + 2, generator=torch.Generator().manual_seed(n))[:pages].to(torch.int32).cuda()
    cache.append(0, k.cuda(), v.cuda(), cache.slots(table, 0, n))
    return cache, table, ref.stored(k).transpose(0, 1), ref.stored(v).transpose(0, 1)


def decode(q, cache, table, n, scale, causal=False):
    return kv4.decode_attention(q.cuda(), cache, 0, table[None], torch.tensor([n], dtype=torch.int32, device="cuda"),
                                scale=scale, causal=causal)


# --------------------------------------------------------------------------- query rows of one tile
@pytest.mark.parametrize("dim,group,L", [(64, 8, 1), (128, 4, 4), (256, 8, 1), (128, 8, 4), (256, 5, 5)])
@pytest.mark.parametrize("dtype,loud,quiet", [(BF, 1e30, 1.0), (BF, -(2.0**36), 1.0), (HF, 60000.0, 2.0**-13)])
def test_quiet_queries_beside_a_loud_one(dim, group, L, dtype, loud, quiet):
    """One row of a tile is ``loud`` in a channel that no key has; the others keep their scores of order 1."""
    n = 150
    k, v = rows((n, 1, dim), dtype, 1, 0.2), rows((n, 1, dim), dtype, 2, 0.2)
    k[..., 1] = 0
    q = (rows((1, group, L, dim), dtype, 3, 0.2).double() * quiet).to(dtype)
    q[0, group // 2, L // 2] = 0
    q[0, group // 2, L // 2, 1] = loud
    scale = dim**-0.5 / quiet
    cache, table, ks, vs = cache_of(k, v, 32)
    got = decode(q, cache, table, n, scale)
    for g in range(group):
        for i in range(L):
            check_rows(got[0, g:g + 1, i:i + 1], q[0, g:g + 1, i:i + 1], ks, vs, scale)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dim,heads,L", [(64, 4, 9), (128, 8, 12), (256, 6, 20)])
def test_padding_queries_of_any_size(monkeypatch, in_place, dim, heads, L):
    """What stands in the query rows behind a block's length reaches no real row."""
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    kv4._plans_of.cache_clear()
    state, lengths = 100, [L - 4, 3, 1, 0]
    k, v = rows((state, 1, dim), BF, 1, 0.2), rows((state, 1, dim), BF, 2, 0.2)
    cache, table, ks, vs = cache_of(k, v, 32)
    q = rows((4, heads, L, dim), BF, 3, 0.2)
    kq, vq = rows((4, 1, L, dim), BF, 4, 0.2), rows((4, 1, L, dim), BF, 5, 0.2)
    pads = [1e30, -3e38] + ([math.nan, math.inf] if in_place else [])
    for pad in pads:
        for b, m in enumerate(lengths):
            q[b, :, m:] = pad
        got = kv4.question_attention(q.cuda(), cache, 0, table, state, kq.cuda(), vq.cuda(), lengths, scale=dim**-0.5)
        for b, m in enumerate(lengths):
            assert bool((got[b, :, m:] == 0).all())
            if m:
                check_rows(got[b, :, :m], q[b, :, :m], torch.cat([ks, kq[b, :, :m].double()], 1),
                           torch.cat([vs, vq[b, :, :m].double()], 1), dim**-0.5, True)
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0


# --------------------------------------------------------------------------- V rows of far powers
def far_values(n, kv_heads, dim, dtype, where, power, seed):
    """V rows of order 1 in channels 2 and up, and rows of 2^power in channel 0 (or, below 1, in channel 1) alone."""
    v = rows((n, kv_heads, dim), dtype, seed, 0.2)
    if dtype == HF:
        v = (v.double() * 2.0**-9).to(dtype)
    v[..., :2] = 0
    at = {"first": [0], "middle": [n // 2], "last": [n - 1], "spread": list(range(3, n, 7)), "half": list(range(0, n, 2)),
          "tail": list(range(n // 3, n))}[where]
    v[at] = 0
    v[at, :, 0 if power > 0 else 1] = 2.0**power
    return v


SHAPES = [(64, 8, 1), (64, 4, 4), (128, 8, 1), (128, 4, 4), (256, 8, 1), (128, 8, 4), (256, 5, 5), (256, 3, 4), (64, 16, 2)]


@pytest.mark.parametrize("dim,group,L", SHAPES)
@pytest.mark.parametrize("dtype,power", [(BF, 16), (BF, 25), (BF, 40), (BF, 90), (BF, 126), (BF, -20), (BF, -40), (HF, 15), (HF, -22)])
@pytest.mark.parametrize("where", ["first", "middle", "last", "spread", "half", "tail"])
def test_far_value_rows(dim, group, L, dtype, power, where):
    n = 200
    k, v = rows((n, 2, dim), dtype, 1, 0.2), far_values(n, 2, dim, dtype, where, power, 2)
    cache, table, ks, vs = cache_of(k, v, 16)
    q = rows((1, 2 * group, L, dim), dtype, 3, 0.2)
    got = decode(q, cache, table, n, dim**-0.5)
    check_rows(got[0], q[0], ks, vs, dim**-0.5)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dim,group,L", [(64, 8, 1), (128, 16, 1), (256, 8, 1), (128, 8, 4), (256, 6, 5)])
def test_many_steps_of_mixed_powers(dim, group, L):
    """Powers that wander over 2^60, rows of zeros and masks; long enough for several CTAs a sequence."""
    n = 3000
    k, v = rows((n, 1, dim), BF, 1, 0.2), rows((n, 1, dim), BF, 2, 0.2)
    g = torch.Generator().manual_seed(4)
    for d in range(dim):  # each channel has its own keys of its own power
        keep = torch.rand(n, generator=g) < 0.15
        v[:, 0, d] = torch.where(keep, v[:, 0, d], 0)
    power = torch.randint(-30, 31, (n,), generator=g).double() * (torch.rand(n, generator=g) < 0.3)
    v = (v.double() * 2.0 ** power[:, None, None]).to(BF)
    v[5::11] = 0
    v[:40] = 0
    cache, table, ks, vs = cache_of(k, v, 64)
    q = rows((1, group, L, dim), BF, 3, 0.2)
    got = decode(q, cache, table, n, dim**-0.5, causal=True)
    for i in range(L):
        m = n - (L - 1 - i)
        check_rows(got[0, :, i:i + 1], q[0, :, i:i + 1], ks[:, :m], vs[:, :m], dim**-0.5)
    assert _lib.device_error() == 0


def test_all_value_rows_at_one_end():
    """Nothing but rows of 2^-40, of 2^126, or of zeros and then of 2^100."""
    dim, n = 128, 100
    k, q = rows((n, 1, dim), BF, 1, 0.2), rows((1, 4, 1, dim), BF, 3, 0.2)
    for power in (-40, 120, None):
        v = rows((n, 1, dim), BF, 2, 0.1)
        if power is None:
            v = (v.double() * 2.0**100).to(BF)
            v[:60] = 0
        else:
            v = (v.double() * 2.0**power).to(BF)
        cache, table, ks, vs = cache_of(k, v, 32)
        check_rows(decode(q, cache, table, n, dim**-0.5)[0], q[0], ks, vs, dim**-0.5)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dim,heads,L", [(64, 4, 9), (128, 8, 12), (256, 6, 20)])
@pytest.mark.parametrize("dtype,power", [(BF, 25), (BF, 60), (BF, -40), (HF, 15)])
def test_question_far_value_rows(monkeypatch, in_place, dim, heads, L, dtype, power):
    """Far rows among the state's and among a block's own: the same whichever way the state is read."""
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    kv4._plans_of.cache_clear()
    state, lengths = 150, [L, L - 3, 1]
    k = rows((state, 1, dim), dtype, 1, 0.2)
    q, kq = rows((3, heads, L, dim), dtype, 3, 0.2), rows((3, 1, L, dim), dtype, 4, 0.2)
    for where, own in (("first", "middle"), ("spread", "spread"), (None, "first"), ("last", None)):
        v = far_values(state, 1, dim, dtype, where or "last", power if where else 1, 5)
        vq = torch.stack([far_values(L, 1, dim, dtype, own or "last", power if own else 1, 6 + b).transpose(0, 1) for b in range(3)])
        cache, table, ks, vs = cache_of(k, v, 32)
        got = kv4.question_attention(q.cuda(), cache, 0, table, state, kq.cuda(), vq.cuda(), lengths, scale=dim**-0.5)
        for b, m in enumerate(lengths):
            check_rows(got[b, :, :m], q[b, :, :m], torch.cat([ks, kq[b, :, :m].double()], 1),
                       torch.cat([vs, vq[b, :, :m].double()], 1), dim**-0.5, True)
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0


# --------------------------------------------------------------------------- a block's own rows that are not finite
@pytest.mark.parametrize("dim,heads,L", [(64, 4, 9), (128, 8, 12), (256, 6, 20)])
@pytest.mark.parametrize("dtype,large", [(BF, 1e6), (BF, 1e30), (HF, 6e4)])
def test_own_rows_with_an_infinity(monkeypatch, dim, heads, L, dtype, large):
    """A V row with an infinity in one channel and large numbers in others: the others stay finite."""
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: True)
    kv4._plans_of.cache_clear()
    state, scale = 70, dim**-0.5
    k, v = rows((state, 1, dim), dtype, 1, 0.2), rows((state, 1, dim), dtype, 2, 0.2)
    cache, table, ks, vs = cache_of(k, v, 32)
    q, kq, vq = rows((2, heads, L, dim), dtype, 3, 0.2), rows((2, 1, L, dim), dtype, 4, 0.2), rows((2, 1, L, dim), dtype, 5, 0.2)
    vq[:, 0, 2, 0], vq[:, 0, 2, 5] = math.inf, -large
    got = kv4.question_attention(q.cuda(), cache, 0, table, state, kq.cuda(), vq.cuda(), [L, L], scale=scale)
    assert bool((got[..., 0] == math.inf).all())
    tame = vq.clone()
    tame[:, 0, 2, 0] = 0
    for b in range(2):
        out, mass, top = ref.attention(q[b], torch.cat([ks, kq[b].double()], 1), torch.cat([vs, tame[b].double()], 1), scale)
        spread = torch.cat([vs, tame[b].double()], 1).abs().sum(1, keepdim=True)
        bound = channel_bound(out, mass, spread, top, state + L, dim, dtype, True)
        assert bool(((got[b].cpu().double() - out).abs() <= bound)[..., 1:].all())
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dim,heads,L", [(64, 4, 9), (128, 8, 12), (256, 6, 20)])
@pytest.mark.parametrize("dtype,large", [(BF, 1e6), (BF, 1e30), (HF, 6e4)])
def test_own_key_with_a_score_of_minus_infinity(monkeypatch, in_place, dim, heads, L, dtype, large):
    """A K row of -infinity where every query is positive, with large numbers where every query is zero: no weight."""
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    kv4._plans_of.cache_clear()
    state, scale = 70, dim**-0.5
    k, v = rows((state, 1, dim), dtype, 1, 0.2), rows((state, 1, dim), dtype, 2, 0.2)
    cache, table, ks, vs = cache_of(k, v, 32)
    q, kq, vq = rows((2, heads, L, dim), dtype, 3, 0.2), rows((2, 1, L, dim), dtype, 4, 0.2), rows((2, 1, L, dim), dtype, 5, 0.2)
    q[..., 0], q[..., 5] = q[..., 0].abs() + 1, 0
    kq[:, 0, 4, 0], kq[:, 0, 4, 5] = -math.inf, large
    got = kv4.question_attention(q.cuda(), cache, 0, table, state, kq.cuda(), vq.cuda(), [L, L], scale=scale)
    keep = [i for i in range(L) if i != 4]
    for b in range(2):
        check_rows(got[b], q[b], torch.cat([ks, kq[b][:, keep].double()], 1), torch.cat([vs, vq[b][:, keep].double()], 1), scale, True)
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dim,heads", [(64, 4), (128, 8), (256, 6)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_share_of_nothing_but_minus_infinity(monkeypatch, in_place, dim, heads, dtype):
    """The only own key has a score of -infinity, and its tile is a CTA's whole share: no weight, not NaN."""
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    kv4._plans_of.cache_clear()
    for state in (640, 5000):
        k, v = rows((state, 1, dim), dtype, 1, 0.2), rows((state, 1, dim), dtype, 2, 0.2)
        cache, table, ks, vs = cache_of(k, v, 32)
        q, kq, vq = (rows((1, n, 1, dim), dtype, s, 0.2) for n, s in ((heads, 3), (1, 4), (1, 5)))
        q[..., 0] = q[..., 0].abs() + 1
        kq[..., 0] = -math.inf
        got = kv4.question_attention(q.cuda(), cache, 0, table, state, kq.cuda(), vq.cuda(), [1], scale=dim**-0.5)
        check_rows(got[0], q[0], ks, vs, dim**-0.5, True)
    kv4._plans_of.cache_clear()
    assert _lib.device_error() == 0
