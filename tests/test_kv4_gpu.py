"""The 4-bit key/value cache on the GPU against the float64 oracle: append and read bit for bit,
decode and question attention within bounds derived below, page moves byte for byte."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import ROOT  # noqa: F401  (puts the repository on sys.path)

from d3_turbo_trt_b200 import _lib
from d3_turbo_trt_b200.kernels import kv4
from oracle import kv4 as ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def rows(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype)


def new_cache(pages, kv_heads, dim, page, layers=1, seed=0):
    """A cache whose bytes are whatever an earlier owner left (NaN scales and marks among them)."""
    size = kv4.page_bytes(kv_heads, dim, page)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = torch.randint(0, 256, (layers, pages, size), generator=g, device="cuda", dtype=torch.uint8)
    return kv4.Kv4Cache.over(pool, kv_heads=kv_heads, head_dim=dim, page_tokens=page)


def cells(cache, layer=0):
    """Granules [pages, kv_heads, grains, bytes] of a layer, on the CPU."""
    return cache.pool[layer].cpu().view(cache.pages, cache.kv_heads, cache.page_tokens // 16, -1)


def row_parts(cache, slot, layer=0):
    """(codes, scales, exponent) of K and of V [kv_heads, ...] at a slot."""
    page, at = divmod(slot, cache.page_tokens)
    grain = cells(cache, layer)[page, :, at // 16]
    return tuple((c[:, at % 16], s[:, at % 16], e[:, at % 16]) for c, s, e in ref.parts(grain, cache.head_dim))


# --------------------------------------------------------------------------- append and read
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,kv_heads,page", [(1, 1, 16), (37, 3, 32), (130, 4, 64)])
def test_append_bytes_and_read(dim, dtype, n, kv_heads, page):
    pages = -(-n // page) + 2
    cache = new_cache(pages, kv_heads, dim, page, seed=n)
    before = cells(cache).clone()
    both = rows((n, 2, kv_heads, dim), dtype, seed=dim + n)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(n))[: pages - 2].to(torch.int32).cuda()
    slots = cache.slots(table, 0, n)
    dev = both.cuda()
    cache.append(0, dev[:, 0], dev[:, 1], slots)  # strided views of one projection
    k, v = cache.read(0, table, n, dtype=dtype)
    assert k.shape == (kv_heads, n, dim)
    for got, x in ((k, both[:, 0]), (v, both[:, 1])):
        # code * scale * 2^e has at most 6 significant bits: no rounding in 16 bits
        assert torch.equal(got.cpu().double(), ref.stored(x).transpose(0, 1))
    want = [ref.quantise(both[:, 0]), ref.quantise(both[:, 1])]
    for i in sorted({0, n // 2, n - 1}):
        for (code, scale, exponent), w in zip(row_parts(cache, int(slots[i])), want):
            assert torch.equal(scale, w[1][i]) and torch.equal(exponent, w[2][i])
            # a value that rounds to zero may keep its sign
            same = (code == w[0][i]) | ((code % 8 == 0) & (w[0][i] % 8 == 0))
            assert bool(same.all())
    # every other row of the pool keeps its bytes
    taken = set(slots.tolist())
    after = cells(cache)
    for slot in range(pages * page):
        if slot in taken:
            continue
        g = (slot // page, slice(None), slot % page // 16)
        for x, y in zip(ref.parts(before[g], dim), ref.parts(after[g], dim)):
            assert all(torch.equal(a[:, slot % 16], b[:, slot % 16]) for a, b in zip(x, y))
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_borders_zeros_and_range(dtype):
    """Quotients on the border of two codes, group maxima on the border of two scales, zero rows, the type's
    smallest and largest values, and rows that are not finite."""
    dim, x = 64, []
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for s in (1.0, 1.125, 13.0, 0.015625 * 1.875):
        x.append(torch.cat([borders * s, -borders * s, borders.flip(0) * s, 6 * s * torch.ones(8),
                            448 * 6 * torch.ones(1), torch.zeros(31)]))
    for m in range(8):  # maxima 6 * (1 + (2 m + 1) / 16): half way between two scales
        x.append(torch.cat([6 * (1 + (2 * m + 1) / 16) * torch.ones(16), torch.linspace(-6, 6, 16), torch.zeros(31),
                            2688 * torch.ones(1)]))
    x.append(torch.zeros(dim))
    x.append(-torch.zeros(dim))
    fi = torch.finfo(dtype)
    x.append(torch.full((dim,), fi.tiny))
    x.append(torch.full((dim,), fi.smallest_normal * 2**-3))
    x.append(torch.full((dim,), float(fi.max) / 4))
    x.append(torch.cat([torch.full((1,), float(fi.max) / 2), torch.full((63,), 1.0)]))
    x.append(torch.cat([torch.full((32,), 2.0**-14), torch.full((32,), 1.0)]))
    x.append(torch.full((dim,), 2688.0))
    x.append(torch.full((dim,), 2704.0))
    bad = [torch.tensor([math.nan] + [1.0] * 63), torch.tensor([1.0] * 63 + [math.inf]), torch.full((dim,), -math.inf)]
    x = torch.stack(x + bad).to(dtype)[:, None]
    n = len(x)
    cache = new_cache(4, 1, dim, 32)
    table = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    cache.append(0, x.cuda(), x.flip(-1).cuda(), cache.slots(table, 0, n))
    k, v = cache.read(0, table, n, dtype=dtype)
    assert torch.equal(torch.nan_to_num(k[0].cpu().double(), nan=7e300), torch.nan_to_num(ref.stored(x)[:, 0], nan=7e300))
    assert torch.equal(torch.nan_to_num(v[0].cpu().double(), nan=7e300),
                       torch.nan_to_num(ref.stored(x.flip(-1))[:, 0], nan=7e300))
    assert bool(k[0, n - 3:].isnan().all()) and bool(k[0, :n - 3].isfinite().all())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_every_scale_and_border(dtype):
    """x = border * scale for every significand of a scale and every border of two codes, both signs: products with a
    rounded reciprocal must not fall off the border; and 6 * border of two scales for every border."""
    x = []
    for m in range(8, 16):
        for power in (-10, -3, 0, 5):
            s = m * 2.0**power
            b = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]) * s
            x.append(torch.cat([b, -b, 448 * 6 * 2.0**power * torch.ones(1), torch.zeros(47)]))
    for m in range(16, 32):  # borders have 5 bits
        for power in (-9, -4, 0, 3):
            x.append(torch.cat([torch.full((16,), 6 * m * 2.0**power), torch.full((1,), 2688.0), torch.zeros(47)]))
    x = torch.stack(x).to(dtype)[:, None]
    n = len(x)
    cache = new_cache(8, 1, 64, 16)
    table = torch.tensor([7, 2, 0, 1, 5, 6], dtype=torch.int32, device="cuda")
    cache.append(0, x.cuda(), x.flip(-1).contiguous().cuda(), cache.slots(table, 0, n))
    k, v = cache.read(0, table, n, dtype=dtype)
    # 2688 * 2^5 is infinite in fp16: those rows read back as NaN
    whole = lambda t: torch.nan_to_num(t.cpu().double(), nan=7e300)  # noqa: E731
    assert torch.equal(whole(k[0]), whole(ref.stored(x)[:, 0]))
    assert torch.equal(whole(v[0]), whole(ref.stored(x.flip(-1))[:, 0]))
    assert bool((k[0].isfinite().all(-1).cpu() == x[:, 0].isfinite().all(-1)).all()) and _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [BF, HF])
def test_read_saturates(dtype):
    """A row whose maximum rounds up beyond the type's largest value reads as that value."""
    top = torch.finfo(dtype).max
    x = torch.full((1, 1, 64), top, dtype=dtype, device="cuda")
    cache = new_cache(1, 1, 64, 16)
    table = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(0, x, -x, torch.zeros(1, dtype=torch.int64, device="cuda"))
    k, v = cache.read(0, table, 1, dtype=dtype)
    want = ref.stored(x.cpu()).clamp(-top, top)
    assert torch.equal(k.cpu().double(), want) and torch.equal(v.cpu().double(), -want)


def test_append_left_out_and_bad_slots():
    cache = new_cache(2, 2, 64, 16)
    before = cache.pool.clone()
    x = rows((4, 2, 64), BF, 1).cuda()
    cache.append(0, x, x, torch.tensor([-1, -7, -1, -(2**40)], device="cuda"))
    assert torch.equal(cache.pool, before) and _lib.device_error() == 0
    cache.append(0, x, x, torch.tensor([-1, 32, 2**40, -1], device="cuda"))
    assert torch.equal(cache.pool, before)
    assert _lib.device_error() == kv4.SITE_BAD_SLOT
    assert _lib.device_error() == 0
    cache.append(0, x[:0], x[:0], torch.zeros(0, dtype=torch.int64, device="cuda"))


def test_append_unaligned_and_expanded_rows():
    """Rows that start off 16 bytes, a last dimension that is not contiguous and a broadcast head are copied, not refused."""
    cache = new_cache(2, 2, 64, 16)
    table = torch.tensor([1], dtype=torch.int32, device="cuda")
    flat = rows((5 * 2 * 64 + 3,), BF, 2).cuda()
    k = flat[3:].view(5, 2, 64)
    v = rows((5, 64, 2), BF, 3).cuda().transpose(1, 2)
    cache.append(0, k, v, cache.slots(table, 3, 5))
    kr, vr = cache.read(0, table, 8)
    assert torch.equal(kr[:, 3:].cpu().double(), ref.stored(k.cpu()).transpose(0, 1))
    assert torch.equal(vr[:, 3:].cpu().double(), ref.stored(v.cpu()).transpose(0, 1))
    one = rows((5, 1, 64), BF, 4).cuda().expand(-1, 2, -1)
    cache.append(0, one, one, cache.slots(table, 0, 5))
    kr, _ = cache.read(0, table, 5)
    assert torch.equal(kr[0], kr[1])


def test_read_bad_page_reads_zeros():
    cache = new_cache(3, 1, 64, 16)
    x = rows((48, 1, 64), BF, 5).cuda()
    good = torch.tensor([2, 1, 0], dtype=torch.int32, device="cuda")
    cache.append(0, x, x, cache.slots(good, 0, 48))
    k, _ = cache.read(0, torch.tensor([2, -1, 3], dtype=torch.int32, device="cuda"), 40)
    assert bool((k[:, 16:] == 0).all()) and torch.equal(k[:, :16], cache.read(0, good, 16)[0])
    assert _lib.device_error() == kv4.SITE_BAD_PAGE


# --------------------------------------------------------------------------- decode
def filled(lengths, kv_heads, dim, page, dtype, seed, extra=2, spread=0.5):
    """(cache, table [B, width], K and V as stored [B] of [kv_heads, n, dim] float64)."""
    need = [-(-n // page) for n in lengths]
    width, pages = max(need + [1]), sum(need) + extra
    cache = new_cache(pages, kv_heads, dim, page, seed=seed)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    kept = []
    for b, n in enumerate(lengths):
        mine, order = order[: need[b]], order[need[b]:]
        table[b, : need[b]] = torch.tensor(mine, dtype=torch.int32)
        k, v = rows((n, kv_heads, dim), dtype, seed + 7 * b + 1, spread), rows((n, kv_heads, dim), dtype, seed + 7 * b + 2, spread)
        if n:
            cache.append(0, k.cuda(), v.cuda(), cache.slots(torch.tensor(mine), 0, n))
        kept.append((ref.stored(k).transpose(0, 1), ref.stored(v).transpose(0, 1)))
    return cache, table.cuda(), kept


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def decode_bound(out, mass, top, keys, vmax, dim, dtype):
    """How far a kernel output may be from ``out``.

    * the output's rounding: half a step of it (and of the subnormals' spacing);
    * scores: a product is exact, its fp32 sum of dim terms is off by at most dim * 2^-24 of the sum
      of magnitudes (``top`` bounds that over the keys), two fp32 factors by 2^-23 more; a score off
      by d changes a weight by at most a factor e^(2 d) relative to the others;
    * weights: rounded to fp16, 2^-11 of each, and to 2^-25 of the largest where that is more
      (at most ``keys`` of them); ex2 is off by 2^-22, the sums of ``keys`` terms by keys * 2^-24.
    """
    d = top * (dim + 4) * 2.0**-24
    weight = 2.0**-11 + 2 * d + 2.0**-20 + keys * 2.0**-23
    tiny = float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    return out.abs() * half_step(dtype) * (1 + 2.0**-10) + mass * weight + keys * 2.0**-25 * vmax + tiny


def check_decode(q, cache, table, lengths, kept, scale, causal, dtype, out=None):
    rows_, heads, L, dim = q.shape
    got = kv4.decode_attention(q.cuda() if not q.is_cuda else q, cache, 0, table,
                               torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale=scale, causal=causal, out=out)
    assert got.shape == q.shape and got.dtype == dtype
    host, qc = got.cpu().double(), q.cpu()
    for b in range(rows_):
        k, v = kept[b]
        for i in range(L):
            n = max(0, lengths[b] - (L - 1 - i)) if causal else lengths[b]
            out_, mass, top = ref.attention(qc[b, :, i:i + 1], k[:, :n], v[:, :n], scale)
            vmax = float(v[:, :n].abs().max()) if n else 0.0
            bound = decode_bound(out_, mass, top, n, vmax, dim, dtype)
            off = (host[b, :, i:i + 1] - out_).abs()
            assert bool((off <= bound).all()), (b, i, n, float((off - bound).max()), float(off.max()))
    assert _lib.device_error() == 0
    return got


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,group,L,page", [(1, 1, 1, 16), (2, 4, 1, 32), (2, 6, 1, 64), (1, 8, 1, 128), (1, 7, 3, 16),
                                                   (2, 16, 1, 256), (1, 5, 7, 64), (3, 2, 2, 16), (1, 33, 1, 32)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode(dim, kv_heads, group, L, page, dtype):
    lengths = [1, 0, 15, 16, 17, 33, 129, 300]
    cache, table, kept = filled(lengths, kv_heads, dim, page, dtype, seed=dim + group)
    q = rows((len(lengths), kv_heads * group, L, dim), dtype, seed=3)
    for causal in (False, True):
        got = check_decode(q, cache, table, lengths, kept, dim**-0.5, causal, dtype)
        assert bool((got[1] == 0).all())  # no keys: zero rows
        if causal and L > 1:
            assert bool((got[0, :, : L - 1] == 0).all())  # tokens before the sequence


@pytest.mark.parametrize("dim,B,heads,kv_heads,length", [(128, 1, 8, 1, 5000), (256, 2, 6, 1, 2049), (64, 3, 8, 4, 3583),
                                                         (128, 70, 8, 8, 65)])
def test_decode_long_and_wide(dim, B, heads, kv_heads, length):
    lengths = [length - 13 * b for b in range(B)] if length > 100 else [1 + (7 * b) % length for b in range(B)]
    cache, table, kept = filled(lengths, kv_heads, dim, 64, BF, seed=length)
    check_decode(rows((B, heads, 1, dim), BF, seed=9), cache, table, lengths, kept, dim**-0.5, False, BF)


def test_decode_sharp_scores_and_far_values():
    """Scores that leave one key, and V rows whose powers differ by 2^40: the far row must not take the others' weights."""
    dim, n = 128, 200
    cache, table, kept = filled([n], 2, dim, 32, BF, seed=5)
    check_decode(rows((1, 8, 1, dim), BF, seed=1) * 30, cache, table, [n], kept, 1.0, False, BF)
    k, v = rows((n, 2, dim), BF, 11), rows((n, 2, dim), BF, 12)
    v[::7] *= 2.0**30
    v[3::7] *= 2.0**-20
    v[5::14] = 0
    k[::7] = -8 * k[::7].abs()  # a positive query gives the far rows weights near 2^-40
    cache.append(0, k.cuda(), v.cuda(), cache.slots(table[0], 0, n))
    kept = [(ref.stored(k).transpose(0, 1), ref.stored(v).transpose(0, 1))]
    q = rows((1, 8, 1, dim), BF, seed=2).abs() * 0.2
    check_decode(q, cache, table, [n], kept, 0.1, False, BF)


def test_decode_queries_beyond_fp16():
    """bf16 queries of 1e30 and 1e-30: brought under a power of two a row, not into fp16's range as they are."""
    dim, n = 64, 50
    cache, table, kept = filled([n, n], 1, dim, 16, BF, seed=6)
    q = rows((2, 4, 1, dim), BF, seed=3)
    q = (q.double() * torch.tensor([1e30, 1e-30], dtype=torch.float64).view(2, 1, 1, 1)).to(BF)
    got = check_decode(q[:1], cache, table[:1], [n], kept[:1], 1e-30, False, BF)
    assert bool(got.isfinite().all())
    check_decode(q[1:], cache, table[1:], [n], kept[1:], 1e28, False, BF)


def test_decode_strides_out_and_single():
    dim, lengths = 128, [70, 3]
    cache, table, kept = filled(lengths, 2, dim, 16, BF, seed=8)
    q = rows((2, 3, 8, dim), BF, seed=4).transpose(1, 2)  # token-major
    out = torch.full((2, 3, 8, dim + 8), 7.0, dtype=BF, device="cuda")
    view = out[..., :dim].transpose(1, 2)
    check_decode(q.cuda(), cache, table, lengths, kept, 0.09, True, BF, out=view)
    assert bool((out[..., dim:] == 7).all())
    one = kv4.decode_attention(q[:, :, 0].cuda(), cache, 0, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale=0.09)
    assert one.shape == (2, 8, dim)
    # a table as a slice of a wider one, and rows of the table in another order of pages
    wide = torch.full((2, 40), -5, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    again = kv4.decode_attention(q[:, :, 0].cuda(), cache, 0, wide[:, 2:], torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale=0.09)
    assert torch.allclose(one.float(), again.float(), atol=0.02, rtol=0.02)


def test_attention_refuses_shared_output_rows_and_scales():
    cache, table, _ = filled([20, 9], 1, 64, 16, BF, seed=3)
    lens = torch.tensor([20, 9], dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 2, 1, 64, dtype=BF, device="cuda")
    k = torch.zeros(2, 1, 1, 64, dtype=BF, device="cuda")
    one = torch.zeros(1, 2, 1, 64, dtype=BF, device="cuda")
    for kw in (dict(out=one.expand(2, 2, 1, 64)), dict(out=one[:, :1].expand(2, 2, 1, 64)), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(scale=0.0)):
        kw = dict(scale=0.1) | kw
        with pytest.raises(RuntimeError):
            kv4.decode_attention(q, cache, 0, table, lens, **kw)
        with pytest.raises(RuntimeError):
            kv4.question_attention(q, cache, 0, table[0], 20, k, k, [1, 1], **kw)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("L", [1, 18])  # both kernels
def test_decode_many_short_sequences(L):
    # 40000 sequences of 0 to 2 granules over 2 pages: thousands to a CTA, most of them without keys
    dim, B = 64, 40000
    cache, table, kept = filled([16, 16], 1, dim, 16, BF, seed=5)
    pages = torch.tensor([int(table[0, 0]), int(table[1, 0])], dtype=torch.int32, device="cuda")
    lens = (torch.arange(B, dtype=torch.int32, device="cuda") * 7919 % 131 - 98).clamp_(0, 32)
    q = rows((1, L, 1, dim), BF, 6).transpose(1, 2)
    out = kv4.decode_attention(q.cuda().expand(B, 1, L, dim), cache, 0, pages[None].expand(B, 2), lens, scale=0.1)
    both = [torch.cat([kept[0][i], kept[1][i]], 1) for i in range(2)]
    for n in range(33):
        got = out[lens == n].cpu().double()
        assert got.shape[0] > 100
        if n == 0:
            assert bool((got == 0).all())
            continue
        want, mass, top = ref.attention(q[0], both[0][:, :n], both[1][:, :n], 0.1)
        bound = decode_bound(want, mass, top, n, float(both[1].abs().max()), dim, BF)
        assert bool(((got - want).abs() <= bound).all()), n
    assert _lib.device_error() == 0


def test_decode_not_finite_rows_reach_only_their_readers():
    dim, n = 128, 40
    cache, table, kept = filled([n, n], 1, dim, 16, BF, seed=10)
    x = rows((1, 1, dim), BF, 1).cuda()
    bad = x.clone()
    bad[0, 0, 5] = math.nan
    lengths = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    q = rows((2, 4, 2, dim), BF, seed=5).cuda()
    clean = kv4.decode_attention(q, cache, 0, table, lengths, scale=0.1, causal=True)
    cache.append(0, x, bad, cache.slots(table[0], n - 1, 1))  # V of sequence 0's last token
    got = kv4.decode_attention(q, cache, 0, table, lengths, scale=0.1, causal=True)
    assert bool(got[0, :, 1].isnan().all())
    assert torch.equal(got[0, :, 0], clean[0, :, 0]) and torch.equal(got[1], clean[1])
    cache.append(0, bad, x, cache.slots(table[0], n - 1, 1))
    got = kv4.decode_attention(q, cache, 0, table, lengths, scale=0.1, causal=True)
    assert bool(got[0, :, 1].isnan().all()) and torch.equal(got[0, :, 0], clean[0, :, 0])


def test_decode_bad_pages_and_lengths():
    dim = 64
    cache, table, kept = filled([48, 48], 1, dim, 16, BF, seed=12)
    q = rows((2, 2, 1, dim), BF, seed=6)
    lengths = torch.tensor([48, 48], dtype=torch.int32, device="cuda")
    broken = table.clone()
    broken[0, 1] = cache.pages
    broken[1, 2] = -3
    got = kv4.decode_attention(q.cuda(), cache, 0, broken, lengths, scale=0.1).cpu().double()
    assert _lib.device_error() == kv4.SITE_BAD_PAGE
    for b, keep in ((0, list(range(16)) + list(range(32, 48))), (1, list(range(32)))):
        out, mass, top = ref.attention(q[b], kept[b][0][:, keep], kept[b][1][:, keep], 0.1)
        bound = decode_bound(out, mass, top, 48, float(kept[b][1].abs().max()), dim, BF)
        assert bool(((got[b] - out).abs() <= bound).all())
    got = kv4.decode_attention(q.cuda(), cache, 0, table, torch.tensor([49, -1], dtype=torch.int32, device="cuda"), scale=0.1)
    assert _lib.device_error() == kv4.SITE_BAD_LENGTH
    whole = kv4.decode_attention(q.cuda(), cache, 0, table, lengths, scale=0.1)
    assert torch.equal(got[0], whole[0]) and bool((got[1] == 0).all())


def test_decode_repeats_bit_for_bit_streams_and_graph():
    dim, lengths = 128, [700, 90, 1, 333]
    cache, table, kept = filled(lengths, 2, dim, 32, BF, seed=14)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = rows((4, 12, 1, dim), BF, seed=7).cuda()
    first = kv4.decode_attention(q, cache, 0, table, lens, scale=0.1)
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in side * 3:
        with torch.cuda.stream(s):
            outs.append(kv4.decode_attention(q, cache, 0, table, lens, scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in outs)
    # two graphs captured on one stream, replayed on two, lengths and queries changed in between
    graphs, held = [], []
    cap = torch.cuda.Stream()
    for i in range(2):
        qs = q.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            out = kv4.decode_attention(qs, cache, 0, table, lens, scale=0.1)
        graphs.append(g)
        held.append((qs, out))
    held[1][0].copy_(-q)
    lens.copy_(torch.tensor([600, 90, 0, 320], dtype=torch.int32))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for qs, out in held:
        assert torch.equal(out, kv4.decode_attention(qs, cache, 0, table, lens, scale=0.1))


def test_decode_pool_beyond_4_gib():
    """Byte offsets past 32 bits: the pages in use are the pool's last."""
    dim, page, kv_heads = 128, 64, 8
    size = kv4.page_bytes(kv_heads, dim, page)
    pages = 5 * 2**30 // (2 * size)
    cache = kv4.Kv4Cache(2, pages, kv_heads=kv_heads, head_dim=dim, page_tokens=page)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    n = 100
    k, v = rows((n, kv_heads, dim), BF, 1), rows((n, kv_heads, dim), BF, 2)
    cache.append(1, k.cuda(), v.cuda(), cache.slots(table[0], 0, n))
    kr, vr = cache.read(1, table[0], n)
    assert torch.equal(kr.cpu().double(), ref.stored(k).transpose(0, 1))
    q = rows((1, kv_heads, 1, dim), BF, 3)
    got = kv4.decode_attention(q.cuda(), cache, 1, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=0.1)
    out, mass, top = ref.attention(q[0], kr.cpu(), vr.cpu(), 0.1)
    assert bool(((got[0].cpu().double() - out).abs() <= decode_bound(out, mass, top, n, float(vr.abs().max()), dim, BF)).all())
    cache.copy_pages([pages - 1], [pages - 2])
    assert torch.equal(cache.pool[1, pages - 1], cache.pool[1, pages - 2])



@pytest.mark.parametrize("dim,group,L", [(64, 8, 1), (128, 5, 3), (256, 6, 1), (256, 6, 5), (64, 3, 11)])
@pytest.mark.parametrize("lengths", [[5000, 0, 17, 3100, 1], [2900], [700] * 32, [64, 4096, 4095, 4097], [900, 0, 31, 350] * 10])
def test_decode_shares_of_ragged_sequences(dim, group, L, lengths):
    """Shares of several tiles: units that begin with a CTA, filled up at their ends, and those that do not."""
    cache, table, kept = filled(lengths, 2, dim, 64, BF, seed=group)
    q = rows((len(lengths), 2 * group, L, dim), BF, seed=L)
    check_decode(q, cache, table, lengths, kept, dim**-0.5, True, BF)


# --------------------------------------------------------------------------- question attention
@pytest.mark.parametrize("lengths", [[40, 3, 0, 17], [0, 0, 40], [1] * 9, [40, 1, 0, 17] * 9])
def test_question_shares_with_tiles_of_padding(monkeypatch, lengths):
    # in place, with shares of several tiles and whole tiles of rows behind their block's length
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: True)
    state, L, dim = 2100, 40, 64
    cache, table, kept = filled([state], 2, dim, 32, BF, seed=3)
    cache._plans.clear()
    q = rows((len(lengths), L, 16, dim), BF, 1, 0.2).transpose(1, 2)
    k, v = (rows((len(lengths), 2, L, dim), BF, s, 0.2) for s in (2, 3))
    out = torch.full((len(lengths), 16, L, dim), 3.0, dtype=BF, device="cuda")
    got = kv4.question_attention(q.cuda(), cache, 0, table[0], state, k.cuda(), v.cuda(), lengths, scale=dim**-0.5, out=out)
    check_question(got, q, kept[0], k, v, lengths, dim**-0.5, BF)
    cache._plans.clear()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dim,heads,kv_heads,page", [(64, 8, 2, 16), (128, 8, 1, 64), (256, 6, 1, 32)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,L,state", [(1, 1, 1), (2, 11, 77), (5, 20, 300), (3, 7, 0)])
def test_question(dim, heads, kv_heads, page, dtype, B, L, state):
    cache, table, kept = filled([state], kv_heads, dim, page, dtype, seed=state + 1)
    q = rows((B, L, heads, dim), dtype, 1, 0.2).transpose(1, 2)
    k, v = (rows((B, kv_heads, L, dim), dtype, s, 0.2) for s in (2, 3))
    lengths = [(L - 3 * b) % (L + 1) for b in range(B)]
    got = kv4.question_attention(q.cuda(), cache, 0, table[0], state, k.cuda(), v.cuda(), lengths, scale=dim**-0.5)
    check_question(got, q, kept[0], k, v, lengths, dim**-0.5, dtype)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dim,heads,kv_heads,B,L,state", [(64, 12, 3, 4, 70, 200), (128, 32, 4, 2, 33, 1000), (128, 7, 1, 9, 1, 129),
                                                          (256, 24, 4, 3, 8, 640), (256, 2, 2, 40, 5, 63)])
def test_question_both_ways(monkeypatch, in_place, dim, heads, kv_heads, B, L, state):
    """Either way of reading the state, whatever the sizes would choose: lengths on the device, strided operands,
    keys of the block behind several tiles of the state, and an output of another layout."""
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    cache, table, kept = filled([state], kv_heads, dim, 32, BF, seed=L)
    cache._plans.clear()
    q = rows((B, L, heads, dim), BF, 1, 0.2).transpose(1, 2)
    both = rows((B, L, 2, kv_heads, dim), BF, 2, 0.2)
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    dev = both.cuda()
    lengths = [(L + 5 * b) % (L + 1) for b in range(B)]
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = torch.full((B, L, heads, dim), 3.0, dtype=BF, device="cuda").transpose(1, 2)
    got = kv4.question_attention(q.cuda(), cache, 0, table[0], state, dev[:, :, 0].transpose(1, 2), dev[:, :, 1].transpose(1, 2),
                                 lens, scale=dim**-0.5, out=out)
    assert got is out
    check_question(got, q, kept[0], k, v, lengths, dim**-0.5, BF)
    assert _lib.device_error() == 0
    lens[0] = L + 1  # clamped to L and recorded; the widened form's waits stop early then, and its results are void
    again = kv4.question_attention(q.cuda(), cache, 0, table[0], state, dev[:, :, 0].transpose(1, 2), dev[:, :, 1].transpose(1, 2),
                                   lens, scale=dim**-0.5)
    if in_place:
        check_question(again, q, kept[0], k, v, [L] + lengths[1:], dim**-0.5, BF)
    assert _lib.device_error() == 2010
    cache._plans.clear()


def test_question_refuses():
    cache = new_cache(4, 2, 64, 16)
    table = torch.arange(4, dtype=torch.int32, device="cuda")
    q, k = torch.zeros(2, 4, 3, 64, dtype=BF, device="cuda"), torch.zeros(2, 2, 3, 64, dtype=BF, device="cuda")
    ask = lambda **kw: kv4.question_attention(**(dict(q=q, cache=cache, layer=0, table=table, state_len=60, k_q=k, v_q=k,  # noqa: E731
                                                      lengths=[3, 2], scale=0.1) | kw))
    ask()
    for kw in (dict(state_len=65), dict(state_len=-1), dict(layer=1), dict(lengths=[3]), dict(lengths=[4, 0]), dict(lengths=[-1, 0]),
               dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(k_q=k.half()), dict(v_q=k[:, :1]), dict(table=table.long()),
               dict(table=table.cpu()), dict(table=table[None]), dict(out=q.float()), dict(q=q.cpu()), dict(scale=0.0)):
        with pytest.raises(RuntimeError):
            ask(**kw)
    deq = lambda **kw: kv4.decode_attention(**(dict(q=q, cache=cache, layer=0, table=table.view(2, 2),  # noqa: E731
                                                    lengths=table[:2], scale=0.1) | kw))
    deq()
    for kw in (dict(table=table), dict(table=table.view(1, 4)), dict(lengths=table[:1]), dict(lengths=table[:2].long()), dict(layer=-1),
               dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[..., :32]), dict(scale=-1.0), dict(out=q[:1]), dict(q=q[0, 0])):
        with pytest.raises(RuntimeError):
            deq(**kw)
    app = lambda **kw: cache.append(**(dict(layer=0, k=k[:, :, 0], v=k[:, :, 0], slots=torch.zeros(2, dtype=torch.int64, device="cuda") - 1) | kw))  # noqa: E731
    app()
    for kw in (dict(layer=2), dict(k=k[:1, :, 0]), dict(v=k[:, :, 0].half()), dict(slots=torch.zeros(2, dtype=torch.int32, device="cuda")),
               dict(slots=torch.zeros(3, dtype=torch.int64, device="cuda")), dict(k=k[:, :, 0].cpu())):
        with pytest.raises(RuntimeError):
            app(**kw)
    for bad in (lambda: cache.read(0, table, 65), lambda: cache.read(0, table.long(), 5), lambda: cache.read(0, table, 5, dtype=torch.float32),
                lambda: cache.copy_pages([0, 1], [1, 2]), lambda: cache.copy_pages([0, 1], [2, 2]), lambda: cache.copy_pages([0], [4]),
                lambda: cache.copy_pages([0], [2, 3]), lambda: cache.move_pages([1, 0], [2, 3], table), lambda: cache.move_pages([0], [2], table.long()),
                lambda: cache.slots([0, 1], 30, 3), lambda: kv4.Kv4Cache.over(cache.pool[:, :, 16:], kv_heads=2, head_dim=64, page_tokens=16)):
        with pytest.raises(RuntimeError):
            bad()
    assert _lib.device_error() == 0


def check_question(got, q, state, k, v, lengths, scale, dtype):
    got, dim = got.cpu().double(), q.shape[-1]
    for b, n in enumerate(lengths):
        assert bool((got[b, :, n:] == 0).all())
        if n == 0:
            continue
        keys = torch.cat([state[0], k[b, :, :n].double()], 1)
        values = torch.cat([state[1], v[b, :, :n].double()], 1)
        out, mass, top = ref.attention(q[b, :, :n], keys, values, scale)
        # weights are rounded to the inputs' type here: half a step of each, twice (unnormalised and scaled)
        bound = decode_bound(out, mass, top, keys.shape[1], float(values.abs().max()), dim, dtype) + mass * 2 * half_step(dtype)
        off = (got[b, :, :n] - out).abs()
        assert bool((off <= bound).all()), (b, n, float((off - bound).max()))


# --------------------------------------------------------------------------- pages
@pytest.mark.parametrize("dim,kv_heads,page,layers", [(64, 1, 16, 1), (128, 3, 32, 3), (256, 4, 128, 2)])
def test_copy_and_move_pages(dim, kv_heads, page, layers):
    cache = new_cache(40, kv_heads, dim, page, layers=layers, seed=dim)
    src, dst = [3, 8, 9, 21, 39], [1, 30, 2, 0, 5]
    want = cache.pool.clone()
    want[:, dst] = want[:, src]
    cache.copy_pages(src, dst)
    assert torch.equal(cache.pool, want)
    tables = torch.tensor([[3, 8, 7, -1], [39, 9, 9, 21], [1, 38, 2, 100]], dtype=torch.int32, device="cuda")
    cache.move_pages(torch.tensor(src, dtype=torch.int32, device="cuda"), torch.tensor(dst, dtype=torch.int32, device="cuda"), tables)
    assert torch.equal(cache.pool, want)
    assert tables.tolist() == [[1, 30, 7, -1], [5, 2, 2, 0], [1, 38, 2, 100]]
    assert _lib.device_error() == 0
    cache.copy_pages([], [])


def test_move_pages_records_bad_lists():
    cache = new_cache(10, 1, 64, 16, seed=1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    tables = i32([[0, 1]])
    cache.move_pages(i32([4, 2]), i32([7, 8]), tables)
    assert _lib.device_error() == kv4.SITE_BAD_MOVE
    before = cache.pool.clone()
    cache.copy_pages(i32([4, 10, -1]), i32([12, 1, 2]))
    assert torch.equal(cache.pool, before) and _lib.device_error() == kv4.SITE_BAD_PAGE
