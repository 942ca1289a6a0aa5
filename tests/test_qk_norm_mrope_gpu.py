"""Query/key norm with multi-axis rotation against the float64 oracle."""

from __future__ import annotations

import pytest
import torch

from conftest import ROOT  # noqa: F401

from d3_turbo_trt_b200.model import fused
from oracle import kv4 as ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def bound(want, x, half, dtype):
    """The output's rounding is half a step. Before it, in fp32: the mean of D squares (D * 2^-24 at
    most), rsqrt (2^-22), three products and the weight's sum (2^-24 each), cos and sin (2^-22), the
    angle brought into one turn in fp64 and rounded to fp32 (2^-24 of pi), a product and a sum. That
    is below 2^-15 of the larger of a pair's two magnitudes."""
    size = want.abs().clone()
    pair = torch.sqrt(want[..., :half] ** 2 + want[..., half:2 * half] ** 2)
    size[..., :half], size[..., half:2 * half] = pair, pair
    tiny = float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    return want.abs() * torch.finfo(dtype).eps / 2 + size * 2.0**-15 + tiny


def check(rows, T, heads, kv_heads, dim, sections, dtype, far, interleaved=False, wide=False):
    g = torch.Generator().manual_seed(rows * 1000 + T)
    q = torch.randn(rows, T, heads, 2 * dim if wide else dim, generator=g).to(dtype)[..., :dim]
    k = (3 * torch.randn(rows, T, kv_heads, dim, generator=g)).to(dtype)
    wq, wk = ((0.2 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2))
    half = sum(sections)
    axes = fused.rotary_axes(sections, interleaved=interleaved)
    freq = (1e7 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float()
    pos = torch.randint(0, far, (len(sections), rows, T), generator=g)
    pos[:, 0, 0] = torch.tensor([0, far, 1])[: len(sections)]
    qd = torch.empty(rows, T, heads, 2 * dim if wide else dim, dtype=dtype, device="cuda")[..., :dim].copy_(q)
    got = fused.qk_norm_mrope(qd, k.cuda(), wq.cuda(), wk.cuda(), pos.cuda(), freq.cuda(), axes, 1e-6)
    for out, x, w in zip(got, (q, k), (wq, wk)):
        want = ref.norm_mrope(x, w, pos, freq, axes, 1e-6)
        assert out.dtype == dtype and out.shape == x.shape
        off = (out.cpu().double() - want).abs()
        lim = bound(want, x, half, dtype)
        assert bool((off <= lim).all()), float((off - lim).max())


@pytest.mark.parametrize("dim,sections", [(64, [8]), (64, [11, 11, 10]), (128, [6, 5, 5]), (128, [30, 34]), (256, [11, 11, 10]),
                                          (256, [43, 43, 42]), (256, [8, 8, 8])])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,T,heads,kv_heads", [(1, 1, 24, 4), (3, 7, 5, 1), (2, 1, 1, 1)])
def test_norm_mrope(dim, sections, dtype, rows, T, heads, kv_heads):
    check(rows, T, heads, kv_heads, dim, sections, dtype, 5000, wide=heads == 24)


@pytest.mark.parametrize("far", [10, 10**6, 2**40])
def test_far_positions(far):
    """The angle is a product in fp64: off by 2^-53 of it. At 2^40 that is 2^-13 rad, so freq 1 alone is left out there."""
    if far < 2**40:
        check(2, 5, 4, 2, 128, [6, 5, 5], BF, far)
    else:
        # frequency 1 and whole positions: the product is exact, fp64's 2 pi reduction costs 2^-53 * 2^40 / (2 pi)
        q = torch.randn(1, 1, 1, 64).to(BF)
        pos = torch.full((1, 1, 1), far)
        freq = torch.ones(8)
        got, _ = fused.qk_norm_mrope(q.cuda(), q.cuda(), torch.zeros(64, dtype=BF, device="cuda"),
                                     torch.zeros(64, dtype=BF, device="cuda"), pos.cuda(), freq.cuda(), [0] * 8, 1e-6)
        want = ref.norm_mrope(q, torch.zeros(64), pos, freq, [0] * 8, 1e-6)
        pair = torch.sqrt(want[..., :8] ** 2 + want[..., 8:16] ** 2).repeat(1, 1, 1, 2)
        off = (got.cpu().double() - want).abs()[..., :16]
        assert bool((off <= bound(want, q, 8, BF)[..., :16] + pair * 2.0**-11).all())


def test_many_heads_and_interleaved():
    check(1, 3, 70, 10, 256, [11, 11, 10], BF, 100, interleaved=True)  # more rows than a CTA's threads hold at once
    check(2, 2, 8, 8, 64, [12, 10, 10], HF, 100, interleaved=True)


def test_text_positions_agree_with_the_single_axis_form():
    """Equal positions on three axes are the framework's text rotation: ``qk_norm_rope`` rounds to bf16
    after the norm (2^-8 of a value), after cos and sin (2^-8), each product and the sum."""
    from d3_turbo_trt_b200.model.backbone import BackboneConfig, rotary_tables

    c = BackboneConfig()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 9, 4, 128, generator=g).to(BF).cuda()
    w = (0.1 * torch.randn(128, generator=g)).to(BF).cuda()
    pos = torch.arange(9, device="cuda")[None].expand(2, -1)
    cos, sin = rotary_tables(c, pos, BF)
    half = cos.shape[-1] // 2
    freq = 1.0 / (c.rope_theta ** (torch.arange(0, 2 * half, 2, device="cuda").float() / (2 * half)))
    old = fused.qk_norm_rope(x, w, cos, sin, 1e-6).double()
    new, _ = fused.qk_norm_mrope(x, x, w, w, pos[None].expand(3, -1, -1), freq, fused.rotary_axes([6, 5, 5]), 1e-6)
    new = new.double()
    pair = torch.sqrt(new[..., :half] ** 2 + new[..., half:2 * half] ** 2)
    size = new.abs()
    size[..., :half] = size[..., half:2 * half] = pair
    # per path: norm, cos/sin, products, sum (two terms of at most the pair's size): 6 half steps of the pair, and new's own
    assert bool(((old - new).abs() <= size * 7 * 2.0**-8).all())


def test_empty():
    z = torch.zeros(0, 3, 2, 64, dtype=BF, device="cuda")
    w = torch.zeros(64, dtype=BF, device="cuda")
    pos = torch.zeros(1, 0, 3, dtype=torch.int64, device="cuda")
    a, b = fused.qk_norm_mrope(z, z, w, w, pos, torch.ones(8, device="cuda"), [0] * 8, 1e-6)
    assert a.shape == z.shape and b.shape == z.shape
