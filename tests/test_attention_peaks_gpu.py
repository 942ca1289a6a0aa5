"""Prefix-bidirectional attention with scores that spread over tens of powers of two, so that the running
maximum moves again and again behind the first key tiles: every launch form against float64.

Bound: the output's rounding is half a step, a weight is rounded to the inputs' type (half a step of it) and
the exponential is off by at most 2^-10; a score's fp32 sum of D products is off by D * 2^-24 of the sum of
magnitudes, which changes a weight by twice that."""

from __future__ import annotations

import pytest
import torch

from conftest import ROOT  # noqa: F401

from d3_turbo_trt_b200 import _lib
from d3_turbo_trt_b200.kernels import prefix_bidir as pb

pytestmark = pytest.mark.gpu


def spread_rows(g, *shape, spread=0.5):
    x = torch.randn(shape, generator=g, device="cuda")
    return x * torch.exp(spread * torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))


def check(B, H, Hkv, L, S, D, dtype, loud, lengths=None, repeats=3):
    g = torch.Generator(device="cuda").manual_seed(D + S + L)
    q = (loud * spread_rows(g, B, H, L, D)).to(dtype)
    ks, vs = spread_rows(g, Hkv, S, D).to(dtype), torch.randn(Hkv, S, D, generator=g, device="cuda").to(dtype)
    k, v = spread_rows(g, B, Hkv, L, D).to(dtype), torch.randn(B, Hkv, L, D, generator=g, device="cuda").to(dtype)
    lengths = lengths or [L] * B
    scale, half = D**-0.5, torch.finfo(dtype).eps / 2
    blocks = sorted({0, B // 2, B - 1})
    want = {}
    for b in blocks:
        n = lengths[b]
        kk = torch.cat([ks, k[b, :, :n]], 1).double().repeat_interleave(H // Hkv, 0)
        vv = torch.cat([vs, v[b, :, :n]], 1).double().repeat_interleave(H // Hkv, 0)
        qq = q[b, :, :n].double()
        p = torch.softmax(qq @ kk.transpose(1, 2) * scale, -1)
        top = (qq.abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True) * scale
        out, mass = p @ vv, p @ vv.abs()
        want[b] = out, out.abs() * half + mass * (half + 2.0**-10 + 2 * top * (D + 4) * 2.0**-24) + 1e-6
    for _ in range(repeats):
        got = pb.prefix_bidir_attention(q, ks, vs, k, v, lengths, scale=scale)
        for b, (out, bound) in want.items():
            off = (got[b, :, : lengths[b]].double() - out).abs()
            assert bool((off <= bound).all()), (b, float((off - bound).max()), int((off > bound).sum()))
    assert _lib.device_error() == 0


# one unit a CTA, several a CTA, units cut into pieces, CTA pairs (long launches at D = 128), and D = 256's tiles
@pytest.mark.parametrize("B,H,Hkv,L,S,D", [(2, 32, 4, 33, 1000, 128), (16, 32, 4, 64, 4096, 128), (40, 32, 4, 48, 2048, 128),
                                           (1, 32, 4, 64, 16384, 128), (4, 24, 4, 37, 3001, 256), (20, 24, 4, 64, 1024, 256),
                                           (4, 8, 2, 32, 512, 64), (6, 8, 2, 20, 700, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("loud", [1.0, 4.0])
def test_moving_maximum(B, H, Hkv, L, S, D, dtype, loud):
    check(B, H, Hkv, L, S, D, dtype, loud, lengths=[1 + (7 * b + L - 1) % L for b in range(B)])


def test_maximum_moves_in_every_tile():
    """Keys that grow along the state: each tile's maximum passes the last one's by more than the threshold."""
    B, H, Hkv, L, S, D = 8, 32, 4, 32, 4096, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.rand(B, H, L, D, generator=g, device="cuda").bfloat16()
    ks = (torch.rand(Hkv, S, D, generator=g, device="cuda") * torch.linspace(0.1, 40, S, device="cuda")[None, :, None]).bfloat16()
    vs = torch.randn(Hkv, S, D, generator=g, device="cuda").bfloat16()
    k, v = torch.zeros(B, Hkv, L, D, device="cuda").bfloat16(), torch.zeros(B, Hkv, L, D, device="cuda").bfloat16()
    out = pb.prefix_bidir_attention(q, ks, vs, k, v, [L] * B, scale=D**-0.5).double()
    kk, vv = ks.double().repeat_interleave(8, 0), vs.double().repeat_interleave(8, 0)
    for b in range(B):
        scores = q[b].double() @ kk.transpose(1, 2) * D**-0.5
        p = torch.softmax(torch.cat([scores, torch.zeros(H, L, L, dtype=torch.float64, device="cuda")], -1), -1)[..., :S]
        want, mass = p @ vv, p @ vv.abs()
        bound = want.abs() * 2.0**-8 + mass * (2.0**-8 + 2.0**-10 + 2 * scores.abs().amax(-1, keepdim=True) * (D + 4) * 2.0**-24) + 1e-6
        assert bool(((out[b] - want).abs() <= bound).all())
    assert _lib.device_error() == 0
