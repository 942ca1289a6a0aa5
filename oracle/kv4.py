"""The 4-bit key/value cache and the multi-axis query/key rotation in float64 (CPU oracle).

Written from the definitions: a row of a granule is brought under a power of two, 16 channels
share an e4m3 scale and every channel takes the nearest e2m1 code. The quantisation works on
numbers (nearest value of a list, ties to the even code), not on bit patterns.
"""

from __future__ import annotations

import math

import torch

E_MIN = -64
CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# every finite e4m3 value from 0 up; index = byte
E4M3 = [m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127]


def _nearest(x: torch.Tensor, values: list[float]) -> torch.Tensor:
    """Index of the nearest of ascending ``values``; of two equally near the even index."""
    v = torch.tensor(values, dtype=torch.float64)
    hi = torch.searchsorted(v, x.contiguous()).clamp(1, len(values) - 1)
    lo = hi - 1
    below, above = x - v[lo], v[hi] - x
    take_hi = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(take_hi, hi, lo)


def quantise(x: torch.Tensor):
    """(codes 0..15 [..., D], scale bytes [..., D/16], exponent bytes [...]) of rows x [..., D]."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], 0.0, x)
    top = x.abs().amax(-1)
    e = torch.full(top.shape, E_MIN)
    for power in range(E_MIN, 118):  # the least power that holds the row
        e = torch.where(top > 2688 * 2.0**power, power + 1, e)
    y = (x * 2.0 ** (-e.double())[..., None]).unflatten(-1, (-1, 16))
    scale = _nearest(y.abs().amax(-1) / 6, E4M3)
    wide = torch.tensor(E4M3, dtype=torch.float64)[scale][..., None]
    code = torch.where(wide > 0, _nearest((y.abs() / torch.where(wide > 0, wide, 1.0)).clamp(max=6.0), CODES), 0)
    code = code + torch.where((y < 0) & (wide > 0), 8, 0)
    return code.flatten(-2), scale, torch.where(bad, 255, e + 127)


def values(code: torch.Tensor, scale: torch.Tensor, exponent: torch.Tensor) -> torch.Tensor:
    """float64 rows [..., D]."""
    grid = torch.tensor(CODES + [-c for c in CODES], dtype=torch.float64)
    x = grid[code].unflatten(-1, (-1, 16)) * torch.tensor(E4M3 + [math.nan], dtype=torch.float64)[scale][..., None]
    power = torch.where(exponent == 255, math.nan, 2.0 ** (exponent.double() - 127))
    return x.flatten(-2) * power[..., None]


def stored(x: torch.Tensor) -> torch.Tensor:
    """What rows read back as, in float64."""
    return values(*quantise(x))


def granule(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Bytes [..., 18 D + 32] of K and V rows [..., 16, D]."""
    out = []
    for x, turned in ((k, False), (v, True)):
        code, scale, exponent = quantise(x)
        out.append((code[..., 0::2] + 16 * code[..., 1::2]).flatten(-2))
        out.append((scale.transpose(-1, -2) if turned else scale).flatten(-2))
        out.append(exponent)
    return torch.cat(out, -1).to(torch.uint8)


def parts(cells: torch.Tensor, dim: int):
    """((codes, scales, exponents) of K, the same of V) of granule bytes [..., 18 D + 32], as integers."""
    out, at = [], 0
    for turned in (False, True):
        pair = cells[..., at:at + 8 * dim].unflatten(-1, (16, dim // 2)).long()
        code = torch.stack([pair % 16, pair // 16], -1).flatten(-2)
        scale = cells[..., at + 8 * dim:at + 9 * dim].long()
        scale = scale.unflatten(-1, (dim // 16, 16)).transpose(-1, -2) if turned else scale.unflatten(-1, (16, dim // 16))
        out.append((code, scale, cells[..., at + 9 * dim:at + 9 * dim + 16].long()))
        at += 9 * dim + 16
    return tuple(out)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float):
    """(out, sum of p |v|, largest sum |q k| scale) in float64 of q [H, n, D] over k, v [Hkv, m, D] (m may be 0)."""
    group = q.shape[0] // k.shape[0]
    q, k, v = q.double(), k.double().repeat_interleave(group, 0), v.double().repeat_interleave(group, 0)
    if k.shape[1] == 0:
        zero = torch.zeros_like(q)
        return zero, zero, 0.0
    p = torch.softmax(q @ k.transpose(1, 2) * scale, -1)
    return p @ v, p @ v.abs(), float((q.abs() @ k.abs().transpose(1, 2)).max() * scale)


def norm_mrope(x: torch.Tensor, weight: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, axes,
               eps: float) -> torch.Tensor:
    """x [rows, T, heads, D] in float64: RMSNorm times (1 + w), then frequency i turned by
    positions[axes[i]] * inv_freq[i]."""
    y = x.double()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * (1 + weight.double())
    half = len(axes)
    out = y.clone()
    for i, a in enumerate(axes):
        angle = (positions[a].double() * inv_freq[i].double())[:, :, None]
        lo, hi = y[..., i], y[..., i + half]
        out[..., i] = lo * angle.cos() - hi * angle.sin()
        out[..., i + half] = hi * angle.cos() + lo * angle.sin()
    return out
