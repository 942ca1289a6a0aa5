"""Inputs on the device that are out of range: recorded, and no other launch hears of it."""

from __future__ import annotations

import pytest
import torch

from conftest import ROOT  # noqa: F401  (puts the repository on sys.path)

from d3_turbo_trt_b200 import _lib
from d3_turbo_trt_b200.kernels import kv4
from d3_turbo_trt_b200.kernels import prefix_bidir as pb
from d3_turbo_trt_b200.model import quant

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def new(*shape, seed=1):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=torch.bfloat16)


def same(a, b):
    """Equal but for the order in which a split unit's parts are added: one bf16 rounding each."""
    return float((a.float() - b.float()).abs().max()) <= 2.0**-7 * float(b.float().abs().max())


def bad_slot(cache, table):
    cache.append(0, new(2, 2, 64), new(2, 2, 64), torch.tensor([10**6, -1], device="cuda"))
    return kv4.SITE_BAD_SLOT


def bad_page(cache, table):
    kv4.decode_attention(new(1, 4, 1, 64), cache, 0, i32([[99, 0]]), i32([30]), scale=0.1)
    return kv4.SITE_BAD_PAGE


def bad_length(cache, table):
    kv4.decode_attention(new(1, 4, 1, 64), cache, 0, table[None], i32([9999]), scale=0.1)
    return kv4.SITE_BAD_LENGTH


def bad_move(cache, table):
    cache.move_pages(i32([3, 2]), i32([7, 8]), i32([[0]]))
    return kv4.SITE_BAD_MOVE


def bad_block(cache, table):
    kv4.question_attention(new(1, 4, 3, 64), cache, 0, table, 40, new(1, 2, 3, 64), new(1, 2, 3, 64), i32([5]), scale=0.1)
    return pb.SITE_BAD_LENGTH


@pytest.mark.parametrize("break_", [bad_slot, bad_page, bad_length, bad_move, bad_block])
def test_other_launches_are_as_ever(break_):
    """State and question attention, the GEMM and a second decode behind a bad input that nobody has read."""
    cache, table = kv4.Kv4Cache(1, 10, kv_heads=2, head_dim=64, page_tokens=16), i32([0, 1, 2, 3])
    cache.append(0, new(64, 2, 64), new(64, 2, 64, seed=2), cache.slots(table, 0, 64))
    q, k, v = new(40, 8, 24, 128, seed=3), new(40, 2, 24, 128, seed=4), new(40, 2, 24, 128, seed=5)
    ks, vs = new(2, 4000, 128, seed=6), new(2, 4000, 128, seed=7)
    x, w = new(300, 512, seed=8), new(256, 512, seed=9)

    def run():
        codes, scale = quant.quantize_rows(x, "fp8")
        wc, ws = quant.quantize_weight(w, "fp8")
        return (pb.prefix_bidir_attention(q, ks, vs, k, v, [24] * 40, scale=0.1), pb.state_attention(q, k, v, scale=0.1),
                quant.scaled_mm(codes, wc, scale, ws, out_dtype=torch.bfloat16),
                kv4.decode_attention(q[:1, :4, :1, :64], cache, 0, table[None], i32([40]), scale=0.1))

    assert _lib.device_error() == 0
    want = run()
    torch.cuda.synchronize()
    code = break_(cache, table)
    torch.cuda.synchronize()
    got = run()
    assert all(same(a, b) for a, b in zip(got, want))
    assert _lib.device_error() == code and _lib.device_error() == 0


@pytest.mark.parametrize("in_place", [True, False])
def test_a_clamped_block_has_results(monkeypatch, in_place):
    """A block's length beyond L counts as L, one below 0 as 0, whichever way the state is read."""
    monkeypatch.setattr(kv4, "_reads_codes", lambda *a: in_place)
    kv4._plans_of.cache_clear()
    cache, table = kv4.Kv4Cache(1, 4, kv_heads=2, head_dim=128, page_tokens=32), i32([0, 1, 2, 3])
    cache.append(0, new(128, 2, 128), new(128, 2, 128, seed=2), cache.slots(table, 0, 128))
    q, k, v = new(3, 8, 9, 128, seed=3), new(3, 2, 9, 128, seed=4), new(3, 2, 9, 128, seed=5)
    ask = lambda n: kv4.question_attention(q, cache, 0, table, 100, k, v, i32(n), scale=0.1)  # noqa: E731
    want = ask([9, 0, 4])
    assert _lib.device_error() == 0
    assert same(ask([1000, -5, 4]), want)
    assert _lib.device_error() == pb.SITE_BAD_LENGTH
    kv4._plans_of.cache_clear()


def test_a_wait_that_gave_up_goes_first():
    cache, table = kv4.Kv4Cache(1, 4, kv_heads=2, head_dim=64, page_tokens=16), i32([0, 1, 2, 3])
    code = bad_slot(cache, table)
    assert _lib.device_error(reset=False) == code
    assert _lib.lib().d3b_selftest_wait_timeout(200, None) == _lib.OK
    torch.cuda.synchronize()
    assert _lib.device_error() == 9001 and _lib.device_error() == 0


def test_lengths_of_another_shape_are_refused():
    """A table of lengths per block and something else: its first column is not its first elements."""
    cache, table = kv4.Kv4Cache(1, 4, kv_heads=2, head_dim=64, page_tokens=16), i32([0, 1, 2, 3])
    q, k = new(2, 4, 3, 64), new(2, 2, 3, 64)
    for lengths in (i32([[3, 1], [2, 1]]), i32([[3], [2]]), i32([3, 2, 1]), i32(3), torch.tensor([[3, 1], [2, 1]])):
        with pytest.raises((RuntimeError, TypeError)):
            kv4.question_attention(q, cache, 0, table, 40, k, k, lengths, scale=0.1)
    assert _lib.device_error() == 0
