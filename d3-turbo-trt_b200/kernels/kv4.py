"""Key/value cache in 4 bits, in pages, and the attention that reads it (sm_100a).

``Kv4Cache`` is a pool of pages for every layer; a page holds ``page_tokens`` tokens' keys and
values of all kv heads. A row is kept as e2m1 codes with one e4m3 scale for 16 channels and one
power of two: 4.56 bits a value at head_dim 128, against 16 in a snapshot (the layout is written
down in ``include/d3b200.h``). What a row reads back as is exact in bf16 and, between fp16's
subnormals and its largest magnitude, in fp16.

* ``cache.append(layer, k, v, slots)`` quantises rows into slots (page * page_tokens + place);
* ``cache.read(layer, table, tokens)`` gives a sequence's rows back in 16 bits;
* ``cache.copy_pages(src, dst)`` / ``cache.move_pages(src, dst, tables)`` copy pages of every
  layer, the latter rewriting page tables in the same launch;
* ``decode_attention(q, cache, layer, table, lengths, scale=...)`` attends with the newest tokens
  of many sequences, each over its own pages;
* ``question_attention(q, cache, layer, table, state_len, k_q, v_q, lengths, scale=...)`` is
  ``prefix_bidir_attention`` over a state that lies in the cache.

Page numbers, slots and lengths given as device tensors are not read on the host: the kernels leave
out what does not fit the pool or the table and record an input error (``SITE_BAD_SLOT``,
``SITE_BAD_PAGE``, ``SITE_BAD_LENGTH``, ``SITE_BAD_MOVE``; ``_lib.device_error()`` reads it).
A row that held a NaN or an infinity reads back as NaN.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Sequence

import torch

from .. import _lib
from .prefix_bidir import _launch as _prefix_bidir, block_offsets

HEAD_DIMS = (64, 128, 256)
PAGE_TOKENS = (16, 32, 64, 128, 256)
SITE_BAD_SLOT, SITE_BAD_PAGE, SITE_BAD_LENGTH, SITE_BAD_MOVE = 2101, 2102, 2103, 2104

append_key = "append"  # tells a plan's kind from the others'
_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


@functools.lru_cache(maxsize=256)
def page_bytes(kv_heads: int, head_dim: int, page_tokens: int) -> int:
    """Bytes of one page of one layer."""
    _check_shape(kv_heads, head_dim, page_tokens)
    return kv_heads * (page_tokens // 16) * (18 * head_dim + 32)


def _check_shape(kv_heads: int, head_dim: int, page_tokens: int) -> None:
    if head_dim not in HEAD_DIMS:
        raise RuntimeError(f"unsupported head_dim {head_dim}")
    if page_tokens not in PAGE_TOKENS:
        raise RuntimeError(f"page_tokens must be one of {PAGE_TOKENS}, got {page_tokens}")
    if not 0 < kv_heads <= 65535:
        raise RuntimeError(f"kv_heads must lie in [1, 65535], got {kv_heads}")


def _index(t: torch.Tensor, dtype: torch.dtype, device: torch.device, what: str) -> None:
    if t.dtype != dtype or t.device != device:
        raise RuntimeError(f"{what} must be {dtype} on {device}, got {t.dtype} on {t.device}")


@functools.lru_cache(maxsize=256)
def _plans_of(kv_heads: int, head_dim: int, page_tokens: int, device: torch.device) -> dict:
    """Checked calls on caches of one shape, by what the checks look at: shapes, strides, types, devices."""
    return {}


class Kv4Cache:
    """``pool`` [layers, pages, page_bytes] uint8, allocated here or, with ``over``, the caller's."""

    def __init__(self, layers: int, pages: int, *, kv_heads: int, head_dim: int, page_tokens: int = 64,
                 device: torch.device | str | int | None = None):
        if layers < 0 or pages < 0:
            raise RuntimeError("layers and pages must not be negative")
        size = page_bytes(kv_heads, head_dim, page_tokens)
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("the 4-bit cache needs CUDA")
        self._adopt(torch.empty(layers, pages, size, dtype=torch.uint8, device=dev), kv_heads, head_dim, page_tokens)

    @classmethod
    def over(cls, pool: torch.Tensor, *, kv_heads: int, head_dim: int, page_tokens: int = 64) -> "Kv4Cache":
        """A cache over an existing uint8 buffer [layers, pages, page_bytes] (contiguous, not copied)."""
        size = page_bytes(kv_heads, head_dim, page_tokens)
        if not pool.is_cuda:
            raise RuntimeError("the 4-bit cache needs CUDA")
        if pool.dtype != torch.uint8 or pool.dim() != 3 or pool.shape[2] != size:
            raise RuntimeError(f"pool must be uint8 [layers, pages, {size}], got {pool.dtype} {tuple(pool.shape)}")
        if not pool.is_contiguous() or pool.data_ptr() % 16:
            raise RuntimeError("pool must be contiguous and 16-byte aligned")
        cache = cls.__new__(cls)
        cache._adopt(pool, kv_heads, head_dim, page_tokens)
        return cache

    def _adopt(self, pool: torch.Tensor, kv_heads: int, head_dim: int, page_tokens: int) -> None:
        self.pool, self.kv_heads, self.head_dim, self.page_tokens = pool, kv_heads, head_dim, page_tokens
        self.layers, self.pages = pool.shape[0], pool.shape[1]
        self.device = pool.device
        self._c = _lib.Kv4CacheStruct(pool.data_ptr(), self.layers, self.pages, kv_heads, head_dim, page_tokens)
        self._ref = ctypes.byref(self._c)
        self._plans = _plans_of(kv_heads, head_dim, page_tokens, self.device)

    @property
    def nbytes(self) -> int:
        return self.pool.numel()

    def _plan(self, key: tuple, make):
        """What ``make()`` checked and worked out for calls of this key, kept for the next one."""
        plan = self._plans.get(key)
        if plan is None:
            plan = make()
            if len(self._plans) >= 512:
                self._plans.clear()
            self._plans[key] = plan
        return plan

    def _check_layer(self, layer: int) -> None:
        if not 0 <= layer < self.layers:
            raise RuntimeError(f"layer {layer} of {self.layers}")

    def slots(self, pages: Sequence[int] | torch.Tensor, start: int, count: int) -> torch.Tensor:
        """int64 slots of tokens ``start`` .. ``start + count`` of the sequence whose pages these are."""
        table = torch.as_tensor(pages, dtype=torch.int64, device=self.device)
        if start < 0 or count < 0 or start + count > table.numel() * self.page_tokens:
            raise RuntimeError(f"tokens {start} .. {start + count} of {table.numel()} pages")
        at = torch.arange(start, start + count, device=self.device)
        return table[at // self.page_tokens] * self.page_tokens + at % self.page_tokens

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise rows k, v [n, kv_heads, head_dim] (fp16 or bf16, any token and head strides) into ``slots``.

        ``slots`` [n] int64 on the device; a negative slot leaves its row out. Slots must differ: one
        that is named twice holds a mixture of the rows."""
        self._check_layer(layer)
        key = (append_key, k.shape, k.dtype, k.device, v.shape, v.dtype, v.device, slots.shape, slots.dtype, slots.device)
        n, code, index, fn = self._plan(key, lambda: self._plan_append(k, v, slots))
        if n == 0:
            return
        k, v, slots = _lib.rows16(k), _lib.rows16(v), slots.contiguous()
        with _lib.on_device(self.device):
            status = fn(self._ref, layer, k.data_ptr(), _lib.strides(k.stride(), 2), v.data_ptr(),
                        _lib.strides(v.stride(), 2), slots.data_ptr(), n, code, _lib.raw_stream(index))
        if status:
            _lib.check(status, "d3b_kv4_append")

    def _plan_append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> tuple:
        n, device, dtype = slots.numel(), self.device, k.dtype
        shape = (n, self.kv_heads, self.head_dim)
        if slots.dim() != 1 or k.shape != shape or v.shape != shape:
            raise RuntimeError(f"k and v must be [n, {self.kv_heads}, {self.head_dim}] and slots [n], got "
                               f"{tuple(k.shape)}, {tuple(v.shape)}, {tuple(slots.shape)}")
        if dtype not in _TYPES or v.dtype != dtype or k.device != device or v.device != device:
            raise RuntimeError(f"k and v must be fp16 or bf16 on {device}, got {dtype} on {k.device} and "
                               f"{v.dtype} on {v.device}")
        _index(slots, torch.int64, device, "slots")
        return n, _TYPES[dtype], device.index, _lib.lib().d3b_kv4_append

    def read(self, layer: int, table: torch.Tensor, tokens: int, *, dtype: torch.dtype = torch.bfloat16,
             ) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [kv_heads, tokens, head_dim] of the first ``tokens`` tokens of pages ``table`` [n] int32."""
        self._check_layer(layer)
        if dtype not in _TYPES:
            raise RuntimeError(f"read gives fp16 or bf16, not {dtype}")
        self._check_table(table, tokens)
        k = torch.empty((self.kv_heads, tokens, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if tokens:
            table = table.contiguous()
            with _lib.on_device(self.device):
                status = _lib.lib().d3b_kv4_read(self._ref, layer, table.data_ptr(), table.numel(), tokens, k.data_ptr(),
                                                 v.data_ptr(), _TYPES[dtype], _lib.raw_stream(self.device.index))
            if status:
                _lib.check(status, "d3b_kv4_read")
        return k, v

    def _check_table(self, table: torch.Tensor, tokens: int) -> None:
        _index(table, torch.int32, self.device, "table")
        if table.dim() != 1 or not 0 <= tokens <= table.numel() * self.page_tokens:
            raise RuntimeError(f"{tokens} tokens in a table of shape {tuple(table.shape)} and pages of {self.page_tokens}")

    def copy_pages(self, src: torch.Tensor | Sequence[int], dst: torch.Tensor | Sequence[int]) -> None:
        """Copy page ``src[i]`` to page ``dst[i]`` in every layer. No destination may be a source or
        stand twice (checked for lists; for device tensors that is the caller's part)."""
        self._move(src, dst, None)

    def move_pages(self, src: torch.Tensor | Sequence[int], dst: torch.Tensor | Sequence[int],
                   tables: torch.Tensor) -> None:
        """``copy_pages``, and every entry of ``tables`` (int32, contiguous) that is some ``src[i]``
        becomes ``dst[i]``, in one launch. ``src`` must be ascending (the kernel records a list that
        is not, or a destination among the sources, as an input error)."""
        _index(tables, torch.int32, self.device, "tables")
        if not tables.is_contiguous():
            raise RuntimeError("tables must be contiguous")
        self._move(src, dst, tables)

    def _move(self, src, dst, tables) -> None:
        if not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
            src, dst = [int(p) for p in src], [int(p) for p in dst]
            if len(src) != len(dst):
                raise RuntimeError(f"{len(src)} pages to {len(dst)}")
            if len(set(src) | set(dst)) < len(set(src)) + len(dst):
                raise RuntimeError("a destination is a source or stands twice")
            if tables is not None and any(a >= b for a, b in zip(src, src[1:])):
                raise RuntimeError("src must be ascending")
            if any(not 0 <= p < self.pages for p in src + dst):
                raise RuntimeError(f"pages must lie in [0, {self.pages})")
            both = torch.tensor([src, dst], dtype=torch.int32).to(self.device)
            src, dst = both[0], both[1]
        else:
            src, dst = (t if isinstance(t, torch.Tensor) else torch.tensor(list(t), dtype=torch.int32, device=self.device)
                        for t in (src, dst))
        _index(src, torch.int32, self.device, "src")
        _index(dst, torch.int32, self.device, "dst")
        n = src.numel()
        if src.dim() != 1 or dst.shape != src.shape or n > self.pages:
            raise RuntimeError(f"src and dst must be [n] with n <= {self.pages}, got {tuple(src.shape)}, {tuple(dst.shape)}")
        if n == 0:
            return
        src, dst = src.contiguous(), dst.contiguous()
        with _lib.on_device(self.device):
            status = _lib.lib().d3b_kv4_move_pages(
                self._ref, src.data_ptr(), dst.data_ptr(), n, None if tables is None else tables.data_ptr(),
                0 if tables is None else tables.numel(), _lib.raw_stream(self.device.index))
        if status:
            _lib.check(status, "d3b_kv4_move_pages")


def _check_query(q: torch.Tensor, cache: Kv4Cache) -> None:
    if not q.is_cuda or q.device != cache.device:
        raise RuntimeError(f"q is on {q.device}, the cache on {cache.device}")
    if q.dtype not in _TYPES:
        raise RuntimeError("the 4-bit cache's attention needs fp16 or bf16 queries")
    if q.shape[-1] != cache.head_dim:
        raise RuntimeError(f"q has head_dim {q.shape[-1]}, the cache {cache.head_dim}")
    if q.shape[1] == 0 or q.shape[1] % cache.kv_heads:
        raise RuntimeError("heads must be divisible by kv heads")


def _check_out(out: torch.Tensor, q: torch.Tensor) -> None:
    if (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(-1) != 1
            or out.data_ptr() % 16 or any(s % 8 or (s == 0 and n > 1) for s, n in zip(out.stride()[:-1], out.shape))):
        raise RuntimeError("out must be like q, with a contiguous last dimension and 16-byte aligned rows of its own")


def decode_attention(q: torch.Tensor, cache: Kv4Cache, layer: int, table: torch.Tensor, lengths: torch.Tensor, *,
                     scale: float, causal: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the newest tokens of B sequences over their cached keys and values.

    q [B, H, L, D] (any strides, D contiguous) or [B, H, D] for one token each; ``table`` [B, width]
    int32 page numbers (entries behind a sequence's last page are not read); ``lengths`` [B] int32
    tokens in the cache, the L newest among them already appended. Every token sees all ``lengths[b]``
    tokens, or with ``causal`` those up to itself. Rows without a key are zero. ``scale`` must
    be positive. Returns a tensor like q.
    """
    if q.dim() == 3:
        out = None if out is None else out.unsqueeze(2)
        return decode_attention(q.unsqueeze(2), cache, layer, table, lengths, scale=scale, causal=causal, out=out).squeeze(2)
    key = (decode_attention, q.shape, q.dtype, q.device, table.shape, table.stride(), table.dtype, table.device,
           lengths.shape, lengths.stride(), lengths.dtype, lengths.device)
    rows, heads, width, code, index, need, fn = cache._plan(key, lambda: _plan_decode(q, cache, table, lengths))
    cache._check_layer(layer)
    if not 0 < scale < math.inf:
        raise RuntimeError(f"scale must be positive and finite, got {scale}")
    q = _lib.rows16(q)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_out(out, q)
    if need:
        if table.stride(1) != 1 or table.stride(0) < 0:
            table = table.contiguous()
        if lengths.stride(0) != 1:
            lengths = lengths.contiguous()
        # from the caching allocator at every call: calls on other streams and captured graphs get
        # their own, and it is ordered with the stream like any tensor
        with _lib.on_device(cache.device):
            work = cache.pool.new_empty(need)
            status = fn(cache._ref, layer, q.data_ptr(), _lib.strides(q.stride(), 3), table.data_ptr(), table.stride(0),
                        table.shape[1], lengths.data_ptr(), rows, heads, width, causal, code, scale, out.data_ptr(),
                        _lib.strides(out.stride(), 3), work.data_ptr(), need, _lib.raw_stream(index))
        if status:
            _lib.check(status, "d3b_kv4_decode")
    return out


def _plan_decode(q: torch.Tensor, cache: Kv4Cache, table: torch.Tensor, lengths: torch.Tensor) -> tuple:
    if q.dim() != 4:
        raise RuntimeError(f"q must be [B, H, L, D] or [B, H, D], got {tuple(q.shape)}")
    _check_query(q, cache)
    rows, heads, width, _ = q.shape
    device, lib = cache.device, _lib.lib()
    _index(table, torch.int32, device, "table")
    _index(lengths, torch.int32, device, "lengths")
    if table.dim() != 2 or table.shape[0] != rows or tuple(lengths.shape) != (rows,):
        raise RuntimeError(f"table must be [{rows}, width] and lengths [{rows}], got {tuple(table.shape)}, "
                           f"{tuple(lengths.shape)}")
    need = 0
    if rows and width:
        with _lib.on_device(device):
            need = lib.d3b_kv4_decode_workspace_size(cache._ref, rows, heads, width, table.shape[1])
        if need == 0:
            raise RuntimeError(f"decode_attention: queries {tuple(q.shape)} over tables {tuple(table.shape)} are too many")
    return rows, heads, width, _TYPES[q.dtype], device.index, need, lib.d3b_kv4_decode


def question_attention(q: torch.Tensor, cache: Kv4Cache, layer: int, table: torch.Tensor, state_len: int,
                       k_q: torch.Tensor, v_q: torch.Tensor, lengths: Sequence[int] | torch.Tensor, *, scale: float,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Bidirectional question attention over a state in the cache: ``prefix_bidir_attention`` whose
    state keys and values are the first ``state_len`` tokens of pages ``table`` [n] int32.

    q [B, H, L, D], k_q/v_q [B, H_kv, L, D], ``lengths`` as there. Returns [B, H, L, D], zero rows
    for padding. Small batches read the codes in place, larger ones widen the state first. A page outside
    the pool (2102) or a device length outside [0, L] (2010) is recorded as an input error: the length is
    clamped, the page's tokens are left out in place and keys and values of zero where the state is widened.
    """
    cache._check_layer(layer)
    if not 0 < scale < math.inf:
        raise RuntimeError(f"scale must be positive and finite, got {scale}")
    key = (question_attention, q.shape, q.dtype, q.device, k_q.shape, k_q.dtype, k_q.device, v_q.shape, v_q.dtype,
           v_q.device, table.shape, table.dtype, table.device, state_len)
    rows, heads, width, code, index, need, fn = cache._plan(key, lambda: _plan_question(q, cache, table, state_len, k_q, v_q))
    if not (isinstance(lengths, torch.Tensor) and lengths.is_cuda):
        lengths = [int(n) for n in (lengths.tolist() if isinstance(lengths, torch.Tensor) else lengths)]
        if any(not 0 <= n <= width for n in lengths):
            raise RuntimeError(f"lengths must lie in [0, {width}]")
    elif lengths.dim() != 1:
        raise RuntimeError(f"lengths must be [{rows}], got {tuple(lengths.shape)}")
    if len(lengths) != rows:
        raise RuntimeError(f"{len(lengths)} lengths for {rows} question blocks")
    q, k_q, v_q = _lib.rows16(q), _lib.rows16(k_q), _lib.rows16(v_q)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_out(out, q)
    if rows == 0 or width == 0:
        return out
    device = cache.device
    with _lib.on_device(device):
        lens = block_offsets(lengths, device)
        if need:
            table, work = table.contiguous(), cache.pool.new_empty(need)
            status = fn(cache._ref, layer, q.data_ptr(), _lib.strides(q.stride(), 3), table.data_ptr(), table.shape[0],
                        state_len, k_q.data_ptr(), _lib.strides(k_q.stride(), 3), v_q.data_ptr(),
                        _lib.strides(v_q.stride(), 3), lens.data_ptr(), rows, heads, width, code, scale, out.data_ptr(),
                        _lib.strides(out.stride(), 3), work.data_ptr(), need, _lib.raw_stream(index))
            if status:
                _lib.check(status, "d3b_kv4_question")
        else:
            k, v = cache.read(layer, table, state_len, dtype=q.dtype)
            if k_q.stride() != v_q.stride():
                k_q, v_q = (x.clone(memory_format=torch.contiguous_format) for x in (k_q, v_q))
            # graphs may be replayed in any order and side by side: each call in one has its own workspace
            _prefix_bidir(q, k, v, k_q, v_q, lens, scale, out, torch.cuda.is_current_stream_capturing())
    return out


def _plan_question(q: torch.Tensor, cache: Kv4Cache, table: torch.Tensor, state_len: int, k_q: torch.Tensor,
                   v_q: torch.Tensor) -> tuple:
    if q.dim() != 4:
        raise RuntimeError(f"q must be [B, H, L, D], got {tuple(q.shape)}")
    _check_query(q, cache)
    rows, heads, width, dim = q.shape
    cache._check_table(table, state_len)
    if k_q.dtype != q.dtype or v_q.dtype != q.dtype or k_q.device != q.device or v_q.device != q.device:
        raise RuntimeError("q, k and v must share a dtype and a device")
    if tuple(k_q.shape) != (rows, cache.kv_heads, width, dim) or v_q.shape != k_q.shape:
        raise RuntimeError(f"k_q/v_q must be [B, H_kv, L, D] = {(rows, cache.kv_heads, width, dim)}")
    need, lib = 0, _lib.lib()
    if rows and width and _reads_codes(rows, heads, cache.kv_heads, width, state_len, dim):
        with _lib.on_device(cache.device):
            need = lib.d3b_kv4_question_workspace_size(cache._ref, rows, heads, width, state_len)
    return rows, heads, width, _TYPES[q.dtype], cache.device.index, need, lib.d3b_kv4_question


# What the two ways of a question batch cost on B200, in us, by head_dim (fitted to 190 measured shapes,
# 1 to 255 blocks of 3 to 48 tokens over 64 to 16384; off by a quarter at most where the two are near).
# In place: a start, a piece of 32 rows x 64 keys of a CTA (296 run), the first pieces' share of the
# merge. Widened: the state's read and a start, a 128-key tile of a unit of 128 rows, and a
# floor and a slope for few units, whose keys that kernel splits.
_IN_PLACE = {64: (7.0, 1.1, 1.5), 128: (7.5, 1.47, 3.0), 256: (9.5, 2.13, 5.0)}
_WIDENED = {64: (9.4, 0.8, 21.0, 0.0), 128: (9.4, 0.87, 24.0, 0.03), 256: (9.4, 1.55, 18.0, 0.33)}


def _reads_codes(rows: int, heads: int, kv_heads: int, width: int, state_len: int, dim: int) -> bool:
    """Whether a question batch is faster reading the state's codes in place than widening the state first
    and running ``prefix_bidir_attention``'s kernel. For instance 32 query and 4 kv heads of 128 over 4096
    tokens: one block of 12 tokens 17 against 37 us, 4 blocks of 12 29 against 37, 16 blocks of 12 82
    against 38."""
    group = heads // kv_heads
    pieces = -(-state_len // 64) + -(-width // 64)
    share = -(-(rows * kv_heads * -(-width * group // 32) * pieces) // 296)
    start, piece, first = _IN_PLACE[dim]
    in_place = start + piece * share + first * min(share, 3) + 8 * (share - 1) / pieces
    units, tiles = rows * kv_heads * -(-width * group // 128), -(-(state_len + width) // 128)
    start, tile, floor, slope = _WIDENED[dim]
    if units <= 148:
        widened = start + max(min(tile * tiles, floor + slope * tiles), 1.2 * tile * tiles * units / 148)
    else:
        widened = start + -(-units // 148) * (3.4 + tile * tiles)
    return in_place < widened
