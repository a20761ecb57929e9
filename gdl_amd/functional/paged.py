"""Attention of streams that keep their whole history, in pages of a shared pool.

A model that is trained with ``window_attention(q, k, v, (-1, 0))`` sees a stream's whole past.  To
answer such streams as their tokens come, ``PagedCache`` holds keys and values of any number of
streams of any length, in the tokens' type or in 8 bits with a scale for each token and head:

    cache = PagedCache.empty(pages, Hk, D, dtype=torch.int8)     # a pool; table: int32 [B, n] page numbers
    cache.write(k, v, table, ptr, start)                         # packed tokens into their streams' pages
    out = paged_attention(q, cache, table, ptr, start)           # [T, H, D]: a prompt, or a piece of one
    out = paged_attention_step(q, k, v, cache, table, positions) # [B, H, D]: one token per stream

Token ``j`` of stream ``b`` lies in page ``table[b, j // page]``, slot ``j % page``; who gets which page is
the caller's to say, and streams may share pages of a common past.  All attention reads what the cache
holds, new tokens included, so pieces of any size give the same results.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from gdl_amd import _native as _nat
from gdl_amd.csrc import paged_attention_hip, paged_attention_step_hip, paged_read_hip, paged_write_hip
from gdl_amd.functional.attention import _plan
from gdl_amd.functional.relative_bias import check_buckets

_NARROW = (torch.int8, torch.float8_e4m3fn)


# ═══════════════════════════════════════════════════════════════════
# Custom ops: what everything but plain eager execution uses (_native.plain_eager)
# ═══════════════════════════════════════════════════════════════════


@torch.library.custom_op("geoembodied::paged_write", mutates_args=("k_pages", "v_pages", "k_scale", "v_scale"))
def _write_op(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, k_scale: Optional[Tensor], v_scale: Optional[Tensor],
              table: Tensor, ptr: Optional[Tensor], start: Optional[Tensor]) -> None:
    paged_write_hip(k, v, k_pages, v_pages, k_scale, v_scale, table, ptr, start)


@_write_op.register_fake
def _(k, v, k_pages, v_pages, k_scale, v_scale, table, ptr, start):
    return None


@torch.library.custom_op("geoembodied::paged_read", mutates_args=())
def _read_op(k_pages: Tensor, v_pages: Tensor, k_scale: Optional[Tensor], v_scale: Optional[Tensor], table: Tensor,
             ptr: Optional[Tensor], start: Optional[Tensor], tokens: int, dtype: torch.dtype) -> Tuple[Tensor, Tensor]:
    return paged_read_hip(k_pages, v_pages, k_scale, v_scale, table, ptr, start, tokens, dtype)


@_read_op.register_fake
def _(k_pages, v_pages, k_scale, v_scale, table, ptr, start, tokens, dtype):
    k, v = (k_pages.new_empty((tokens, k_pages.shape[1], k_pages.shape[3]), dtype=dtype) for _ in range(2))
    return k, v


@torch.library.custom_op("geoembodied::paged_attention_step", mutates_args=("k_pages", "v_pages", "k_scale", "v_scale"))
def _step_op(q: Tensor, k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, k_scale: Optional[Tensor],
             v_scale: Optional[Tensor], table: Tensor, positions: Tensor, bias: Optional[Tensor], max_distance: int,
             scale: float) -> Tensor:
    return paged_attention_step_hip(q, k, v, k_pages, v_pages, k_scale, v_scale, table, positions, scale, bias,
                                    _plan(bias, max_distance, False))


@_step_op.register_fake
def _(q, k, v, k_pages, v_pages, k_scale, v_scale, table, positions, bias, max_distance, scale):
    return q.new_empty(q.shape)


@torch.library.custom_op("geoembodied::paged_attention", mutates_args=())
def _attention_op(q: Tensor, k_pages: Tensor, v_pages: Tensor, k_scale: Optional[Tensor], v_scale: Optional[Tensor], table: Tensor,
                  ptr: Optional[Tensor], start: Optional[Tensor], bias: Optional[Tensor], max_distance: int,
                  scale: float) -> Tensor:
    return paged_attention_hip(q, k_pages, v_pages, k_scale, v_scale, table, ptr, start, scale, bias, _plan(bias, max_distance, False))


@_attention_op.register_fake
def _(q, k_pages, v_pages, k_scale, v_scale, table, ptr, start, bias, max_distance, scale):
    return q.new_empty(q.shape)


def _check_table(name: str, table: Tensor, batch: int) -> None:
    if table.dtype is not torch.int32:
        raise TypeError(f"{name}: table must be int32, got {table.dtype}")
    shape = table.shape
    if len(shape) != 2 or shape[0] != batch or shape[1] < 1:
        raise ValueError(f"{name}: table [{batch}, pages of a stream], got {tuple(shape)}")


def _check_spans(name: str, table: Tensor, ptr: Optional[Tensor], start: Optional[Tensor]) -> None:
    batch = 1 if ptr is None else ptr.numel() - 1
    if ptr is not None and (ptr.dim() != 1 or batch < 1 or ptr.dtype.is_floating_point):
        raise ValueError(f"{name}: ptr must be int64 [B + 1] with at least one sequence, got {ptr.dtype} {tuple(ptr.shape)}")
    _check_table(name, table, batch)
    if start is not None and (start.shape != (batch,) or start.dtype.is_floating_point):
        raise ValueError(f"{name}: start int64 [{batch}], got {start.dtype} {tuple(start.shape)}")


def _no_grad(name: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward: call it under torch.no_grad()")


class PagedCache:
    """A pool of pages for keys and values: ``k [P, Hk, page, D]``, ``v [P, Hk, page / blk, D, blk]``.

    ``blk`` tokens take 64 bytes (16 in float32, 32 in 16 bits, 64 in 8 bits).  Pools of int8 or
    float8_e4m3fn have ``k_scale, v_scale``, float32 ``[P, Hk, page]``: a token's row of a head, of largest
    magnitude a, is kept as codes ``round(x * M / a)``, M = 127 or 448, and stands for ``code * a / M``.  Rows
    below 2^-100 are kept as zeros; one with an infinity or a NaN reads back as NaN throughout.  The object
    holds the tensors (given ones are used as they are); calls on it are ordered by the caller's stream.
    """

    def __init__(self, k: Tensor, v: Tensor, k_scale: Optional[Tensor] = None, v_scale: Optional[Tensor] = None):
        if k.dtype not in _nat.PAGED_DTYPES or v.dtype is not k.dtype:
            raise TypeError("PagedCache: float32, bfloat16, float16, int8 or float8_e4m3fn pools of one type, got "
                            f"{k.dtype}, {v.dtype}")
        narrow, blk = k.dtype in _NARROW, 64 // k.element_size()
        if k.dim() != 4 or k.shape[0] < 1 or k.shape[1] < 1:
            raise ValueError(f"PagedCache: k [pages, Hk, page, D], got {tuple(k.shape)}")
        pages, heads, page, d = k.shape
        if page % 64 or not 64 <= page <= 1 << 20:
            raise ValueError(f"PagedCache: pages of {page} tokens (a multiple of 64 up to 2^20)")
        if d % (16 if narrow else 8) or not 8 <= d <= 128:
            raise ValueError(f"PagedCache: head size {d} (a multiple of {16 if narrow else 8} up to 128 for {k.dtype})")
        if v.shape != (pages, heads, page // blk, d, blk):
            raise ValueError(f"PagedCache: v [{pages}, {heads}, {page // blk}, {d}, {blk}], got {tuple(v.shape)}")
        scales = (k_scale, v_scale) if narrow else ()
        if not narrow and (k_scale is not None or v_scale is not None):
            raise ValueError(f"PagedCache: a pool of {k.dtype} has no scales")
        for t in scales:
            if t is None or t.dtype is not torch.float32 or t.shape != (pages, heads, page):
                raise ValueError(f"PagedCache: a pool of {k.dtype} needs float32 scales [{pages}, {heads}, {page}] for k and v")
        tensors = (k, v, *scales)
        for t in tensors:
            if t.device != k.device:
                raise ValueError("PagedCache: tensors on different devices")
            if not t.is_contiguous() or (_nat.plain_eager(t) and t.data_ptr() % 16):
                raise ValueError("PagedCache: pools must be contiguous, on a multiple of 16 bytes")
            if t.requires_grad:
                raise ValueError("PagedCache: pools that need gradients")
        if all(_nat.plain_eager(t) for t in tensors):
            spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors)
            if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
                raise ValueError("PagedCache: tensors share memory")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.page, self.kv_heads, self.head_dim = page, heads, d

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, *, page: int = 64, dtype: torch.dtype = torch.float32,
              device="cuda") -> "PagedCache":
        """A pool of ``pages`` pages of ``page`` tokens, of no content."""
        if dtype not in _nat.PAGED_DTYPES:
            raise TypeError(f"PagedCache: float32, bfloat16, float16, int8 or float8_e4m3fn, got {dtype}")
        if pages < 1 or kv_heads < 1 or page < 64 or head_dim < 8:
            raise ValueError(f"PagedCache: {pages} pages of {page} tokens (from 64), {kv_heads} heads of {head_dim} (from 8)")
        blk = 64 // dtype.itemsize
        k = torch.empty(pages, kv_heads, page, head_dim, dtype=dtype, device=device)
        v = torch.empty(pages, kv_heads, page // blk, head_dim, blk, dtype=dtype, device=device)
        if dtype not in _NARROW:
            return cls(k, v)
        scales = (torch.empty(pages, kv_heads, page, dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, *scales)

    def _token_dtype(self, name: str, dtype: torch.dtype) -> None:
        stored = self.k.dtype
        if dtype not in _nat.SEQUENCE_DTYPES or (dtype is not stored and stored not in _NARROW):
            wanted = "float32, bfloat16 or float16" if stored in _NARROW else f"{stored} as the pool"
            raise TypeError(f"{name}: tokens of {wanted}, got {dtype}")

    def write(self, k: Tensor, v: Tensor, table: Tensor, ptr: Optional[Tensor] = None, start: Optional[Tensor] = None) -> None:
        """Tokens ``k, v [T, Hk, D]`` of packed sequences into their pages.

        Args:
            k, v: of the pool's type, or float32, bfloat16 or float16 for an 8-bit pool.
            table: int32 [B, n], the streams' pages.  Entries that no token needs may be anything; tokens
                whose entry is outside the pool, or that lie beyond the table, are left out.
            ptr: int64 [B + 1] offsets of the sequences in the T tokens; None: one sequence.
            start: int64 [B], position of each sequence's first token in its stream; None: 0.  Tokens at
                negative positions are left out.
        """
        shape = k.shape
        if len(shape) != 3 or v.shape != shape or shape[1:] != (self.kv_heads, self.head_dim):
            raise ValueError(f"PagedCache.write: k and v [T, {self.kv_heads}, {self.head_dim}], got {tuple(k.shape)}, "
                             f"{tuple(v.shape)}")
        _check_spans("PagedCache.write", table, ptr, start)
        self._token_dtype("PagedCache.write", k.dtype)
        _no_grad("PagedCache.write", k, v)
        if dev := _nat.plain_device(k, v, self.k, self.v, self.k_scale, self.v_scale, table, ptr, start):
            paged_write_hip(k, v, self.k, self.v, self.k_scale, self.v_scale, table, ptr, start, dev)
        else:
            _nat.no_tangents("PagedCache.write", k, v)
            torch.ops.geoembodied.paged_write(k, v, self.k, self.v, self.k_scale, self.v_scale, table, ptr, start)

    def read(self, table: Tensor, ptr: Optional[Tensor], tokens: int, *, start: Optional[Tensor] = None,
             dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
        """The values of ``tokens`` tokens of packed sequences, ``k, v [tokens, Hk, D]``: what ``write`` with the
        same ``table``, ``ptr`` and ``start`` has put there.

        ``dtype``: float32, bfloat16 or float16 from an 8-bit pool (bfloat16 by default), the pool's own
        otherwise.  NaN for tokens without a page, 0 for tokens outside ``ptr[0] .. ptr[B]``.
        """
        tokens = int(tokens)
        if tokens < 0:
            raise ValueError(f"PagedCache.read: {tokens} tokens")
        if dtype is None:
            dtype = torch.bfloat16 if self.k.dtype in _NARROW else self.k.dtype
        _check_spans("PagedCache.read", table, ptr, start)
        self._token_dtype("PagedCache.read", dtype)
        if dev := _nat.plain_device(self.k, self.v, self.k_scale, self.v_scale, table, ptr, start):
            return paged_read_hip(self.k, self.v, self.k_scale, self.v_scale, table, ptr, start, tokens, dtype, dev)
        return torch.ops.geoembodied.paged_read(self.k, self.v, self.k_scale, self.v_scale, table, ptr, start, tokens, dtype)


def _check_queries(name: str, q: Tensor, cache: PagedCache, bias: Optional[Tensor]) -> int:
    """The number of queries."""
    shape = q.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or shape[1] < 1 or shape[1] % cache.kv_heads:
        raise ValueError(f"{name}: q [N, H, {cache.head_dim}], H a multiple of {cache.kv_heads}, got {tuple(shape)}")
    cache._token_dtype(name, q.dtype)
    if bias is not None and (bias.dim() != 2 or bias.shape[1] != shape[1]):
        raise ValueError(f"{name}: bias must be [buckets, {shape[1]}], got {tuple(bias.shape)}")
    return shape[0]


def paged_attention(
    q: Tensor,
    cache: PagedCache,
    table: Tensor,
    ptr: Optional[Tensor] = None,
    start: Optional[Tensor] = None,
    *,
    bias: Optional[Tensor] = None,
    max_distance: int = 128,
    scale: Optional[float] = None,
) -> Tensor:
    """Several new tokens of each stream: packed queries ``q [T, H, D]`` attend to all tokens of their streams up to
    themselves, which the cache holds already (``PagedCache.write`` with the same ``table``, ``ptr`` and ``start``).

    Args:
        q: ``H`` a multiple of the cache's heads (query head ``h`` reads key head ``h // (H / Hk)``), of the
            pool's type, or float32, bfloat16 or float16 over an 8-bit pool.
        table: int32 [B, n], the streams' pages.
        ptr: int64 [B + 1] offsets of the sequences in the T tokens; None: one sequence.
        start: int64 [B], position of each sequence's first token in its stream; None: 0.
        bias: [buckets, H], one-sided, as ``window_attention``'s.  The first call with a number of buckets and a
            ``max_distance`` copies their table to the device and cannot be captured into a graph.
        max_distance: where the bias's last bucket begins (at most 1024).
        scale: of the scores; ``D ** -0.5`` by default.

    Returns:
        [T, H, D] of q's type: ``window_attention``'s rows with the window ``(-1, 0)``.  0 for tokens outside
        ``ptr[0] .. ptr[B]`` and at negative positions, NaN for one of whose tokens has no page.  No gradients.
    """
    name = "paged_attention"
    _check_queries(name, q, cache, bias)
    _check_spans(name, table, ptr, start)
    _no_grad(name, q, bias)
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    pools = cache.k, cache.v, cache.k_scale, cache.v_scale
    if dev := _nat.plain_device(q, *pools, table, ptr, start, bias):
        return paged_attention_hip(q, *pools, table, ptr, start, scale, bias, _plan(bias, int(max_distance), False), dev)
    _nat.no_tangents(name, q, bias)
    if bias is not None:
        check_buckets(bias.shape[0], int(max_distance), False)
    return torch.ops.geoembodied.paged_attention(q, *pools, table, ptr, start, bias, int(max_distance), scale)


def paged_attention_step(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    cache: PagedCache,
    table: Tensor,
    positions: Tensor,
    *,
    bias: Optional[Tensor] = None,
    max_distance: int = 128,
    scale: Optional[float] = None,
) -> Tensor:
    """One token of each stream: ``k, v [B, Hk, D]`` go into the pages at ``positions`` (int64 [B], from 0), and
    ``q [B, H, D]`` attends to all the stream's tokens up to them, as the cache holds them.

    Over a pool of the tokens' type the result is ``window_attention``'s with the window ``(-1, 0)`` for the
    last token of such streams.  A stream at a negative position is left alone (its row is 0); one with a
    token that has no page (an entry of ``table`` [B, n] outside the pool, a position beyond it) gives NaN.
    No two streams may write to one slot.  No gradients.  ``bias`` is one-sided.  No streams: an empty result.
    """
    name, (hk, d) = "paged_attention_step", (cache.kv_heads, cache.head_dim)
    batch = _check_queries(name, q, cache, bias)
    rows = batch, hk, d
    if k.shape != rows or v.shape != rows:
        raise ValueError(f"{name}: k and v [{batch}, {hk}, {d}], got {tuple(k.shape)}, {tuple(v.shape)}")
    _check_table(name, table, batch)
    if positions.shape != (batch,) or positions.dtype.is_floating_point:
        raise ValueError(f"{name}: positions int64 [{batch}], got {positions.dtype} {tuple(positions.shape)}")
    _no_grad(name, q, k, v, bias)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    pools = cache.k, cache.v, cache.k_scale, cache.v_scale
    if dev := _nat.plain_device(q, k, v, *pools, table, positions, bias):
        return paged_attention_step_hip(q, k, v, *pools, table, positions, scale, bias, _plan(bias, int(max_distance), False), dev)
    _nat.no_tangents(name, q, k, v, bias)
    if bias is not None:
        check_buckets(bias.shape[0], int(max_distance), False)
    return torch.ops.geoembodied.paged_attention_step(q, k, v, *pools, table, positions, bias, int(max_distance), scale)
