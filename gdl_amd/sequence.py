"""A block for point clouds taken as sequences, and the order to take them in.

    order = serial_order(pos, ptr)                       # Morton order within each cloud
    block = PointSequenceBlock(64, heads=4, window=64).cuda()
    y = block(x[order], ptr)                             # [T, C], training or inference
    cache = block.new_cache(B); y_t = block.step(x_t, positions, cache)   # causal: token by token

The block mixes along the order twice: over the whole cloud by ``gated_recurrence``, near by
``window_attention`` with a relative position bias, each behind a norm and added to its input.
``window=None`` attends to the whole stream; its cache keeps that in pages, in 8 bits if asked, and takes
packets of points too:

    cache = block.new_cache(B, torch.int8, tokens=100_000); y = block.extend(x, ptr, start, cache)
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch
from torch import Tensor, nn

from gdl_amd.functional.attention import WindowCache, window_attention, window_attention_step
from gdl_amd.functional.paged import PagedCache, paged_attention, paged_attention_step
from gdl_amd.functional.recurrence import gated_recurrence, gated_recurrence_step, packets_as_sequences


def serial_order(pos: Tensor, ptr: Optional[Tensor] = None) -> Tensor:
    """int64 [T]: the points of each cloud along the Morton curve of its bounding box (1024 cells an
    axis), the clouds in their order; points of one cell keep theirs."""
    if pos.dim() != 2 or pos.shape[1] != 3:
        raise ValueError(f"serial_order: pos must be [T, 3], got {tuple(pos.shape)}")
    T, dev = pos.shape[0], pos.device
    if ptr is None:
        ptr = torch.tensor([0, T], device=dev)
    clouds = ptr.numel() - 1
    cloud = torch.searchsorted(ptr[1:].contiguous(), torch.arange(T, device=dev), right=True).clamp(max=clouds - 1)
    index = cloud.unsqueeze(1).expand(-1, 3)
    low = pos.new_full((clouds, 3), torch.inf).scatter_reduce(0, index, pos, "amin")
    high = pos.new_full((clouds, 3), -torch.inf).scatter_reduce(0, index, pos, "amax")
    size = (high - low).amax(1, keepdim=True).clamp(min=torch.finfo(pos.dtype).tiny)
    cell = ((pos - low[cloud]) / size[cloud] * 1024).long().clamp(0, 1023)
    code = torch.zeros(T, dtype=torch.int64, device=dev)
    for bit in range(10):
        for axis in range(3):
            code |= (cell[:, axis] >> bit & 1) << (3 * bit + axis)
    return torch.argsort(cloud << 30 | code, stable=True)


@dataclass
class BlockCache:
    """What a causal block keeps of its streams: recurrence states [B, C], and the attention's window, or all
    of the streams in pages and the ``table`` (int32 [B, n]) that says which are whose."""

    state: Tensor
    window: Union[WindowCache, PagedCache]
    table: Optional[Tensor] = None


class PointSequenceBlock(nn.Module):
    """Gated recurrence and window attention over packed sequences ``[T, channels]``.

    Args:
        channels: width; ``channels / heads`` is the head size (a multiple of 8 up to 128 for ``step``).
        heads, kv_heads: query heads and the key heads that they share (all by default).
        window: tokens seen before a token, and behind it unless ``causal``; None for all.
        sinks: first tokens of a sequence that stay visible (of a window).
        buckets, max_distance: of the relative position bias.
        causal: tokens see earlier ones alone; else the recurrence runs both ways and its results are
            added.
    """

    def __init__(self, channels: int, heads: int, window: Optional[int], *, kv_heads: Optional[int] = None, sinks: int = 0,
                 buckets: int = 32, max_distance: int = 128, causal: bool = True):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channels % heads or heads % kv_heads:
            raise ValueError(f"PointSequenceBlock: {channels} channels, {heads} heads, {kv_heads} key heads do not divide")
        if window is None and sinks:
            raise ValueError(f"PointSequenceBlock: {sinks} first tokens of no window")
        self.channels, self.heads, self.kv_heads, self.head_dim = channels, heads, kv_heads, channels // heads
        self.window, self.sinks, self.max_distance, self.causal = window, sinks, max_distance, causal
        self.scan_norm, self.attend_norm = nn.LayerNorm(channels), nn.LayerNorm(channels)
        self.scan_in, self.scan_out = nn.Linear(channels, 3 * channels), nn.Linear(channels, channels)
        # a half-open gate keeps from 0.9 to 0.999 of a state: log a = -8 softplus(decay) / 2
        keep = torch.linspace(0.9, 0.999, channels, dtype=torch.float64)
        self.decay = nn.Parameter(torch.log(torch.expm1(-torch.log(keep) / 4)).float())
        self.attend_in = nn.Linear(channels, (heads + 2 * kv_heads) * self.head_dim)
        self.attend_out = nn.Linear(channels, channels)
        self.bias = nn.Parameter(torch.zeros(buckets, heads))

    def _split(self, x: Tensor):
        """q, k, v as views of the projection of x [N, channels]."""
        y = self.attend_in(self.attend_norm(x)).unflatten(1, (self.heads + 2 * self.kv_heads, self.head_dim))
        return y.split((self.heads, self.kv_heads, self.kv_heads), 1)

    def forward(self, x: Tensor, ptr: Optional[Tensor] = None, mask: Optional[Tensor] = None) -> Tensor:
        """x [T, channels] of sequences ``ptr``.  Points whose ``mask`` (bool [T]) is False count for
        nothing: no other point's row depends on them, whatever they hold, and their own mean nothing."""
        if mask is not None:
            hidden = ~mask.unsqueeze(1)
            x = x.masked_fill(hidden, 0.0)  # NaN among them would reach the weights' gradients
        parts = self.scan_in(self.scan_norm(x)).split(self.channels, 1)
        if mask is not None:  # a closed gate hands the state on as it is
            parts = parts[0], parts[1].masked_fill(hidden, -torch.inf), parts[2]
        h, _ = gated_recurrence(*parts, self.decay, ptr=ptr)
        if not self.causal:
            h = h + gated_recurrence(*parts, self.decay, ptr=ptr, reverse=True)[0]
        x = x + self.scan_out(h)
        reach = -1 if self.window is None else self.window
        out = window_attention(*self._split(x), (reach, 0 if self.causal else reach), sinks=self.sinks, ptr=ptr,
                               mask=mask, bias=self.bias, max_distance=self.max_distance)
        return x + self.attend_out(out.flatten(1))

    def new_cache(self, batch: int, dtype: Optional[torch.dtype] = None, *, tokens: Optional[int] = None,
                  page: int = 64) -> BlockCache:
        """The cache of ``batch`` streams without tokens.  Without a window it has pages for ``tokens`` tokens of each
        stream, of the block's type, torch.int8 or torch.float8_e4m3fn; to share a pool among streams of
        unequal lengths, make a ``BlockCache`` of your own ``PagedCache`` and table."""
        if not self.causal:
            raise ValueError("PointSequenceBlock: only a causal block answers token by token")
        dev = self.decay.device
        if self.window is None:
            if tokens is None or tokens < 1 or batch < 1 or page < 1:
                raise ValueError("PointSequenceBlock: a cache without a window is for a number of tokens, got "
                                 f"{tokens} for {batch} streams in pages of {page}")
            each = -(-tokens // page)
            pool = PagedCache.empty(batch * each, self.kv_heads, self.head_dim, page=page, dtype=dtype or self.attend_in.weight.dtype,
                                    device=dev)
            table = torch.arange(batch * each, dtype=torch.int32, device=dev).view(batch, each)
            return BlockCache(torch.zeros(batch, self.channels, device=dev), pool, table)
        if tokens is not None:
            raise ValueError("PointSequenceBlock: a window's cache has no number of tokens")
        window = WindowCache.empty(batch, self.kv_heads, self.head_dim, self.window, sinks=self.sinks,
                                   dtype=dtype or self.attend_in.weight.dtype, device=dev)
        return BlockCache(torch.zeros(batch, self.channels, device=dev), window)

    @torch.no_grad()
    def step(self, x: Tensor, positions: Tensor, cache: BlockCache) -> Tensor:
        """One token x [B, channels] of each stream at ``positions`` (int64 [B], from 0), which ``cache``
        then holds; the forward's row for it.  A stream at position 0 begins anew; one at a negative
        position has no token: the cache keeps what it holds of it, and its row means nothing."""
        parts = self.scan_in(self.scan_norm(x)).split(self.channels, 1)
        h, state = gated_recurrence_step(*parts, self.decay, cache.state, positions=positions)
        x = x + self.scan_out(h)
        near = dict(bias=self.bias, max_distance=self.max_distance)
        if cache.table is None:
            out = window_attention_step(*self._split(x), cache.window, positions, **near)
        else:
            out = paged_attention_step(*self._split(x), cache.window, cache.table, positions, **near)
        cache.state = state  # a call that is refused above leaves the cache as it was
        return x + self.attend_out(out.flatten(1))

    @torch.no_grad()
    def extend(self, x: Tensor, ptr: Tensor, start: Tensor, cache: BlockCache) -> Tensor:
        """New tokens x [T, channels] of the streams, packed (``ptr`` int64 [B + 1]), from the positions ``start``
        (int64 [B]) on, which ``cache`` then holds; the forward's rows for them.  For a block without a window.
        A stream begins anew with its token at position 0; one without tokens from there on is left alone.  Tokens at
        negative positions are none, as in ``step``: the cache keeps nothing of them, and their rows mean nothing."""
        if cache.table is None:
            raise ValueError("PointSequenceBlock: only a block without a window takes several tokens of a stream")
        if ptr.shape != (cache.state.shape[0] + 1,) or start.shape != (cache.state.shape[0],):
            raise ValueError(f"PointSequenceBlock: ptr and start of {cache.state.shape[0]} streams, got {tuple(ptr.shape)}, "
                             f"{tuple(start.shape)}")
        parts = self.scan_in(self.scan_norm(x)).split(self.channels, 1)
        pieces, before = packets_as_sequences(ptr, start, cache.state)
        h, state = gated_recurrence(*parts, self.decay, ptr=pieces, state=before)
        x = x + self.scan_out(h)
        q, k, v = self._split(x)
        cache.window.write(k, v, cache.table, ptr, start)
        out = paged_attention(q, cache.window, cache.table, ptr, start, bias=self.bias, max_distance=self.max_distance)
        cache.state = state[::2].contiguous()  # as a caller may view it
        return x + self.attend_out(out.flatten(1))
