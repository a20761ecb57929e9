"""Attention within a window over packed point sequences.

    out = window_attention(q, k, v, (left, right), ptr=ptr, sinks=4, mask=valid, bias=table)

mixes clouds that are taken as sequences (points in scan order or along a space-filling curve):
token ``i`` sees the keys of its own sequence from ``i - left`` to ``i + right`` and the sequence's
first ``sinks`` tokens, as far as they lie at or before ``i + right``.  The softmax, the relative
position bias and every gradient (of ``q``, ``k``, ``v`` and the bias table) are computed tile by
tile on the matrix units; no score, weight or bias matrix is ever written.

For streams that are answered token by token ``WindowCache`` keeps what a causal window
``(left, 0)`` still reaches, and ``window_attention_step`` adds one token to it and attends:

    cache = WindowCache.empty(B, Hk, D, left, sinks=4, dtype=torch.bfloat16, device="cuda")
    cache.fill(k, v, ptr)                                     # the tokens that are there already
    out = window_attention_step(q, k, v, cache, positions)    # [B, H, D], one token per stream
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from gdl_amd import _native as _nat
from gdl_amd.csrc import (
    window_attention_backward_hip,
    window_attention_forward_hip,
    window_attention_step_hip,
    window_cache_fill_hip,
)
from gdl_amd.functional.relative_bias import bucket_plan, check_buckets

_UNBOUNDED = 1 << 40


def _plan(bias: Optional[Tensor], max_distance: int, two_sided: bool):
    """(bucket of each distance, spans, max_distance) of a bias table on its device, None without one."""
    if bias is None:
        return None
    return bucket_plan(bias.shape[0], max_distance, two_sided, bias.device) + (max_distance,)


# ═══════════════════════════════════════════════════════════════════
# Custom ops: what everything but plain eager execution uses (_native.plain_eager)
# ═══════════════════════════════════════════════════════════════════


@torch.library.custom_op("geoembodied::window_attention", mutates_args=())
def _attention_op(q: Tensor, k: Tensor, v: Tensor, bias: Optional[Tensor], ptr: Optional[Tensor], mask: Optional[Tensor],
                  left: int, right: int, sinks: int, max_distance: int, scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    out, rest, lse = window_attention_forward_hip(q, k, v, left, right, sinks, scale, ptr, mask, bias,
                                                  _plan(bias, max_distance, right != 0), True)
    return out, out.new_empty(0) if rest is None else rest, lse


@_attention_op.register_fake
def _(q, k, v, bias, ptr, mask, left, right, sinks, max_distance, scale):
    rest = q.new_empty(0) if q.dtype is torch.float32 else q.new_empty(q.shape)
    return q.new_empty(q.shape), rest, q.new_empty((1 if bias is None else 2, q.shape[1], q.shape[0]), dtype=torch.float32)


@torch.library.custom_op("geoembodied::window_attention_backward", mutates_args=())
def _attention_backward_op(grad: Tensor, out: Tensor, rest: Tensor, lse: Tensor, q: Tensor, k: Tensor, v: Tensor,
                           bias: Optional[Tensor], ptr: Optional[Tensor], mask: Optional[Tensor], left: int, right: int,
                           sinks: int, max_distance: int, scale: float, need_q: bool, need_kv: bool,
                           need_bias: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    grads = window_attention_backward_hip(
        grad, out, rest if rest.numel() else None, lse, q, k, v, left, right, sinks, scale, ptr, mask, bias,
        _plan(bias, max_distance, right != 0), need_q, need_kv, need_bias)
    return tuple(lse.new_empty(0) if g is None else g for g in grads)


@_attention_backward_op.register_fake
def _(grad, out, rest, lse, q, k, v, bias, ptr, mask, left, right, sinks, max_distance, scale, need_q, need_kv, need_bias):
    needs = need_q, need_kv, need_kv, need_bias and bias is not None
    return tuple(t.new_empty(t.shape) if need else lse.new_empty(0) for t, need in zip((q, k, v, bias), needs))


def _attention_setup(ctx, inputs, output) -> None:
    q, k, v, bias, ptr, mask, *ctx.sizes = inputs
    ctx.save_for_backward(q, k, v, bias, *output, ptr, mask)


def _needs(ctx):
    """Whether the gradients of q, of k or v, and of the bias are needed."""
    q, k, v, bias = ctx.needs_input_grad[:4]
    return q, k or v, bias


def _attention_grads(ctx, grad, grad_rest, grad_lse):
    q, k, v, bias, out, rest, lse, ptr, mask = ctx.saved_tensors
    _nat.no_tangents("window_attention backward", grad, q, k, v, bias)
    needs = _needs(ctx)
    grads = torch.ops.geoembodied.window_attention_backward(
        grad, out, out.new_empty(0) if rest is None else rest, lse, q, k, v, bias, ptr, mask, *ctx.sizes, *needs)
    grads = (g if need else None for g, need in zip(grads, (needs[0], needs[1], needs[1], needs[2])))
    return (*grads, None, None, None, None, None, None, None)


_attention_op.register_autograd(_attention_grads, setup_context=_attention_setup)


@torch.library.custom_op("geoembodied::window_attention_step", mutates_args=("k_cache", "v_cache"))
def _step_op(q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, positions: Tensor, bias: Optional[Tensor],
             sinks: int, max_distance: int, scale: float) -> Tensor:
    return window_attention_step_hip(q, k, v, k_cache, v_cache, sinks, positions, scale, bias,
                                     _plan(bias, max_distance, False))


@_step_op.register_fake
def _(q, k, v, k_cache, v_cache, positions, bias, sinks, max_distance, scale):
    return q.new_empty(q.shape)


@torch.library.custom_op("geoembodied::window_cache_fill", mutates_args=("k_cache", "v_cache"))
def _fill_op(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, sinks: int, ptr: Optional[Tensor],
             start: Optional[Tensor]) -> None:
    window_cache_fill_hip(k, v, k_cache, v_cache, sinks, ptr, start)


@_fill_op.register_fake
def _(k, v, k_cache, v_cache, sinks, ptr, start):
    return None


class _WindowAttention(torch.autograd.Function):
    """Eager mode: the op's kernels called directly, without the custom-op layers."""

    @staticmethod
    def forward(ctx, q, k, v, bias, ptr, mask, left, right, sinks, max_distance, scale):
        plan = _plan(bias, max_distance, right != 0)
        out, rest, lse = window_attention_forward_hip(q, k, v, left, right, sinks, scale, ptr, mask, bias, plan, True)
        ctx.save_for_backward(q, k, v, bias, out, rest, lse, ptr, mask)
        ctx.sizes, ctx.plan = (left, right, sinks, max_distance, scale), plan
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if not _nat.plain_eager(grad):
            return _attention_grads(ctx, grad, None, None)
        q, k, v, bias, out, rest, lse, ptr, mask = ctx.saved_tensors
        left, right, sinks, _, scale = ctx.sizes
        grads = window_attention_backward_hip(grad, out, rest, lse, q, k, v, left, right, sinks, scale, ptr, mask, bias, ctx.plan,
                                              *_needs(ctx))
        return (*grads, None, None, None, None, None, None, None)


def _reach(name: str, n: Optional[int]) -> int:
    if n is None or n == -1:
        return _UNBOUNDED
    n = int(n)
    if n < 0:
        raise ValueError(f"window_attention: window's {name} is {n} (a count of tokens, -1 or None for all)")
    return n


def window_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    window: Union[int, Tuple[Optional[int], Optional[int]]],
    *,
    sinks: int = 0,
    ptr: Optional[Tensor] = None,
    mask: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    max_distance: int = 128,
    scale: Optional[float] = None,
) -> Tensor:
    """Softmax attention of ``q [T, H, D]`` over ``k, v [T, Hk, D]`` within a window.

    Args:
        q, k, v: float32, bfloat16 or float16; ``H`` a multiple of ``Hk`` (query head ``h`` reads key
            head ``h // (H / Hk)``), ``D`` up to 128.  Token and head strides are free.
        window: ``(left, right)`` tokens that are seen before and after a token (its own aside), one
            number for both; -1 or None for all.  ``(n, 0)`` is causal.
        sinks: first tokens of each sequence (at most 256) that stay visible left of the window.
        ptr: int64 [B + 1] ascending offsets of the sequences in the T tokens; None: one sequence.
            Tokens outside ``ptr[0] .. ptr[B]`` see nothing.
        mask: bool [T], False keys are seen by no one (and may hold anything).
        bias: [buckets, H] learned relative position bias, added to the scores (``relative_buckets``);
            two-sided unless ``window`` has no right side.  The first call with a number of buckets and
            a ``max_distance`` copies their table to the device and cannot be captured into a graph.
        max_distance: where the bias's last bucket begins (at most 1024).
        scale: of the scores; ``D ** -0.5`` by default.

    Returns:
        [T, H, D] of q's type; 0 for a token that sees no key, NaN for one that sees keys with scores
        of -inf alone.
    """
    left, right = window if isinstance(window, (tuple, list)) else (window, window)
    left, right = _reach("left", left), _reach("right", right)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"window_attention: q [T, H, D], k and v [T, Hk, D]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    d = q.shape[2]
    if not 1 <= d <= 128:
        raise ValueError(f"window_attention: head size {d} (from 1 to 128)")
    if bias is not None and (bias.dim() != 2 or bias.shape[1] != q.shape[1]):
        raise ValueError(f"window_attention: bias must be [buckets, {q.shape[1]}], got {tuple(bias.shape)}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if d % 8:  # rows are read in pieces of 8 values: zeros beyond D change no score and no gradient
        q, k, v = (torch.nn.functional.pad(x, (0, 8 - d % 8)) for x in (q, k, v))
    sizes = left, right, int(sinks), int(max_distance), scale
    if not _nat.plain_call(q, k, v, bias, ptr, mask):
        _nat.no_tangents("window_attention", q, k, v, bias)
        if bias is not None:
            check_buckets(bias.shape[0], sizes[3], right != 0)
        out, _, _ = torch.ops.geoembodied.window_attention(q, k, v, bias, ptr, mask, *sizes)
    elif torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                      or (bias is not None and bias.requires_grad)):
        out = _WindowAttention.apply(q, k, v, bias, ptr, mask, *sizes)
    else:
        out, _, _ = window_attention_forward_hip(q, k, v, left, right, sizes[2], scale, ptr, mask, bias,
                                                 _plan(bias, sizes[3], right != 0), False)
    return out[..., :d] if d % 8 else out


def _apart(t: Tensor) -> bool:
    """No two heads of two streams of t [B, Hk, slots, D], each head's slots adjoining, share memory."""
    reach = t.shape[2] * t.shape[3]
    for stride, n in sorted((t.stride(n), t.shape[n]) for n in (0, 1) if t.shape[n] > 1):
        if stride < reach:
            return False
        reach += stride * (n - 1)
    return True


class WindowCache:
    """Keys and values of streams that a causal window reaches: ``k, v [B, Hk, sinks + ring, D]``.

    Token ``j`` of a stream lies in slot ``j`` for ``j < sinks``, else in slot
    ``sinks + (j - sinks) % ring``, ``ring`` = left + 1 tokens of the window.  The object holds the two
    tensors (given ones are used as they are); calls on it are ordered by the caller's stream.
    """

    def __init__(self, k: Tensor, v: Tensor, *, sinks: int = 0):
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"WindowCache: k and v [B, Hk, sinks + ring, D], got {tuple(k.shape)}, {tuple(v.shape)}")
        if not 0 <= sinks < k.shape[2]:
            raise ValueError(f"WindowCache: {sinks} of {k.shape[2]} slots for first tokens (at least one is the window's)")
        if k.shape[3] % 8 or not 8 <= k.shape[3] <= 128:
            raise ValueError(f"WindowCache: head size {k.shape[3]} (a multiple of 8 up to 128)")
        for t in (k, v):
            size = t.element_size()
            at = t.data_ptr() if _nat.plain_eager(t) else 0  # traced: looked at when the program runs
            if t.stride(3) != 1 or t.stride(2) != t.shape[3] or any(x % 16 for x in (at, t.stride(0) * size, t.stride(1) * size)):
                raise ValueError("WindowCache: a head's slots must adjoin, on multiples of 16 bytes")
            if not _apart(t):
                raise ValueError(f"WindowCache: streams or heads share memory (strides {t.stride()} of {tuple(t.shape)})")
        if k.numel() and _nat.plain_eager(k) and _nat.plain_eager(v) and k.data_ptr() == v.data_ptr():
            raise ValueError("WindowCache: k and v are the same memory")
        self.k, self.v, self.sinks = k, v, int(sinks)
        self.left = k.shape[2] - self.sinks - 1

    @classmethod
    def empty(cls, batch: int, kv_heads: int, head_dim: int, left: int, *, sinks: int = 0,
              dtype: torch.dtype = torch.float32, device="cuda") -> "WindowCache":
        """A cache of no tokens for a window of ``left`` tokens and the current one."""
        if left < 0 or sinks < 0:
            raise ValueError(f"WindowCache: window of {left} tokens, {sinks} first tokens")
        k, v = (torch.empty(batch, kv_heads, sinks + left + 1, head_dim, dtype=dtype, device=device) for _ in range(2))
        return cls(k, v, sinks=sinks)

    def fill(self, k: Tensor, v: Tensor, ptr: Optional[Tensor] = None, start: Optional[Tensor] = None) -> None:
        """Tokens ``k, v [T, Hk, D]`` of packed sequences (``ptr`` int64 [B + 1]; None: one stream) into the
        cache; sequence ``b`` begins at position ``start[b]`` (0)."""
        batch, heads, _, d = self.k.shape
        if k.dim() != 3 or v.shape != k.shape or k.shape[1:] != (heads, d):
            raise ValueError(f"WindowCache.fill: k and v [T, {heads}, {d}], got {tuple(k.shape)}, {tuple(v.shape)}")
        if (ptr is None and batch != 1) or (ptr is not None and ptr.shape != (batch + 1,)):
            raise ValueError(f"WindowCache.fill: ptr [{batch + 1}] of {batch} streams")
        if start is not None and start.shape != (batch,):
            raise ValueError(f"WindowCache.fill: start [{batch}], got {tuple(start.shape)}")
        if _nat.plain_call(k, v, self.k, self.v, ptr, start):
            window_cache_fill_hip(k, v, self.k, self.v, self.sinks, ptr, start)
        else:
            _nat.no_tangents("WindowCache.fill", k, v)
            torch.ops.geoembodied.window_cache_fill(k, v, self.k, self.v, self.sinks, ptr, start)


def window_attention_step(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    cache: WindowCache,
    positions: Tensor,
    *,
    bias: Optional[Tensor] = None,
    max_distance: int = 128,
    scale: Optional[float] = None,
) -> Tensor:
    """One token of each stream: ``k, v [B, Hk, D]`` go into the cache at ``positions`` (int64 [B], from
    0), and ``q [B, H, D]`` attends to the tokens that the cache then holds.

    The result is ``window_attention``'s for the last token of such streams with the window
    ``(cache.left, 0)`` and ``cache.sinks`` first tokens.  A stream at a negative position is left
    alone (its row is 0).  No gradients.  ``bias`` is one-sided.
    """
    batch, hk, _, d = cache.k.shape
    if q.dim() != 3 or q.shape[0] != batch or q.shape[2] != d or k.shape != (batch, hk, d) or v.shape != k.shape:
        raise ValueError(f"window_attention_step: q [{batch}, H, {d}], k and v [{batch}, {hk}, {d}]; got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.shape[1] < 1 or q.shape[1] % hk:
        raise ValueError(f"window_attention_step: {q.shape[1]} heads are no multiple of {hk} key heads")
    if positions.shape != (batch,) or positions.dtype.is_floating_point:
        raise ValueError(f"window_attention_step: positions int64 [{batch}], got {positions.dtype} {tuple(positions.shape)}")
    if bias is not None and (bias.dim() != 2 or bias.shape[1] != q.shape[1]):
        raise ValueError(f"window_attention_step: bias must be [buckets, {q.shape[1]}], got {tuple(bias.shape)}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        raise RuntimeError("window_attention_step has no backward: call it under torch.no_grad()")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if _nat.plain_call(q, k, v, cache.k, cache.v, positions, bias):
        return window_attention_step_hip(q, k, v, cache.k, cache.v, cache.sinks, positions, scale, bias,
                                         _plan(bias, int(max_distance), False))
    _nat.no_tangents("window_attention_step", q, k, v, bias)
    if bias is not None:
        check_buckets(bias.shape[0], int(max_distance), False)
    return torch.ops.geoembodied.window_attention_step(q, k, v, cache.k, cache.v, positions, bias, cache.sinks,
                                                       int(max_distance), scale)
