"""Attention within a window over packed point sequences.

    out = window_attention(q, k, v, (left, right), ptr=ptr, sinks=4, mask=valid, bias=table)

mixes clouds that are taken as sequences (points in scan order or along a space-filling curve):
token ``i`` sees the keys of its own sequence from ``i - left`` to ``i + right`` and the sequence's
first ``sinks`` tokens, as far as they lie at or before ``i + right``.  The softmax, the relative
position bias and every gradient (of ``q``, ``k``, ``v`` and the bias table) are computed tile by
tile on the matrix units; no score, weight or bias matrix is ever written.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from gdl_amd.csrc import window_attention_backward_hip, window_attention_forward_hip
from gdl_amd.functional.relative_bias import bucket_plan

_UNBOUNDED = 1 << 40


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, plan, ptr, mask, left, right, sinks, scale):
        out, lse = window_attention_forward_hip(q, k, v, left, right, sinks, scale, ptr, mask, bias, plan, True)
        ctx.save_for_backward(q, k, v, bias, out, lse, ptr, mask)
        ctx.rest = (plan, left, right, sinks, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, bias, out, lse, ptr, mask = ctx.saved_tensors
        plan, left, right, sinks, scale = ctx.rest
        dq, dk, dv, dbias = window_attention_backward_hip(grad, out, lse, q, k, v, left, right, sinks, scale, ptr, mask,
                                                          bias, plan)
        return dq, dk, dv, dbias, None, None, None, None, None, None, None


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
            two-sided unless ``window`` has no right side.
        max_distance: where the bias's last bucket begins (at most 1024).
        scale: of the scores; ``D ** -0.5`` by default.

    Returns:
        [T, H, D] of q's type; 0 for a token that sees no key.
    """
    left, right = window if isinstance(window, (tuple, list)) else (window, window)
    left, right = _reach("left", left), _reach("right", right)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"window_attention: q [T, H, D], k and v [T, Hk, D]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    d = q.shape[2]
    if not 1 <= d <= 128:
        raise ValueError(f"window_attention: head size {d} (from 1 to 128)")
    plan = None
    if bias is not None:
        if bias.dim() != 2 or bias.shape[1] != q.shape[1]:
            raise ValueError(f"window_attention: bias must be [buckets, {q.shape[1]}], got {tuple(bias.shape)}")
        plan = bucket_plan(bias.shape[0], int(max_distance), right != 0, q.device) + (int(max_distance),)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if d % 8:  # rows are read in pieces of 8 values: zeros beyond D change no score and no gradient
        q, k, v = (torch.nn.functional.pad(x, (0, 8 - d % 8)) for x in (q, k, v))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        out = _WindowAttention.apply(q, k, v, bias, plan, ptr, mask, left, right, int(sinks), scale)
    else:
        out, _ = window_attention_forward_hip(q, k, v, left, right, int(sinks), scale, ptr, mask, bias, plan, False)
    return out[..., :d] if d % 8 else out
