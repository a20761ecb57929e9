"""Gated linear recurrence over packed point sequences.

    h, last = gated_recurrence(x, gate_a, gate_x, decay, ptr=ptr)        # [T, C], float32 [B, C]
    h, state = gated_recurrence_step(x, gate_a, gate_x, decay, state)    # one token per stream

mixes a whole cloud along its order with a state per channel: with ``r = sigmoid(gate_a)``,
``z = sigmoid(gate_x)`` and ``log a = -rate * softplus(decay) * r``,

    h_t = a_t * h_{t-1} + sqrt(1 - a_t ** 2) * z_t * x_t,

so a channel keeps its scale whatever it forgets.  The scan runs over all chunks of all sequences at
once, in float32 whatever the inputs' type; the backward forms the states again from the chunks'
first ones instead of reading the rounded outputs.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from gdl_amd import _native as _nat
from gdl_amd.csrc import (
    gated_recurrence_backward_hip,
    gated_recurrence_forward_hip,
    gated_recurrence_step_hip,
    recurrence_packets_hip,
)


# ═══════════════════════════════════════════════════════════════════
# Custom ops: what everything but plain eager execution uses (_native.plain_eager)
# ═══════════════════════════════════════════════════════════════════


@torch.library.custom_op("geoembodied::gated_recurrence", mutates_args=())
def _recurrence_op(x: Tensor, gate_a: Tensor, gate_x: Tensor, decay: Tensor, state: Optional[Tensor], ptr: Optional[Tensor],
                   reverse: bool, rate: float) -> Tuple[Tensor, Tensor, Tensor]:
    return gated_recurrence_forward_hip(x, gate_a, gate_x, decay, ptr, state, reverse, rate, True)


def _carry_size(tokens, channels):
    """geo_recurrence_carry_size (0 of no tokens or channels), of symbolic sizes too."""
    return (tokens + 63) // 64 * ((channels + 3) // 4 * 4)


@_recurrence_op.register_fake
def _(x, gate_a, gate_x, decay, state, ptr, reverse, rate):
    T, C = x.shape
    last = x.new_empty((1 if ptr is None else ptr.shape[0] - 1, C), dtype=torch.float32)
    return x.new_empty(x.shape), last, x.new_empty(_carry_size(T, C), dtype=torch.float32)


@torch.library.custom_op("geoembodied::gated_recurrence_backward", mutates_args=())
def _recurrence_backward_op(dh: Optional[Tensor], dlast: Optional[Tensor], carry: Tensor, x: Tensor, gate_a: Tensor,
                            gate_x: Tensor, decay: Tensor, state: Optional[Tensor], ptr: Optional[Tensor], reverse: bool,
                            rate: float) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    *grads, dstate = gated_recurrence_backward_hip(dh, dlast, carry, x, gate_a, gate_x, decay, ptr, state, reverse, rate)
    return (*grads, carry.new_empty(0) if dstate is None else dstate)


@_recurrence_backward_op.register_fake
def _(dh, dlast, carry, x, gate_a, gate_x, decay, state, ptr, reverse, rate):
    return (*(x.new_empty(x.shape) for _ in range(3)), carry.new_empty(decay.shape),
            carry.new_empty(0 if state is None else state.shape))


def _recurrence_setup(ctx, inputs, output) -> None:
    x, gate_a, gate_x, decay, state, ptr, *ctx.rest = inputs
    ctx.save_for_backward(x, gate_a, gate_x, decay, state, ptr, output[2])
    ctx.set_materialize_grads(False)


def _recurrence_grads(ctx, dh, dlast, dcarry):
    x, gate_a, gate_x, decay, state, ptr, carry = ctx.saved_tensors
    _nat.no_tangents("gated_recurrence backward", dh, dlast, x, gate_a, gate_x, decay, state)
    dx, dga, dgx, ddecay, dstate = torch.ops.geoembodied.gated_recurrence_backward(dh, dlast, carry, x, gate_a, gate_x, decay,
                                                                                   state, ptr, *ctx.rest)
    return (dx, dga, dgx, ddecay.to(decay.dtype), None if state is None else dstate.to(state.dtype), None, None, None)


_recurrence_op.register_autograd(_recurrence_grads, setup_context=_recurrence_setup)


@torch.library.custom_op("geoembodied::gated_recurrence_step", mutates_args=())
def _step_op(x: Tensor, gate_a: Tensor, gate_x: Tensor, decay: Tensor, state: Tensor, positions: Optional[Tensor],
             rate: float) -> Tuple[Tensor, Tensor]:
    return gated_recurrence_step_hip(x, gate_a, gate_x, decay, state, positions, rate)


@_step_op.register_fake
def _(x, gate_a, gate_x, decay, state, positions, rate):
    return x.new_empty(x.shape), state.new_empty(state.shape)


@torch.library.custom_op("geoembodied::recurrence_packets", mutates_args=())
def _packets_op(ptr: Tensor, start: Tensor, state: Tensor) -> Tuple[Tensor, Tensor]:
    return recurrence_packets_hip(ptr, start, state)


@_packets_op.register_fake
def _(ptr, start, state):
    B, C = state.shape
    return ptr.new_empty(2 * B, dtype=torch.int64), state.new_empty((2 * B - 1, C), dtype=torch.float32)


class _GatedRecurrence(torch.autograd.Function):
    """Eager mode: the op's kernels called directly, without the custom-op layers."""

    @staticmethod
    def forward(ctx, x, gate_a, gate_x, decay, state, ptr, reverse, rate):
        h, last, carry = gated_recurrence_forward_hip(x, gate_a, gate_x, decay, ptr, state, reverse, rate, True)
        ctx.save_for_backward(x, gate_a, gate_x, decay, state, ptr, carry)
        ctx.rest = (reverse, rate)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        x, gate_a, gate_x, decay, state, ptr, carry = ctx.saved_tensors
        if (dh is None or _nat.plain_eager(dh)) and (dlast is None or _nat.plain_eager(dlast)):
            dx, dga, dgx, ddecay, dstate = gated_recurrence_backward_hip(dh, dlast, carry, x, gate_a, gate_x, decay, ptr,
                                                                         state, *ctx.rest)
            return (dx, dga, dgx, ddecay.to(decay.dtype), None if dstate is None else dstate.to(state.dtype), None, None,
                    None)
        return _recurrence_grads(ctx, dh, dlast, None)


def _check(name: str, x: Tensor, gate_a: Tensor, gate_x: Tensor, decay: Tensor) -> None:
    shape = x.shape
    if len(shape) != 2 or gate_a.shape != shape or gate_x.shape != shape or decay.dim() != 1 or decay.shape[0] != shape[1]:
        raise ValueError(f"{name}: x, gate_a and gate_x [T, C], decay [C]; got {tuple(x.shape)}, {tuple(gate_a.shape)}, "
                         f"{tuple(gate_x.shape)}, {tuple(decay.shape)}")
    if not decay.dtype.is_floating_point:
        raise TypeError(f"{name}: decay must be a floating type, got {decay.dtype}")


def gated_recurrence(
    x: Tensor,
    gate_a: Tensor,
    gate_x: Tensor,
    decay: Tensor,
    *,
    ptr: Optional[Tensor] = None,
    state: Optional[Tensor] = None,
    reverse: bool = False,
    rate: float = 8.0,
) -> Tuple[Tensor, Tensor]:
    """The recurrence over packed sequences.

    Args:
        x, gate_a, gate_x: [T, C] of one type, float32, bfloat16 or float16; rows may be strided.
        decay: [C], any floating type.
        ptr: int64 [B + 1] ascending offsets of the sequences; None: one sequence.
        state: [B, C] states before the first tokens; None: 0.
        reverse: from each sequence's last token to its first.
        rate: positive; scales the decay.

    Returns:
        (h [T, C] of x's type, last float32 [B, C]: the state after each sequence's last token in scan
        order, its ``state`` where it has no tokens).  Tokens of no sequence give 0.
    """
    _check("gated_recurrence", x, gate_a, gate_x, decay)
    batch = 1 if ptr is None else ptr.numel() - 1
    if ptr is not None and (ptr.dim() != 1 or batch < 1):
        raise ValueError(f"gated_recurrence: ptr must be [B + 1] with at least one sequence, got {tuple(ptr.shape)}")
    if state is not None and (state.shape != (batch, x.shape[1]) or not state.dtype.is_floating_point):
        raise ValueError(f"gated_recurrence: state must be [{batch}, {x.shape[1]}], got {state.dtype} {tuple(state.shape)}")
    rate = float(rate)
    if not rate > 0:
        raise ValueError(f"gated_recurrence: rate {rate} must be positive")
    tensors = x, gate_a, gate_x, decay, state, ptr
    if not _nat.plain_call(*tensors):
        _nat.no_tangents("gated_recurrence", *tensors)
        h, last, _ = torch.ops.geoembodied.gated_recurrence(*tensors, bool(reverse), rate)
        return h, last
    if torch.is_grad_enabled() and (x.requires_grad or gate_a.requires_grad or gate_x.requires_grad or decay.requires_grad
                                    or (state is not None and state.requires_grad)):
        return _GatedRecurrence.apply(*tensors, bool(reverse), rate)
    h, last, _ = gated_recurrence_forward_hip(x, gate_a, gate_x, decay, ptr, state, bool(reverse), rate, False)
    return h, last


def packets_as_sequences(ptr: Tensor, start: Tensor, state: Tensor) -> Tuple[Tensor, Tensor]:
    """Packets of streams, ``ptr`` [B + 1] from the positions ``start`` [B] on behind the states [B, C], as the
    ``ptr`` [2 B] and ``state`` of 2 B - 1 sequences of ``gated_recurrence``: number 2 b holds stream b's tokens from
    position 0 on and begins from 0 where that position is in the packet, those between hold tokens at
    negative positions.  ``last[::2]`` are then the streams' states, which tokens at negative positions leave as they were."""
    batch = start.numel()
    if batch < 1 or start.dim() != 1 or ptr.shape != (batch + 1,) or state.dim() != 2 or len(state) != batch:
        raise ValueError(f"packets_as_sequences: ptr [B + 1], start [B] and state [B, C] of one stream at least, got {tuple(ptr.shape)}, "
                         f"{tuple(start.shape)}, {tuple(state.shape)}")
    if _nat.plain_call(ptr, start, state):
        return recurrence_packets_hip(ptr, start, state)
    return torch.ops.geoembodied.recurrence_packets(ptr, start, state)


def gated_recurrence_step(
    x: Tensor,
    gate_a: Tensor,
    gate_x: Tensor,
    decay: Tensor,
    state: Tensor,
    *,
    positions: Optional[Tensor] = None,
    rate: float = 8.0,
) -> Tuple[Tensor, Tensor]:
    """One token of each stream: x, gates [B, C] and the streams' float32 states [B, C] to
    (h [B, C] of x's type, new states float32 [B, C]).  No gradients.

    With ``positions`` (int64 [B], as ``window_attention_step`` takes them) a stream at position 0 begins
    from 0 whatever its state holds, and one at a negative position keeps its state and gives 0.
    """
    _check("gated_recurrence_step", x, gate_a, gate_x, decay)
    if state.shape != x.shape or state.dtype is not torch.float32:
        raise ValueError(f"gated_recurrence_step: state must be float32 {tuple(x.shape)}, got {state.dtype} {tuple(state.shape)}")
    if positions is not None and (positions.shape != x.shape[:1] or positions.dtype.is_floating_point):
        raise ValueError(f"gated_recurrence_step: positions int64 [{x.shape[0]}], got {positions.dtype} {tuple(positions.shape)}")
    if not rate > 0:
        raise ValueError(f"gated_recurrence_step: rate {rate} must be positive")
    if torch.is_grad_enabled() and (x.requires_grad or gate_a.requires_grad or gate_x.requires_grad or decay.requires_grad
                                    or state.requires_grad):
        raise RuntimeError("gated_recurrence_step has no backward: call it under torch.no_grad()")
    if _nat.plain_call(x, gate_a, gate_x, decay, state, positions):
        return gated_recurrence_step_hip(x, gate_a, gate_x, decay, state, positions, float(rate))
    _nat.no_tangents("gated_recurrence_step", x, gate_a, gate_x, decay, state)
    return torch.ops.geoembodied.gated_recurrence_step(x, gate_a, gate_x, decay, state, positions, float(rate))
