"""Buckets of the relative position bias that ``window_attention`` and ``window_attention_step`` take.

A bias table ``[buckets, heads]`` is learned for the distance ``d`` = key position - query position,
which is first mapped to a bucket: one bucket for each of the nearest distances, then logarithmically
wider ones up to ``max_distance``, beyond which all share the last.  One-sided (keys at or before
the query: ``d <= 0``, a later key counts as distance 0) all buckets serve the past; two-sided the
second half of the buckets serves ``d > 0``.

With ``half`` the buckets of one side, ``exact = half // 2``, and ``n = |d|``: bucket ``n`` for
``n < exact``, else ``exact +`` the number of ``k`` in ``1 .. half - exact - 1`` with
``n >= exact ** (1 - k / (half - exact)) * max_distance ** (k / (half - exact))``, decided in whole
numbers (both sides to the power ``half - exact``), so no logarithm's rounding moves a boundary.
"""

from __future__ import annotations

import functools
from typing import Tuple

import torch
from torch import Tensor

MAX_BUCKETS = 256
MAX_DISTANCE = 1024


def check_buckets(buckets: int, max_distance: int, two_sided: bool) -> None:
    least = 4 if two_sided else 2
    if not least <= buckets <= MAX_BUCKETS or (two_sided and buckets % 2):
        raise ValueError(f"relative bias: {buckets} buckets (from {least} to {MAX_BUCKETS}, an even number "
                         "for both sides)")
    half = buckets // 2 if two_sided else buckets
    if not half // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"relative bias: max_distance {max_distance} (above {half // 2}, the distances with a "
                         f"bucket of their own, up to {MAX_DISTANCE})")


@functools.lru_cache(maxsize=None)
def _table(buckets: int, max_distance: int, two_sided: bool) -> Tuple[Tuple[int, ...], Tuple[Tuple[int, int], ...]]:
    """The bucket of each distance -max_distance .. max_distance, and for each bucket the places
    first <= x < end of that list which hold it."""
    check_buckets(buckets, max_distance, two_sided)
    half = buckets // 2 if two_sided else buckets
    exact = half // 2
    power = half - exact
    bounds = [exact ** (power - k) * max_distance ** k for k in range(1, power)]
    side = [n if n < exact else exact + sum(n ** power >= b for b in bounds) for n in range(max_distance + 1)]
    lut = side[:0:-1] + [side[0]] + ([half + b for b in side[1:]] if two_sided else [side[0]] * max_distance)
    places = {b: [] for b in range(buckets)}
    for x, b in enumerate(lut):
        places[b].append(x)
    spans = tuple((p[0], p[-1] + 1) if p else (0, 0) for p in places.values())
    return tuple(lut), spans


@functools.lru_cache(maxsize=None)
def bucket_plan(buckets: int, max_distance: int, two_sided: bool, device: torch.device) -> Tuple[Tensor, Tensor]:
    """(bucket of each distance int32 [2 max_distance + 1], spans int32 [buckets, 2]) on a device,
    laid out once per configuration, by a copy that the host waits for."""
    lut, spans = _table(buckets, max_distance, two_sided)
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"relative bias: a graph cannot capture the first call with {buckets} buckets up to distance "
                           f"{max_distance} (its table is copied to the device): make one call before the capture")
    return (torch.tensor(lut, dtype=torch.int32, device=device),
            torch.tensor(spans, dtype=torch.int32, device=device))


def relative_buckets(distance: Tensor, buckets: int, max_distance: int = 128, two_sided: bool = True) -> Tensor:
    """Bucket of each distance (key position - query position), int64 of ``distance``'s shape."""
    if distance.dtype.is_floating_point or distance.dtype is torch.bool:
        raise TypeError(f"relative_buckets: distances are whole numbers, got {distance.dtype}")
    lut, _ = _table(int(buckets), int(max_distance), bool(two_sided))
    at = distance.long().clamp(-max_distance, max_distance) + max_distance
    return torch.tensor(lut, dtype=torch.int64, device=distance.device)[at]
