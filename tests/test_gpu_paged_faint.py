"""Softmax weights far below the largest: a token whose value is 0 stands high above thousands of others, which are
what its row consists of.  Every weight keeps its digits, however small.

Bounds as in paged_ref, but without its half step of float16's least numbers for each weight: weights are
off by 2^-11 of themselves at most in float16 (2^-8 in bfloat16), by 2^-16 where they are kept in two parts.
"""

import math

import pytest
import torch

import paged_ref as ref
from attention_ref import SPACING, UNIT

pytestmark = pytest.mark.gpu
F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F16, I8), (BF16, E4)]
IDS = ["f32", "bf16", "f16", "f16-i8", "bf16-e4m3"]


def _history(dev, dtype, n, H, Hk, d, gap, sink, gen):
    """(q, k, v): token ``sink`` has a score of ``gap`` powers of two above the others' and the value 0."""
    q = (1 + 0.02 * torch.randn(n, H, d, generator=gen)).to(dtype).to(dev)
    k = 0.1 * torch.randn(n, Hk, d, generator=gen)
    k[sink] = gap * math.log(2) / math.sqrt(d)
    v = 8000 * (1 + 0.3 * torch.randn(n, Hk, d, generator=gen))
    v[sink] = 0
    return q, k.to(dtype).to(dev), v.to(dtype).to(dev)


def _check_row(out, q, K, V, unit):
    """One row [H, D] of q [H, D] over K, V float64 [n, Hk, D]."""
    e, (H, D), (n, Hk, _) = 2.0 ** -24, q.shape, K.shape
    dtype, q = q.dtype, q.double().cpu().unsqueeze(1)
    K, V = (x.transpose(0, 1).repeat_interleave(H // Hk, 0) for x in (K, V))
    s, S = q @ K.transpose(1, 2) / math.sqrt(D), q.abs() @ K.abs().transpose(1, 2) / math.sqrt(D)
    p = s.softmax(-1)
    w = 2 * e * ((D + 8) * S.amax(-1, keepdim=True) + 4) + e * n
    o = (p @ V).squeeze(1)
    ref.assert_near(out, o, UNIT[dtype] * o.abs() + SPACING[dtype] / 2 + ((unit + w + e) * (p @ V.abs())).squeeze(1))


def _pool(dev, n, Hk, d, stored, k, v, gen):
    from gdl_amd.functional import PagedCache
    pages = -(-n // 64)
    cache = PagedCache.empty(pages, Hk, d, dtype=stored, device=dev)
    table = torch.randperm(pages, generator=gen).int().view(1, -1).to(dev)
    cache.write(k, v, table)
    return cache, table


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("gap", [12, 20, 26, 33])
@pytest.mark.parametrize("n,H,Hk,d,sink", [(1400, 2, 1, 64, 0), (1400, 20, 1, 128, 700), (9000, 8, 2, 32, 5)])
def test_steps_and_short_prompts(dev, dtype, stored, gap, n, H, Hk, d, sink):
    from gdl_amd.functional import paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(gap + d)
    q, k, v = _history(dev, dtype, n, H, Hk, d, gap, sink, gen)
    cache, table = _pool(dev, n, Hk, d, stored, k, v, gen)
    K, V = ref.stored(k, stored), ref.stored(v, stored)
    unit = 2.0 ** -24 if dtype is F32 else 2.0 ** -16
    out = paged_attention(q[-4:], cache, table, None, torch.tensor([n - 4], device=dev))
    for i in range(4):
        _check_row(out[i], q[n - 4 + i], K[:n - 3 + i], V[:n - 3 + i], unit)
    out = paged_attention_step(q[-1:], k[-1:], v[-1:], cache, table, torch.tensor([n - 1], device=dev))
    _check_row(out[0], q[-1], K, V, unit)


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("gap,d", [(12, 32), (20, 64), (26, 128), (33, 64)])
def test_long_prompts(dev, dtype, stored, gap, d):
    from gdl_amd.functional import paged_attention
    gen = torch.Generator().manual_seed(gap + d)
    n, H, Hk = 5000, 16, 2
    q, k, v = _history(dev, dtype, n, H, Hk, d, gap, 3, gen)
    cache, table = _pool(dev, n, Hk, d, stored, k, v, gen)
    K, V = ref.stored(k, stored), ref.stored(v, stored)
    # codes meet float16 queries' weights in two parts of bfloat16
    unit = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11 if stored is F16 else 2.0 ** -16}[dtype]
    out = paged_attention(q, cache, table)
    for t in (2, 3, 4, 70, 1100, 2600, 4095, 4999):
        _check_row(out[t], q[t], K[:t + 1], V[:t + 1], unit)
