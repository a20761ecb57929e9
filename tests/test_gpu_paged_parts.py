"""Weights in two parts: steps and short prompts of 16-bit types are off by the output's rounding and little more.

Two roundings leave 2^-16 of a weight in bfloat16 and 2^-22 in float16 (2^-16 where codes meet bfloat16 parts)."""

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
BF16, F16, I8, E4 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
TYPES = [(BF16, BF16, 2.0 ** -16), (F16, F16, 2.0 ** -22), (BF16, I8, 2.0 ** -16), (F16, E4, 2.0 ** -16)]
IDS = ["bf16", "f16", "bf16-i8", "f16-e4m3"]


@pytest.mark.parametrize("dtype,stored,unit", TYPES, ids=IDS)
@pytest.mark.parametrize("n,H,Hk,d", [(1, 2, 1, 16), (3, 4, 4, 32), (90, 8, 2, 64), (700, 6, 2, 128), (3000, 4, 1, 64)])
def test_steps_and_short_prompts(dev, dtype, stored, unit, n, H, Hk, d):
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(n + d)
    pages = -(-n // 64)
    cache = PagedCache.empty(pages, Hk, d, dtype=stored, device=dev)
    table = torch.randperm(pages, generator=gen).int().view(1, -1).to(dev)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(dtype).to(dev) for h in (H, Hk, Hk))
    cache.write(k, v, table)
    new = min(n, 5)
    want, tol = ref.attend(q[-new:], ref.stored(k, stored), ref.stored(v, stored), n - new, stored, unit=unit)
    ref.assert_near(paged_attention(q[-new:], cache, table, None, torch.tensor([n - new], device=dev)), want, tol)
    out = paged_attention_step(q[-1:], k[-1:], v[-1:], cache, table, torch.tensor([n - 1], device=dev))
    ref.assert_near(out, want[-1:], tol[-1:])
