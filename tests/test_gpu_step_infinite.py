"""GPU tests of the single-token form where the cache holds infinities in tokens that the query sees."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [8, 24, 32, 40, 56, 64, 72, 120, 128])
@pytest.mark.parametrize("column", ["first", "last"])
@pytest.mark.parametrize("H", [2, 8])
def test_a_key_of_weight_zero(dev, dtype, D, column, H):
    """One infinite component that makes a token's scores -inf: its weight is exactly 0 whichever
    component it is, so what its value holds does not matter, and the rest is softmax attention.
    Bound: products and sums in float32 (scores' error (D + 4) units, 60 keys), one rounding to the type."""
    from gdl_amd.functional import WindowCache, window_attention_step
    print(dtype, D, column, H, flush=True)
    B, Hk, left, at = 3, 2, 59, 17
    c = 0 if column == "first" else D - 1
    gen = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(B, h, D, generator=gen).to(dev, dtype) for h in (H, Hk, Hk))
    q[..., c] = q[..., c].abs() + 0.25
    cache = WindowCache.empty(B, Hk, D, left, dtype=dtype, device=dev)
    for x in (cache.k, cache.v):
        x.copy_(torch.randn(x.shape, generator=gen))
    cache.k[:, :, at, c] = -math.inf
    pos = torch.full((B,), 99, device=dev)
    out = window_attention_step(q, k, v, cache, pos).double().cpu()
    kc, vc = (x.double().cpu().repeat_interleave(H // Hk, 1) for x in (cache.k, cache.v))
    keep = torch.arange(left + 1) != at
    kc, vc = kc[:, :, keep], vc[:, :, keep]
    s = (kc * q.double().cpu().unsqueeze(2)).sum(-1) / math.sqrt(D)
    S = (kc * q.double().cpu().unsqueeze(2)).abs().sum(-1) / math.sqrt(D)
    p = s.softmax(-1)
    want = (p.unsqueeze(-1) * vc).sum(2)
    u = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
    w = 2 * 2.0 ** -24 * ((D + 4) * S.amax(-1) + 4 + left)
    bound = u * want.abs() + w.unsqueeze(-1) * (p.unsqueeze(-1) * vc.abs()).sum(2) + 2.0 ** -25
    assert ((out - want).abs() <= bound).all(), (out - want).abs().max()
