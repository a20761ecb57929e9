"""GPU tests of window attention, both forms, for queries that see keys but only with scores of -inf: the
softmax is 0 / 0 there, and NaN says so.  Queries that see no key give 0."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("heads", [2, 48], ids=["few", "many"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("how", ["key", "query", "bias"])
def test_forward_and_gradients(dev, dtype, heads, how):
    from gdl_amd.functional import window_attention
    T, D = 800 if heads > 2 else 200, 32
    print(dtype, heads, how, flush=True)
    gen = torch.Generator().manual_seed(3)
    q, k, v, g = (torch.randn(T, heads, D, generator=gen).to(dev, dtype) for _ in range(4))
    ptr = torch.tensor([0, 40, 110, T], device=dev)
    table = torch.zeros(8, heads, device=dev, dtype=dtype)
    mask = torch.ones(T, dtype=torch.bool, device=dev)
    mask[30:36] = False  # tokens 33 .. 35 see no key at all
    if how == "bias":    # the distances up to 2 back are hidden: each sequence's first tokens have no others
        table[:3] = -math.inf
        bad = torch.tensor([0, 1, 2, 40, 41, 42, 110, 111, 112])
    elif how == "key":   # a stretch of keys longer than the window
        q[..., 7] = q[..., 7].abs() + 0.25
        k[60:80, :, 7] = -math.inf
        bad = torch.arange(63, 80)
    else:
        k[40:110, :, 7] = k[40:110, :, 7].abs() + 0.25
        q[90, :, 7] = -math.inf
        bad = torch.tensor([90])
    leaves = [x.requires_grad_() for x in (q, k, v, table)]
    out = window_attention(*leaves[:3], (3, 0), ptr=ptr, mask=mask, bias=leaves[3], max_distance=9)
    dq, dk, dv, dt = torch.autograd.grad(out, leaves, g)
    blank = torch.arange(33, 36)
    rest = torch.ones(T, dtype=torch.bool)
    rest[bad], rest[blank] = False, False
    if how == "bias":
        rest[33] = True  # sees no key either way
        bad = bad[bad != 33]
    # with the near distances hidden a token needs a key exactly three back
    if how == "bias":
        first = torch.zeros(T, dtype=torch.long)
        first[40:110], first[110:] = 40, 110
        i = torch.arange(T)
        sees = torch.stack([(i - n >= first) & mask.cpu()[(i - n).clamp(0)] for n in range(4)])
        blank, bad = i[~sees.any(0)], i[sees.any(0) & ~sees[3]]
        rest = sees[3]
    assert torch.isnan(out[bad.to(dev)].float()).all() and torch.isnan(dq[bad.to(dev)].float()).all()
    assert (out[blank.to(dev)] == 0).all() and (dq[blank.to(dev)] == 0).all()
    assert torch.isfinite(out[rest.to(dev)].float()).all()
    # the keys that such a query sees have its NaN in their gradients, the others do not
    touched = torch.zeros(T, dtype=torch.bool)
    for b in bad.tolist():
        lo = max(b - 3, [a for a in (0, 40, 110) if a <= b][-1])
        touched[lo:b + 1] = True
    touched &= mask.cpu()
    assert torch.isnan(dv[touched.to(dev)].float()).all() and torch.isfinite(dv[~touched.to(dev)].float()).all()
    assert torch.isnan(dk[touched.to(dev)].float()).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("left", [9, 4000])
def test_step(dev, dtype, left):
    from gdl_amd.functional import WindowCache, window_attention_step
    B, H, Hk, D = 4, 4, 2, 64
    gen = torch.Generator().manual_seed(4)
    cache = WindowCache.empty(B, Hk, D, left, dtype=dtype, device=dev)
    for x in (cache.k, cache.v):
        x.copy_(torch.randn(x.shape, generator=gen))
    q, k, v = (torch.randn(B, h, D, generator=gen).to(dev, dtype) for h in (H, Hk, Hk))
    q[..., 7] = q[..., 7].abs() + 0.25
    cache.k[0, ..., 7], k[0, :, 7] = -math.inf, -math.inf
    cache.k[1, ..., 7] = -math.inf  # its new token is a key like any other
    out = window_attention_step(q, k, v, cache, torch.tensor([left + 5, left + 5, -1, left + 5], device=dev)).float()
    assert torch.isnan(out[0]).all()
    assert torch.equal(out[1], v[1].float().repeat_interleave(H // Hk, 0))
    assert (out[2] == 0).all() and torch.isfinite(out[3]).all()
