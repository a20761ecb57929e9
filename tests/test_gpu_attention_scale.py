"""GPU tests of window attention with a scale of its own, positive, negative or zero, in every kernel and both
forms, and of float16 in the four-wave kernels, against the dense definition in float64."""

import pytest
import torch

from attention_ref import assert_within, reference, visible

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _want(q, k, v, g, seen, scale, **kw):
    """The definition, its bounds for a positive scale: a negative one as negative queries."""
    sign = -1.0 if scale < 0 else 1.0
    want, tol = reference(sign * q, k, v, g, seen, scale=abs(scale), **kw)
    if "dq" in want:
        want["dq"] = sign * want["dq"]
    return want, tol


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scale", [0.7, -0.3, 0.0])
@pytest.mark.parametrize("T,H,D", [(300, 2, 48), (1300, 48, 32)])
def test_forward_and_gradients(dev, dtype, bias, scale, T, H, D):
    from gdl_amd.functional import window_attention
    print(dtype, bias, scale, T, flush=True)
    gen = torch.Generator().manual_seed(T)
    q, k, v, g = (torch.randn(T, H, D, generator=gen).to(dev, dtype) for _ in range(4))
    table = torch.randn(16, H, generator=gen).to(dev, dtype) if bias else None
    mask = (torch.rand(T, generator=gen) < 0.8).to(dev)
    ptr = [0, 77, 78, T]
    leaves = [x.clone().requires_grad_() for x in (q, k, v) + ((table,) if bias else ())]
    out = window_attention(*leaves[:3], (50, 9), sinks=4, ptr=torch.tensor(ptr, device=dev), mask=mask, scale=scale,
                           bias=leaves[3] if bias else None, max_distance=30)
    got = dict(zip(("dq", "dk", "dv", "dbias"), torch.autograd.grad(out, leaves, g)), out=out)
    seen = visible(T, 50, 9, 4, ptr, mask)
    for h in (0, H - 1):
        one = slice(h, h + 1)
        want, tol = _want(q[:, one], k[:, one], v[:, one], g[:, one], seen, scale, table=table[:, one] if bias else None, maxd=30)
        assert_within({n: x[:, one] for n, x in got.items()}, want, tol, h)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scale", [0.7, -0.3, 0.0])
def test_step(dev, dtype, bias, scale):
    from gdl_amd.functional import WindowCache, window_attention_step
    T, H, Hk, D, left, sinks = 40, 4, 2, 40, 11, 2
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(T, h, D, generator=gen).to(dev, dtype) for h in (H, Hk, Hk))
    table = torch.randn(8, H, generator=gen).to(dev, dtype) if bias else None
    want, tol = _want(q, k, v, None, visible(T, left, 0, sinks), scale, table=table, maxd=9, two_sided=False)
    cache = WindowCache.empty(1, Hk, D, left, sinks=sinks, dtype=dtype, device=dev)
    for t in range(T):
        out = window_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], cache, torch.tensor([t], device=dev), bias=table,
                                    max_distance=9, scale=scale)
        assert_within({"out": out[0]}, {"out": want["out"][t]}, {"out": tol["out"][t]}, t)


@pytest.mark.parametrize("D,H,Hk", [(64, 32, 8), (32, 40, 40), (128, 24, 12), (96, 16, 16)])
def test_float16_in_shared_tiles(dev, D, H, Hk):
    from gdl_amd.functional import window_attention
    T = 2100
    gen = torch.Generator().manual_seed(D)
    q, g = (torch.randn(T, H, D, generator=gen).to(dev, F16) for _ in range(2))
    k, v = (torch.randn(T, Hk, D, generator=gen).to(dev, F16) for _ in range(2))
    table = torch.randn(16, H, generator=gen).to(dev, F16)
    mask = (torch.rand(T, generator=gen) < 0.8).to(dev)
    ptr = [0, 700, 701, 2100]
    leaves = [x.clone().requires_grad_() for x in (q, k, v, table)]
    out = window_attention(*leaves[:3], (90, 33), sinks=5, ptr=torch.tensor(ptr, device=dev), mask=mask, bias=leaves[3],
                           max_distance=50)
    got = dict(zip(("dq", "dk", "dv", "dbias"), torch.autograd.grad(out, leaves, g)), out=out)
    seen, n = visible(T, 90, 33, 5, ptr, mask), H // Hk
    for hk in (0, Hk - 1):
        a, b = hk * n, hk * n + n
        want, tol = reference(q[:, a:b], k[:, hk:hk + 1], v[:, hk:hk + 1], g[:, a:b], seen, table=table[:, a:b], maxd=50)
        part = {x: got[x][:, a:b] for x in ("out", "dq", "dbias")} | {x: got[x][:, hk:hk + 1] for x in ("dk", "dv")}
        assert_within(part, want, tol, (D, hk))
