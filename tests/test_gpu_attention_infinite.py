"""GPU tests of window attention where a visible key has an infinite component that makes its scores -inf:
a weight of exactly 0, so every output and gradient is that of the call that hides the key, but for dq in
the infinite column, where the definition has 0 times infinity."""

import math

import pytest
import torch

from attention_ref import assert_within, reference, visible

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("heads", [2, 40], ids=["few", "many"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("buckets", [0, 16], ids=["plain", "bias"])
@pytest.mark.parametrize("sign", [1.0, -1.0], ids=["scale+", "scale-"])
def test_gradients_beside_a_key_of_weight_zero(dev, heads, dtype, buckets, sign):
    from gdl_amd.functional import window_attention
    T, D, column, at = 900 if heads > 2 else 300, 32, 5, [0, 90, 91, 200]
    print(heads, dtype, buckets, sign, flush=True)
    gen = torch.Generator().manual_seed(heads + buckets)
    q, k, v, g = (torch.randn(T, heads, D, generator=gen).to(dev, dtype) for _ in range(4))
    q[..., column] = q[..., column].abs() + 0.25
    table = torch.randn(buckets, heads, generator=gen).to(dev, dtype) if buckets else None
    scale = sign / math.sqrt(D)
    bad = k.clone()
    bad[at, :, column] = -sign * math.inf
    leaves = [x.detach().requires_grad_() for x in (q, bad, v) + ((table,) if buckets else ())]
    out = window_attention(*leaves[:3], (40, 12), sinks=1, bias=leaves[3] if buckets else None, max_distance=20, scale=scale)
    got = dict(zip(("dq", "dk", "dv", "dbias"), torch.autograd.grad(out, leaves, g)), out=out)
    everywhere = visible(T, 40, 12, 1)
    seen = everywhere.clone()
    seen[:, at] = False
    # one head at a time of a few; each has all its sums to itself
    for h in (0, heads - 1):
        one = slice(h, h + 1)
        # with the sign on the queries: the reference's bounds are for a positive scale
        want, tol = reference(sign * q[:, one], k[:, one], v[:, one], g[:, one], seen, scale=1 / math.sqrt(D),
                              table=table[:, one] if buckets else None, maxd=20)
        want["dq"] = sign * want["dq"]
        part = {n: x[:, one].detach().clone() for n, x in got.items()}
        beside = everywhere[:, at].any(1)
        assert not torch.isfinite(part["dq"][beside.to(dev)][..., column].float()).any()
        part["dq"][..., column], want["dq"][..., column] = 0, 0
        assert_within(part, want, tol, h)
