"""GPU tests of the attention's backward where some inputs need no gradient: the others' are the same bit by
bit, and kernels for what is not needed do not run."""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("H,T", [(4, 500), (24, 1500)])
def test_the_needed_gradients_are_the_same(dev, dtype, bias, H, T):
    from gdl_amd.functional import window_attention
    gen = torch.Generator().manual_seed(T)
    q, g = (torch.randn(T, H, 32, generator=gen).to(dev, dtype) for _ in range(2))
    k, v = (torch.randn(T, H // 2, 32, generator=gen).to(dev, dtype) for _ in range(2))
    inputs = [q, k, v] + ([torch.randn(8, H, generator=gen).to(dev)] if bias else [])
    kw = dict(sinks=3, ptr=torch.tensor([0, 17, T], device=dev), max_distance=20)

    def grads(needs):
        leaves = [x.clone().requires_grad_(n) for x, n in zip(inputs, needs)]
        out = window_attention(*leaves[:3], (60, 0), bias=leaves[3] if bias else None, **kw)
        return torch.autograd.grad(out, [x for x, n in zip(leaves, needs) if n], g)

    everything = grads([True] * len(inputs))
    for needs in itertools.product([False, True], repeat=len(inputs)):
        if any(needs):
            want = [x for x, n in zip(everything, needs) if n]
            assert all(torch.equal(a, b) for a, b in zip(grads(needs), want)), needs


def test_kernels_that_run(dev):
    from torch.profiler import ProfilerActivity, profile
    from gdl_amd.functional import window_attention
    q, k, v = (torch.randn(400, 2, 32, device=dev) for _ in range(3))
    table = torch.randn(8, 2, device=dev)

    def names(*needs):
        leaves = [x.clone().requires_grad_(n) for x, n in zip((q, k, v, table), needs)]
        out = window_attention(*leaves[:3], (30, 0), sinks=2, bias=leaves[3], max_distance=20)
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            out.backward(q)
            torch.cuda.synchronize()
        return {n for e in p.events() for n in ("attend_bwd_q", "attend_bwd_kv", "attend_bwd_join", "attend_bwd_bias") if n in e.name}

    assert names(True, True, True, True) == {"attend_bwd_q", "attend_bwd_kv", "attend_bwd_join", "attend_bwd_bias"}
    assert names(False, False, False, True) == {"attend_bwd_q", "attend_bwd_bias"}
    assert names(True, False, False, False) == {"attend_bwd_q"}
    assert names(False, True, False, False) == {"attend_bwd_q", "attend_bwd_kv", "attend_bwd_join"}
