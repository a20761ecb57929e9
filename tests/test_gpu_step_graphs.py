"""GPU tests of captured steps beside eager calls on the same cache."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_captured_step_keeps_its_scratch(dev):
    """A graph of a step whose window is split over workgroups, captured after an eager call with as many
    heads and replayed after one with more: it writes to no memory that others have been given since."""
    from gdl_amd.csrc import _nat
    from gdl_amd.functional import WindowCache, window_attention_step
    B, Hk, D, left = 1, 2, 64, 4000
    gen = torch.Generator().manual_seed(1)
    caches = [WindowCache.empty(B, Hk, D, left, device=dev) for _ in range(2)]
    for x in ("k", "v"):
        getattr(caches[0], x).copy_(torch.randn(caches[0].k.shape, generator=gen))
        getattr(caches[1], x).copy_(getattr(caches[0], x))
    q, wide = (torch.randn(B, h, D, generator=gen).to(dev) for h in (4, 64))
    k, v = (torch.randn(B, Hk, D, generator=gen).to(dev) for _ in range(2))
    pos = torch.tensor([5000], device=dev)
    size = _nat.lib().geo_window_attention_step_workspace_bytes(B, 4, Hk, left + 1, D)
    assert size > 0
    window_attention_step(q, k, v, caches[0], pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention_step(q, k, v, caches[0], pos)
    window_attention_step(wide, k, v, caches[0], pos)
    torch.cuda.synchronize()
    others = [torch.full((size,), 7, dtype=torch.uint8, device=dev) for _ in range(50)]
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, window_attention_step(q, k, v, caches[1], pos))
        assert all((x == 7).all() for x in others)
