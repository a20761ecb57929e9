"""Paged histories at the ends of what their arguments may be, and in calls that run at once."""

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
BF16, I8 = torch.bfloat16, torch.int8
ENDS = [-(1 << 63), -(1 << 62), (1 << 62), (1 << 63) - 1]


@pytest.mark.parametrize("columns", [2, 60])
def test_positions_as_far_out_as_they_go(dev, columns):
    """Streams that begin there are as those at other positions without a page; their neighbours stay right."""
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(21)
    Hk, H, d, n = 2, 4, 32, 70
    cache = PagedCache.empty(2 * len(ENDS) + 2, Hk, d, dtype=BF16, device=dev)
    for t in (cache.k, cache.v):
        t.fill_(2.0)
    table = torch.full((len(ENDS) + 1, columns), -1, dtype=torch.int32)
    table[:, :2] = torch.arange(2 * len(ENDS) + 2).view(-1, 2)
    table = table.to(dev)
    start = torch.tensor([0, *ENDS], device=dev)
    ptr = torch.arange(len(ENDS) + 2, device=dev) * n
    q, k, v = (torch.randn(n * (len(ENDS) + 1), h, d, generator=gen).bfloat16().to(dev) for h in (H, Hk, Hk))
    want = ref.copy(cache)
    for t in range(n):
        ref.put(want, "k", t // 64, t % 64, k[t]), ref.put(want, "v", t // 64, t % 64, v[t])
    cache.write(k, v, table, ptr, start)
    ref.same(cache, want)
    for x in cache.read(table, ptr, len(q), start=start):
        assert x[:n].isfinite().all() and x[n:].isnan().all()
    out = paged_attention(q, cache, table, ptr, start)
    ref.assert_near(out[:n], *ref.attend(q[:n], ref.stored(k[:n], BF16), ref.stored(v[:n], BF16), 0, BF16))
    assert (out[n:3 * n] == 0).all() and out[3 * n:].isnan().all()
    rows = torch.arange(len(ENDS) + 1, device=dev) * n
    out = paged_attention_step(q[rows], k[rows], v[rows], cache, table, start)
    assert torch.equal(out[0], v[0].repeat_interleave(H // Hk, 0))
    assert (out[1:3] == 0).all() and out[3:].isnan().all()
    ref.same(cache, want)


def test_calls_that_run_at_once(dev):
    """Prompts and steps over one pool on several streams, each with pieces of its own to join."""
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(22)
    Hk, H, d, n = 2, 8, 64, 6000
    pages = n // 64 + 2
    cache = PagedCache.empty(pages, Hk, d, dtype=I8, device=dev)
    table = torch.randperm(pages, generator=gen).int().view(1, -1).to(dev)
    k, v = (torch.randn(n + 1, Hk, d, generator=gen).bfloat16().to(dev) for _ in range(2))
    cache.write(k, v, table)
    at = torch.tensor([n], device=dev)
    q = [torch.randn(40, H, d, generator=gen).bfloat16().to(dev) for _ in range(6)]

    def call(x, step):
        if step:
            return paged_attention_step(x[:1], k[n:], v[n:], cache, table, at)
        return paged_attention(x, cache, table, None, at - 40)

    want = [call(x, i % 2) for i, x in enumerate(q)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    got = [[] for _ in q]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(q[i], i % 2))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(o, want[i]) for o in outs), i


def test_two_graphs_and_eager_calls_in_turn(dev):
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(23)
    Hk, H, d, n, B = 1, 4, 32, 5000, 2
    pages = 80
    cache = PagedCache.empty(B * pages, Hk, d, dtype=BF16, device=dev)
    table = torch.randperm(B * pages, generator=gen).int().view(B, -1).to(dev)
    k, v = (torch.randn(B * n, Hk, d, generator=gen).bfloat16().to(dev) for _ in range(2))
    cache.write(k, v, table, torch.tensor([0, n, 2 * n], device=dev))
    ptr, start = torch.tensor([0, 20, 33], device=dev), torch.tensor([n - 60, n - 80], device=dev)
    q, k1, v1 = (torch.randn(33, h, d, generator=gen).bfloat16().to(dev) for h in (H, Hk, Hk))
    at = torch.tensor([n, n - 7], device=dev)

    def prompt():
        return paged_attention(q, cache, table, ptr, start)

    def step():
        return paged_attention_step(q[:B], k1[:B], v1[:B], cache, table, at)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        prompt(), step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for call in (prompt, step):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for turn in range(4):
        q.copy_(torch.randn(q.shape, generator=gen)), k1.copy_(torch.randn(k1.shape, generator=gen)), at.add_(1)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(kept, (prompt(), step()))), turn
