"""GPU tests of the single-token form of window attention over its ring cache: every step of growing
streams against the dense definition in float64, the cache's contents, offsets beyond 32 bits,
refusals."""

import math

import pytest
import torch

from attention_ref import assert_within, reference, visible

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,H,Hk,D,left,sinks,buckets,maxd", [
    (1, 1, 1, 8, 0, 0, 0, 0), (2, 4, 1, 32, 5, 0, 8, 9), (3, 6, 2, 24, 9, 4, 0, 0), (1, 8, 1, 64, 31, 1, 16, 20),
    (2, 7, 7, 48, 12, 3, 0, 0), (2, 10, 2, 128, 17, 2, 16, 40), (1, 5, 1, 80, 40, 0, 8, 5)])
def test_streams_token_by_token(dev, dtype, B, H, Hk, D, left, sinks, buckets, maxd):
    from gdl_amd.functional import WindowCache, window_attention_step
    T = 2 * (left + sinks) + 7
    print(B, H, Hk, D, left, sinks, dtype, flush=True)
    gen = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(B, T, h, D, generator=gen).to(dev, dtype) for h in (H, Hk, Hk))
    table = torch.randn(buckets, H, generator=gen).to(dev, dtype) if buckets else None
    cache = WindowCache.empty(B, Hk, D, left, sinks=sinks, dtype=dtype, device=dev)
    cache.k.fill_(math.nan), cache.v.fill_(math.nan)  # slots without a token are not read
    refs = [reference(q[b], k[b], v[b], None, visible(T, left, 0, sinks), table=table, maxd=maxd, two_sided=False)
            for b in range(B)]
    for t in range(T):
        out = window_attention_step(q[:, t], k[:, t], v[:, t], cache, torch.full((B,), t, device=dev), bias=table,
                                    max_distance=maxd or 128)
        for b, (want, tol) in enumerate(refs):
            assert_within({"out": out[b]}, {"out": want["out"][t]}, {"out": tol["out"][t]}, (t, b))
        # the cache holds exactly the window
        for j in range(t + 1):
            if j < sinks or j >= t - left:
                slot = j if j < sinks else sinks + (j - sinks) % (left + 1)
                assert torch.equal(cache.k[:, :, slot], k[:, j]) and torch.equal(cache.v[:, :, slot], v[:, j])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,H,Hk,D,left,sinks", [(1, 2, 2, 64, 5000, 4), (5, 8, 2, 32, 900, 0), (2, 16, 1, 128, 2500, 16)])
def test_long_windows_after_fill(dev, dtype, B, H, Hk, D, left, sinks):
    """Windows that are split over workgroups, streams of unequal age, filled from packed sequences;
    the result is window_attention's for the last token."""
    from gdl_amd.functional import WindowCache, window_attention, window_attention_step
    gen = torch.Generator().manual_seed(left)
    ages = [(left + 700) * (b + 1) // B - 3 * b for b in range(B)]
    ptr = torch.tensor([0] + ages).cumsum(0)
    q, k, v = (torch.randn(int(ptr[-1]), h, D, generator=gen).to(dev, dtype) for h in (H, Hk, Hk))
    table = torch.randn(32, H, generator=gen).to(dev, dtype)
    last = ptr[1:] - 1
    keep = torch.ones(int(ptr[-1]), dtype=torch.bool)
    keep[last] = False
    cache = WindowCache.empty(B, Hk, D, left, sinks=sinks, dtype=dtype, device=dev)
    before = (ptr - torch.arange(B + 1)).to(dev)
    kk, vv = k[keep.to(dev)], v[keep.to(dev)]
    half = before[:-1] + (before[1:] - before[:-1]) // 2  # in two portions
    pieces = [[], []]
    for b in range(B):
        lo, mid, hi = int(before[b]), int(half[b]), int(before[b + 1])
        pieces[0].append((lo, mid)), pieces[1].append((mid, hi))
    for n in (0, 1):
        rows = torch.cat([torch.arange(a, b) for a, b in pieces[n]]).to(dev)
        p = torch.tensor([0] + [b - a for a, b in pieces[n]]).cumsum(0).to(dev)
        start = None if n == 0 else (half - before[:-1])
        cache.fill(kk[rows], vv[rows], p if B > 1 else (p if n else None), start)
    pos = torch.tensor(ages, device=dev) - 1
    out = window_attention_step(q[last.to(dev)], k[last.to(dev)], v[last.to(dev)], cache, pos, bias=table)
    full = window_attention(q, k, v, (left, 0), sinks=sinks, ptr=ptr.to(dev), bias=table)[last.to(dev)]
    for b in range(B):
        a, e = int(ptr[b]), int(ptr[b + 1])
        seen = visible(e - a, left, 0, sinks)[-1:]
        want, tol = _last(q[a:e], k[a:e], v[a:e], seen, table)
        assert_within({"out": out[b]}, want, tol, b)
        assert_within({"out": full[b]}, want, tol, b)


def _last(q, k, v, seen, table):
    """The definition for the last token alone."""
    u, e = {F32: 2.0 ** -24, BF16: 2.0 ** -8}[q.dtype], 2.0 ** -24
    from attention_ref import bucket
    T, H, D = q.shape
    n = H // k.shape[1]
    kd, vd = (x.double().cpu().transpose(0, 1).repeat_interleave(n, 0) for x in (k, v))
    x = q[-1].double().cpu()
    b = torch.tensor([bucket(j - T + 1, table.shape[0], 128, False) for j in range(T)])
    t = table.double().cpu().t()[:, b]
    s = (kd * x[:, None]).sum(-1) / math.sqrt(D) + t
    S = (kd * x[:, None]).abs().sum(-1) / math.sqrt(D) + t.abs()
    p = s.masked_fill(~seen, -math.inf).softmax(-1)
    w = 2 * e * ((D + 4) * S.amax(-1, keepdim=True) + 4) + e * T
    o = (p[..., None] * vd).sum(1)
    return {"out": o}, {"out": u * o.abs() + ((p * (u + w))[..., None] * vd.abs()).sum(1)}


def test_inactive_streams_and_strides(dev):
    from gdl_amd.functional import WindowCache, window_attention_step
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(3, 8, 32, generator=gen).to(dev)  # one projection's output
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    caches = [WindowCache.empty(3, 2, 32, 6, sinks=1, device=dev) for _ in range(2)]
    for c in caches:
        c.k.fill_(0.5), c.v.fill_(0.25)
    pos = torch.tensor([20, -1, 3], device=dev)
    out = window_attention_step(q, k, v, caches[0], pos)
    assert (out[1] == 0).all() and (caches[0].k[1] == 0.5).all() and (caches[0].v[1] == 0.25).all()
    same = window_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), caches[1], pos.int())
    assert torch.equal(out, same) and torch.equal(caches[0].k, caches[1].k)
    # a cache that is part of a larger buffer
    buf = torch.zeros(3, 2, 2, 8, 32, device=dev)
    part = WindowCache(buf[:, 0], buf[:, 1], sinks=1)
    part.k.fill_(0.5), part.v.fill_(0.25)
    assert torch.equal(window_attention_step(q, k, v, part, pos), out)


def test_cache_beyond_32_bit_offsets(dev):
    """A cache of over 2^32 bytes and 2^31 elements: the last stream's slots are the right ones."""
    from gdl_amd.functional import WindowCache, window_attention_step
    B, Hk, D, left = 130, 8, 128, 16383
    cache = WindowCache.empty(B, Hk, D, left, dtype=BF16, device=dev)
    assert cache.k.numel() > 2 ** 31
    gen = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(B, Hk, D, generator=gen).to(dev, BF16) for _ in range(3))
    pos = torch.full((B,), 40, device=dev)
    pos[-1] = 100000
    cache.k[-1].normal_(), cache.v[-1].normal_()
    cache.k[:, :, :41].normal_(), cache.v[:, :, :41].normal_()
    out = window_attention_step(q, k, v, cache, pos)
    slot = 100000 % (left + 1)
    assert torch.equal(cache.k[-1, :, slot], k[-1])
    kc, vc = cache.k[-1].double(), cache.v[-1].double()
    p = ((kc * q[-1].double()[:, None]).sum(-1) / math.sqrt(D)).softmax(-1)
    want = (p[..., None] * vc).sum(1)
    bound = 2.0 ** -8 * want.abs() + (p[..., None] * vc.abs()).sum(1) * 1e-4
    assert ((out[-1].double() - want).abs() <= bound).all()


def test_steps_in_a_graph(dev):
    from gdl_amd.functional import WindowCache, window_attention_step
    B, H, Hk, D, left = 2, 4, 2, 64, 1000
    caches = [WindowCache.empty(B, Hk, D, left, sinks=2, dtype=BF16, device=dev) for _ in range(2)]
    for c in caches:
        c.k.fill_(0.125), c.v.fill_(0.5)
    q, k, v = (torch.randn(B, h, D, device=dev).to(BF16) for h in (H, Hk, Hk))
    pos = torch.tensor([1200, 7], device=dev)
    table = torch.randn(16, H, device=dev, dtype=BF16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        window_attention_step(q, k, v, caches[0], pos, bias=table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention_step(q, k, v, caches[0], pos, bias=table)
    caches[1].k.copy_(caches[0].k), caches[1].v.copy_(caches[0].v)
    for n in range(5):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(n)))
        pos += 1
        graph.replay()
        torch.cuda.synchronize()
        want = window_attention_step(q, k, v, caches[1], pos, bias=table)
        assert torch.equal(out, want) and torch.equal(caches[0].k, caches[1].k)


def test_refusals(dev):
    from gdl_amd.functional import WindowCache, window_attention_step
    with pytest.raises(ValueError):
        WindowCache.empty(1, 1, 12, 4, device=dev)
    with pytest.raises(ValueError):
        WindowCache.empty(1, 1, 16, -1, device=dev)
    with pytest.raises(ValueError):
        WindowCache(torch.zeros(1, 1, 4, 16, device=dev), torch.zeros(1, 1, 4, 16, device=dev), sinks=4)
    with pytest.raises(ValueError):
        WindowCache(torch.zeros(1, 4, 1, 16, device=dev).transpose(1, 2).expand(1, 1, 4, 16)[..., ::2],
                    torch.zeros(1, 1, 4, 8, device=dev))
    cache = WindowCache.empty(2, 2, 16, 4, device=dev)
    q, k, v = (torch.zeros(2, h, 16, device=dev) for h in (4, 2, 2))
    pos = torch.zeros(2, dtype=torch.int64, device=dev)
    bad = [(ValueError, dict(q=q[:1])), (ValueError, dict(q=q[:, :3])), (ValueError, dict(k=k[:, :1])),
           (TypeError, dict(q=q.bfloat16())), (ValueError, dict(positions=pos.float())), (ValueError, dict(positions=pos[:1])),
           (RuntimeError, dict(positions=pos.cpu())), (ValueError, dict(bias=torch.zeros(8, 3, device=dev))),
           (RuntimeError, dict(q=q.clone().requires_grad_()))]
    for error, change in bad:
        with pytest.raises(error):
            window_attention_step(**(dict(q=q, k=k, v=v, cache=cache, positions=pos) | change))
    for args in ((k, v), (k[:, :1], v[:, :1], pos.new_tensor([0, 1, 2])), (k, v, pos.new_tensor([0, 2])),
                 (k, v, pos.new_tensor([0, 1, 2]), pos[:1])):
        with pytest.raises(ValueError):
            cache.fill(*args)
