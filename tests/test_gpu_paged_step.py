"""GPU tests of attention of single tokens over paged caches, against the definition in float64."""

import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, I8), (F16, I8), (F32, E4), (BF16, E4), (F16, E4)]
IDS = [f"{str(a)[6:]}-{str(b)[6:]}" for a, b in TYPES]


def _filled(dev, lengths, heads, d, page, dtype, stored, gen, spare=1):
    """(cache, table, rows k, v of all tokens): tokens 0 .. n - 1 of each stream are in; all else is NaN."""
    from gdl_amd.functional import PagedCache
    pages = sum(-(-n // page) for n in lengths) + 3
    table = ref.random_table(lengths, page, pages, gen, spare)
    cache = PagedCache.empty(pages, heads, d, page=page, dtype=stored, device=dev)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0xFF) if stored is not I8 else t.fill_(-128)
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(math.nan)
    return cache, table.to(dev)


def _rows(lengths, heads, d, dtype, gen, dev):
    return [torch.randn(n, heads, d, generator=gen).to(dtype).to(dev) for n in lengths]


def _check(dev, dtype, stored, lengths, H, Hk, d, page, buckets=0, maxd=128, scale=None, spare=1):
    from gdl_amd.functional import paged_attention_step
    print(dtype, stored, lengths, H, Hk, d, page, buckets, flush=True)
    gen = torch.Generator().manual_seed(sum(lengths) + H + d)
    cache, table = _filled(dev, lengths, Hk, d, page, dtype, stored, gen, spare)
    ks, vs = _rows(lengths, Hk, d, dtype, gen, dev), _rows(lengths, Hk, d, dtype, gen, dev)
    B = len(lengths)
    q = torch.randn(B, H, d, generator=gen).to(dtype).to(dev)
    bias = torch.randn(buckets, H, generator=gen).to(dtype).to(dev) if buckets else None
    before = [n - 1 for n in lengths]
    ptr = torch.tensor([0] + before).cumsum(0).to(dev)
    if sum(before):
        cache.write(torch.cat([k[:-1] for k in ks]), torch.cat([v[:-1] for v in vs]), table, ptr)
    want_pool = ref.copy(cache)
    for b, n in enumerate(lengths):
        at = int(table[b, (n - 1) // page]), (n - 1) % page
        ref.put(want_pool, "k", *at, ks[b][-1]), ref.put(want_pool, "v", *at, vs[b][-1])
    out = paged_attention_step(q, torch.stack([k[-1] for k in ks]), torch.stack([v[-1] for v in vs]), cache, table,
                               torch.tensor(before, device=dev), bias=bias, max_distance=maxd, scale=scale)
    for b in range(B):
        want, tol = ref.attend(q[b:b + 1], ref.stored(ks[b], stored), ref.stored(vs[b], stored), lengths[b] - 1, stored, scale, bias, maxd)
        ref.assert_near(out[b:b + 1], want, tol, (b, lengths[b]))
    ref.same(cache, want_pool)
    return out


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("lengths,H,Hk,d,page", [
    ([1], 1, 1, 16, 64), ([2, 64, 65, 63, 1], 6, 2, 32, 64), ([16, 17, 31, 33, 130], 4, 1, 64, 128), ([300, 5], 3, 3, 48, 192),
    ([129, 1, 257], 16, 1, 128, 64), ([200, 70], 20, 1, 80, 64), ([513], 34, 2, 112, 64)])
def test_lengths_heads_and_pages(dev, dtype, stored, lengths, H, Hk, d, page):
    _check(dev, dtype, stored, lengths, H, Hk, d, page)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [8, 24, 40, 56, 72, 104, 120])
def test_head_sizes_between_powers_of_two(dev, dtype, d):
    _check(dev, dtype, dtype, [70, 1, 33], 4, 2, d, 64)


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("lengths,H,Hk,d,page", [([5000], 8, 2, 64, 64), ([1, 3000, 257, 1500], 4, 4, 32, 256), ([2305], 16, 1, 128, 128)])
def test_long_streams_in_pieces(dev, dtype, stored, lengths, H, Hk, d, page):
    _check(dev, dtype, stored, lengths, H, Hk, d, page, spare=40)


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("lengths,H,Hk,d,buckets,maxd", [([1, 40, 700], 6, 2, 32, 16, 20), ([129, 2], 20, 1, 64, 32, 128),
                                                       ([3000], 2, 2, 128, 8, 1000)])
def test_bias(dev, dtype, stored, lengths, H, Hk, d, buckets, maxd):
    _check(dev, dtype, stored, lengths, H, Hk, d, 64, buckets, maxd)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.5])
@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, BF16), (F16, I8), (BF16, E4)], ids=["f32", "bf16", "f16-i8", "bf16-e4m3"])
def test_scales(dev, dtype, stored, scale):
    _check(dev, dtype, stored, [100, 1, 333], 4, 2, 64, 64, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_it_is_window_attention_s_last_row(dev, dtype):
    """Token by token over a pool of the tokens' type: the rows of the whole history's forward, within the two's bounds."""
    from gdl_amd.functional import PagedCache, paged_attention_step, window_attention
    gen = torch.Generator().manual_seed(8)
    T, H, Hk, d = 150, 4, 2, 32
    q, k, v = (torch.randn(T, h, d, generator=gen).to(dtype).to(dev) for h in (H, Hk, Hk))
    bias = torch.randn(8, H, generator=gen).to(dtype).to(dev)
    rows = window_attention(q, k, v, (-1, 0), bias=bias, max_distance=40)
    _, tol = ref.attend(q, k.double().cpu(), v.double().cpu(), 0, dtype, table=bias, maxd=40)
    cache = PagedCache.empty(3, Hk, d, dtype=dtype, device=dev)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    for t in range(T):
        out = paged_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], cache, table, torch.tensor([t], device=dev), bias=bias, max_distance=40)
        ref.assert_near(out[0], rows[t].double().cpu(), 2 * tol[t], t)


@pytest.mark.parametrize("stored", [F32, I8], ids=["f32", "i8"])
@pytest.mark.parametrize("columns", [3, 60])
def test_streams_without_a_token_or_a_page(dev, stored, columns):
    """Left alone at negative positions, NaN where a page is not there, the other streams as ever; few pieces
    and many."""
    from gdl_amd.functional import PagedCache, paged_attention_step
    gen = torch.Generator().manual_seed(6)
    Hk, H, d, B = 2, 4, 32, 6
    cache = PagedCache.empty(20, Hk, d, dtype=stored, device=dev)
    k, v = (torch.randn(20 * 64, Hk, d, generator=gen).to(dev) for _ in range(2))
    cache.write(k, v, torch.arange(20, dtype=torch.int32, device=dev).view(1, 20))
    table = torch.full((B, columns), -1, dtype=torch.int32)
    table[:, :3] = torch.arange(18).view(B, 3)
    table[2, 1] = 20     # stream 2: a page of its history is outside the pool
    table[3, 2] = -7     # stream 3: its new token's page is
    want_pool = ref.copy(cache)
    pos = torch.tensor([150, -1, 150, 150, columns * 64 + 5, 0])
    q, k1, v1 = (torch.randn(B, h, d, generator=gen).to(dev) for h in (H, Hk, Hk))
    for b, (page, slot) in {0: (2, 22), 2: (8, 22), 5: (15, 0)}.items():
        ref.put(want_pool, "k", page, slot, k1[b]), ref.put(want_pool, "v", page, slot, v1[b])
    out = paged_attention_step(q, k1, v1, cache, table.to(dev), pos.to(dev))
    assert (out[1] == 0).all() and out[2:5].isnan().all() and out[[0, 5]].isfinite().all()
    ref.same(cache, want_pool)
    for b, first in ((0, 0), (5, 15 * 64)):
        n = int(pos[b])
        K, V = (torch.cat([ref.stored(x[first:first + n], stored), ref.stored(y[b:b + 1], stored)]) for x, y in ((k, k1), (v, v1)))
        ref.assert_near(out[b:b + 1], *ref.attend(q[b:b + 1], K, V, n, stored), b)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_infinities_and_lowest_values(dev, dtype):
    """Keys with scores of -inf have no weight, alone they give NaN; an infinite value shows where it is seen
    and only there; keys that all have the lowest finite bias weigh alike."""
    from gdl_amd.functional import PagedCache, paged_attention_step
    Hk, d, n = 1, 24, 100
    gen = torch.Generator().manual_seed(7)
    cache = PagedCache.empty(4, Hk, d, dtype=dtype, device=dev)
    k, v = (torch.randn(n, Hk, d, generator=gen).to(dtype).to(dev) for _ in range(2))
    q = torch.ones(2, 1, d, dtype=dtype, device=dev)
    k[10, 0, 3] = -math.inf
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    cache.write(torch.cat([k, k]), torch.cat([v, v]), table, torch.tensor([0, n, 2 * n], device=dev))
    all_low = torch.full((n, Hk, d), -math.inf, dtype=dtype, device=dev)
    cache.write(all_low, v, table[1:])
    new = torch.stack([k[20], all_low[0]]), torch.stack([v[20], v[20]])
    out = paged_attention_step(q, *new, cache, table, torch.tensor([n, n], device=dev))
    keep = [i for i in range(n) if i != 10] + [20]
    ref.assert_near(out[:1], *ref.attend(q[:1], k[keep].double().cpu(), v[keep].double().cpu(), n - 1, dtype))
    assert out[1].isnan().all()
    low = torch.full((4, 1), torch.finfo(dtype).min, dtype=dtype, device=dev)
    out = paged_attention_step(torch.zeros_like(q[:1]), k[:1], v[:1], cache, table[:1], torch.tensor([5], device=dev), bias=low, max_distance=9)
    V = torch.cat([v[:5], v[:1]]).double().cpu()
    ref.assert_near(out, *ref.attend(torch.zeros_like(q[:1]), torch.zeros_like(V), V, 5, dtype))
    v2 = v.clone()
    v2[30, 0, 2] = math.inf
    cache.write(k, v2, table[:1])
    out = paged_attention_step(q[:1], k[:1], v[:1], cache, table[:1], torch.tensor([40], device=dev))
    assert not out[0, 0, 2].isfinite() and out[0, 0, [i for i in range(d) if i != 2]].isfinite().all()
    out = paged_attention_step(q[:1], k[:1], v[:1], cache, table[:1], torch.tensor([30], device=dev))
    assert out.isfinite().all()


def test_large_scores(dev):
    """Scores of some thousand: no overflow, the largest takes all."""
    _check(dev, F32, F32, [700, 3], 4, 1, 64, 64, scale=40.0)
    _check(dev, BF16, E4, [700, 3], 4, 1, 64, 64, scale=40.0)


def test_captured_steps_and_shared_scratch(dev):
    """Two graphs of steps on two caches, replayed in turn with eager calls of other sizes between them."""
    from gdl_amd.functional import PagedCache, paged_attention_step
    gen = torch.Generator().manual_seed(11)
    Hk, H, d, n = 2, 8, 64, 3000
    caches = [PagedCache.empty(60, Hk, d, dtype=t, device=dev) for t in (BF16, I8)]
    table = torch.randperm(60, generator=gen).int().view(1, 60).to(dev)
    k, v = (torch.randn(n, Hk, d, generator=gen).bfloat16().to(dev) for _ in range(2))
    for c in caches:
        c.write(k, v, table)
    q, k1, v1 = (torch.randn(1, h, d, generator=gen).bfloat16().to(dev) for h in (H, Hk, Hk))
    pos = torch.tensor([n], device=dev)
    graphs, outs = [], []
    for c in caches:
        paged_attention_step(q, k1, v1, c, table, pos)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(paged_attention_step(q, k1, v1, c, table, pos))
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=gen)), k1.copy_(torch.randn(k1.shape, generator=gen)), pos.add_(1)
        for g in graphs:
            g.replay()
        for c, out in zip(caches, outs):
            again = paged_attention_step(q, k1, v1, c, table, pos)
            torch.cuda.synchronize()
            assert torch.equal(out, again)


def test_results_are_the_same_from_run_to_run(dev):
    assert all(torch.equal(_check(dev, F16, E4, [2000, 30], 8, 2, 64, 64), _check(dev, F16, E4, [2000, 30], 8, 2, 64, 64)) for _ in range(3))


def test_strided_inputs_and_offsets_of_other_types(dev):
    from gdl_amd.functional import paged_attention_step
    gen = torch.Generator().manual_seed(12)
    lengths = [50, 1, 130]
    cache, table = _filled(dev, lengths, 2, 32, 64, F32, F32, gen)
    k, v = (torch.randn(178, 2, 32, generator=gen).to(dev) for _ in range(2))
    cache.write(k, v, table, torch.tensor([0, 49, 49, 178], device=dev))
    x = torch.randn(3, 8, 32, generator=gen).to(dev)  # one projection's output
    pos = torch.tensor([49, 0, 129], device=dev)
    a = paged_attention_step(x[:, :4], x[:, 4:6], x[:, 6:], cache, table, pos)
    b = paged_attention_step(x[:, :4].contiguous(), x[:, 4:6].clone(), x[:, 6:].contiguous(), cache, table.t().contiguous().t(), pos.int())
    odd = torch.zeros(3, 4, 33, device=dev)
    odd[..., 1:] = x[:, :4]
    c = paged_attention_step(odd[..., 1:], x[:, 4:6], x[:, 6:], cache, table, pos)
    assert torch.equal(a, b) and torch.equal(a, c)
