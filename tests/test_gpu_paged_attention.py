"""GPU tests of attention of prompts and their pieces over paged caches, against the definition in float64."""

import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, I8), (F16, I8), (F32, E4), (BF16, E4), (F16, E4)]
IDS = [f"{str(a)[6:]}-{str(b)[6:]}" for a, b in TYPES]


def _poisoned(dev, pages, heads, d, page, stored):
    """A pool of which every place without a token reads as NaN."""
    from gdl_amd.functional import PagedCache
    cache = PagedCache.empty(pages, heads, d, page=page, dtype=stored, device=dev)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0xFF) if stored is not I8 else t.fill_(-128)
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(math.nan)
    return cache


def _check(dev, dtype, stored, spans, H, Hk, d, page, buckets=0, maxd=128, scale=None, lead=0, tail=0, spare=1):
    """spans: (tokens before, new tokens) of each stream."""
    from gdl_amd.functional import paged_attention
    print(dtype, stored, spans, H, Hk, d, page, buckets, flush=True)
    gen = torch.Generator().manual_seed(sum(map(sum, spans)) + H + d)
    ends = [a + n for a, n in spans]
    pages = sum(-(-n // page) for n in ends) + 2
    table = ref.random_table(ends, page, pages, gen, spare).to(dev)
    cache = _poisoned(dev, pages, Hk, d, page, stored)
    k, v = ([torch.randn(n, Hk, d, generator=gen).to(dtype).to(dev) for n in ends] for _ in range(2))
    cache.write(torch.cat(k), torch.cat(v), table, torch.tensor([0] + ends).cumsum(0).to(dev))
    news = [n for _, n in spans]
    T = lead + sum(news) + tail
    x = torch.randn(T, H + 2 * Hk, d, generator=gen).to(dtype).to(dev)  # one projection's output
    q = x[:, :H]
    bias = torch.randn(buckets, H, generator=gen).to(dtype).to(dev) if buckets else None
    ptr, start = torch.tensor([lead] + news).cumsum(0), torch.tensor([a for a, _ in spans])
    out = paged_attention(q, cache, table, ptr.to(dev), start.to(dev), bias=bias, max_distance=maxd, scale=scale)
    for b, (a, n) in enumerate(spans):
        if n:
            rows = slice(int(ptr[b]), int(ptr[b + 1]))
            want, tol = ref.attend(q[rows], ref.stored(k[b], stored), ref.stored(v[b], stored), a, stored, scale, bias, maxd)
            ref.assert_near(out[rows], want, tol, (b, a, n))
    assert (out[:lead] == 0).all() and (out[T - tail:] == 0).all()
    return out


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("spans,H,Hk,d,page", [
    ([(0, 1)], 1, 1, 16, 64), ([(0, 64), (0, 65), (5, 1)], 4, 2, 32, 64), ([(63, 2), (0, 0), (10, 200), (1, 31)], 4, 1, 64, 128),
    ([(0, 300), (257, 5)], 3, 3, 48, 192), ([(100, 130), (0, 33)], 16, 2, 128, 64), ([(70, 129)], 6, 1, 80, 64),
    ([(3, 40), (64, 64)], 8, 1, 112, 64)])
def test_packets_heads_and_pages(dev, dtype, stored, spans, H, Hk, d, page):
    _check(dev, dtype, stored, spans, H, Hk, d, page, lead=2, tail=67)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [8, 24, 40, 56, 72, 104, 120])
def test_head_sizes_between_powers_of_two(dev, dtype, d):
    _check(dev, dtype, dtype, [(20, 70), (0, 1)], 4, 2, d, 64)


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("spans,H,Hk,d,page", [([(3000, 3)], 4, 2, 64, 64), ([(2500, 40), (0, 7), (700, 1)], 2, 2, 32, 256),
                                              ([(1100, 20)], 16, 2, 128, 64)])
def test_long_histories_in_pieces(dev, dtype, stored, spans, H, Hk, d, page):
    _check(dev, dtype, stored, spans, H, Hk, d, page, lead=1, tail=1, spare=30)


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("spans,H,Hk,d,buckets,maxd", [([(0, 90), (100, 3)], 6, 2, 32, 16, 20), ([(129, 200)], 4, 1, 64, 32, 128),
                                                      ([(1500, 9)], 2, 2, 128, 8, 1000)])
def test_bias(dev, dtype, stored, spans, H, Hk, d, buckets, maxd):
    _check(dev, dtype, stored, spans, H, Hk, d, 64, buckets, maxd)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.5])
@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, BF16), (F16, I8), (BF16, E4)], ids=["f32", "bf16", "f16-i8", "bf16-e4m3"])
def test_scales(dev, dtype, stored, scale):
    _check(dev, dtype, stored, [(40, 100), (0, 3)], 4, 2, 64, 64, scale=scale)


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
def test_later_tokens_may_hold_anything(dev, dtype, stored):
    """A token's row depends on no later one, whatever it holds; those that see an infinity or NaN show it."""
    from gdl_amd.functional import PagedCache, paged_attention
    Hk, H, d, n = 2, 4, 48, 150
    gen = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(dtype).to(dev) for h in (H, Hk, Hk))
    clean = PagedCache.empty(3, Hk, d, dtype=stored, device=dev)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    clean.write(k, v, table)
    want = paged_attention(q, clean, table)
    for row, value, of_k in ((40, math.inf, False), (70, math.nan, False), (100, -math.inf, True), (149, math.nan, True), (64, -math.inf, False)):
        cache = PagedCache.empty(3, Hk, d, dtype=stored, device=dev)
        k2, v2 = k.clone(), v.clone()
        (k2 if of_k else v2)[row, 1, 7] = value
        cache.write(k2, v2, table)
        out = paged_attention(q, cache, table)
        assert torch.equal(out[:row], want[:row]), (row, value, of_k)
        assert torch.equal(out[:, :2], want[:, :2])  # the other key head's
        if not of_k:
            wide = stored in ref.MOST  # its scale is NaN: so is the row
            for t in range(row, n):
                bad = ~out[t, 2:].isfinite()
                assert bad.all() if wide else bad[:, 7].all() and not bad[:, :7].any() and not bad[:, 8:].any(), (row, t)


@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, BF16), (F16, I8)], ids=["f32", "bf16", "f16-i8"])
@pytest.mark.parametrize("columns", [3, 50])
def test_tokens_without_a_page(dev, dtype, stored, columns):
    """NaN from the page that is not there on, 0 at negative positions, the tokens before as ever; in one piece and several."""
    from gdl_amd.functional import PagedCache, paged_attention
    Hk, H, d, B = 1, 2, 32, 4
    gen = torch.Generator().manual_seed(5)
    cache = PagedCache.empty(12, Hk, d, dtype=stored, device=dev)
    k, v = (torch.randn(12 * 64, Hk, d, generator=gen).to(dtype).to(dev) for _ in range(2))
    cache.write(k, v, torch.arange(12, dtype=torch.int32, device=dev).view(1, 12))
    table = torch.full((B, columns), -1, dtype=torch.int32)
    table[:, :3] = torch.arange(12).view(B, 3)
    table[1, 1] = 12
    starts, news = [0, 20, -30, columns * 64 - 2], [150, 100, 80, 5]
    ptr = torch.tensor([0] + news).cumsum(0)
    q = torch.randn(int(ptr[-1]), H, d, generator=gen).to(dtype).to(dev)
    out = paged_attention(q, cache, table.to(dev), ptr.to(dev), torch.tensor(starts, device=dev))
    rows = [slice(int(a), int(b)) for a, b in zip(ptr[:-1], ptr[1:])]
    K, V = ref.stored(k, stored), ref.stored(v, stored)
    ref.assert_near(out[rows[0]], *ref.attend(q[rows[0]], K[:150], V[:150], 0, stored), 0)
    ref.assert_near(out[120 + 30:120 + 30 + 44], *ref.attend(q[150:194], K[192:256], V[192:256], 20, stored), 1)
    assert out[194:250].isnan().all()
    assert (out[250:280] == 0).all()
    ref.assert_near(out[280:330], *ref.attend(q[280:330], K[384:434], V[384:434], 0, stored), 2)
    far = out[rows[3]]
    assert far[2:].isnan().all() and (far[:2].isnan().all() if columns > 3 else far[:2].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_scores_of_minus_infinity_alone(dev, dtype):
    from gdl_amd.functional import PagedCache, paged_attention
    cache = PagedCache.empty(1, 1, 16, dtype=dtype, device=dev)
    k, v = torch.full((5, 1, 16), -math.inf, dtype=dtype, device=dev), torch.ones(5, 1, 16, dtype=dtype, device=dev)
    k[3] = 0
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    cache.write(k, v, table)
    out = paged_attention(torch.ones(5, 1, 16, dtype=dtype, device=dev), cache, table)
    assert out[:3].isnan().all() and (out[3:] == 1).all()


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
def test_pieces_steps_and_the_whole_agree(dev, dtype, stored):
    """One stream in one piece, in uneven pieces and token by token: rows within the sum of their bounds."""
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(8)
    T, H, Hk, d = 140, 4, 2, 32
    q, k, v = (torch.randn(T, h, d, generator=gen).to(dtype).to(dev) for h in (H, Hk, Hk))
    bias = torch.randn(8, H, generator=gen).to(dtype).to(dev)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    want, tol = ref.attend(q, ref.stored(k, stored), ref.stored(v, stored), 0, stored, table=bias, maxd=40)
    caches = [PagedCache.empty(3, Hk, d, dtype=stored, device=dev) for _ in range(3)]
    caches[0].write(k, v, table)
    ref.assert_near(paged_attention(q, caches[0], table, bias=bias, max_distance=40), want, tol)
    for a, b in ((0, 1), (1, 50), (50, 64), (64, 140)):
        at = torch.tensor([a], device=dev)
        caches[1].write(k[a:b], v[a:b], table, None, at)
        ref.assert_near(paged_attention(q[a:b], caches[1], table, None, at, bias=bias, max_distance=40), want[a:b], tol[a:b], (a, b))
    for t in range(T):
        out = paged_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], caches[2], table, torch.tensor([t], device=dev), bias=bias, max_distance=40)
        ref.assert_near(out, want[t:t + 1], tol[t:t + 1], t)
    for c in caches[1:]:
        a, b = caches[0].read(table, None, T, dtype=dtype), c.read(table, None, T, dtype=dtype)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_and_replayed(dev):
    from gdl_amd.functional import PagedCache, paged_attention
    gen = torch.Generator().manual_seed(11)
    Hk, H, d, n = 2, 8, 64, 2000
    cache = PagedCache.empty(40, Hk, d, dtype=I8, device=dev)
    table = torch.randperm(40, generator=gen).int().view(1, 40).to(dev)
    k, v = (torch.randn(n + 60, Hk, d, generator=gen).bfloat16().to(dev) for _ in range(2))
    cache.write(k, v, table)
    q, start = torch.randn(50, H, d, generator=gen).bfloat16().to(dev), torch.tensor([n], device=dev)
    paged_attention(q, cache, table, None, start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, cache, table, None, start)
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=gen)), start.add_(1)
        graph.replay()
        want = paged_attention(q, cache, table, None, start)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_beyond_32_bit_offsets(dev):
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    heads, d, page = 8, 128, 256
    pages = (1 << 31) // (heads * d * page) + 40
    cache = PagedCache.empty(pages, heads, d, page=page, dtype=E4, device=dev)
    gen = torch.Generator().manual_seed(2)
    k, v, q = (torch.randn(300, heads, d, generator=gen).bfloat16().to(dev) for _ in range(3))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    cache.write(k, v, table)
    want, tol = ref.attend(q, ref.stored(k, E4), ref.stored(v, E4), 0, E4)
    ref.assert_near(paged_attention(q, cache, table), want, tol)
    out = paged_attention_step(q[-1:], k[-1:], v[-1:], cache, table, torch.tensor([299], device=dev))
    ref.assert_near(out, want[-1:], tol[-1:])
