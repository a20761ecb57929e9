"""GPU tests of paged caches: tokens written to pages and read back, bit by bit against the definition."""

import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, I8), (F16, I8), (F32, E4), (BF16, E4), (F16, E4)]
IDS = [f"{str(a)[6:]}-{str(b)[6:]}" for a, b in TYPES]


def _cache(dev, pages, heads, d, page, stored, gen):
    """A pool of random bits that read back as finite numbers."""
    from gdl_amd.functional import PagedCache
    cache = PagedCache.empty(pages, heads, d, page=page, dtype=stored, device=dev)
    for t in (cache.k, cache.v):
        x = torch.randn(t.shape, generator=gen) * (50 if stored is I8 else 1)
        t.copy_(x.to(stored))
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.copy_(torch.rand(t.shape, generator=gen))
    return cache


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("lengths,starts,heads,d,page", [
    ([1], [0], 1, 16, 64), ([1], [63], 2, 32, 64), ([64, 65], [0, 0], 1, 64, 64), ([3, 0, 200, 1], [62, 5, 1, 128], 3, 48, 128),
    ([130, 7, 300], [127, 64, 1], 2, 128, 64), ([500], [190], 1, 80, 192), ([2] * 70, [i % 65 for i in range(70)], 1, 16, 64)])
def test_write_and_read(dev, dtype, stored, lengths, starts, heads, d, page):
    print(dtype, stored, lengths, starts, heads, d, page, flush=True)
    gen = torch.Generator().manual_seed(len(lengths) + d)
    ends = [a + n for a, n in zip(starts, lengths)]
    table = ref.random_table(ends, page, sum(-(-n // page) for n in ends) + 2, gen)
    cache = _cache(dev, sum(-(-n // page) for n in ends) + 2, heads, d, page, stored, gen)
    lead, tail = 3, 70  # tokens of no sequence on both sides
    T = lead + sum(lengths) + tail
    x = torch.randn(T, 2 * heads + 1, d, generator=gen).to(dtype)
    x[:, :, 0] *= 7
    x = x.to(dev)
    k, v = x[:, :heads], x[:, heads + 1:]
    ptr = torch.tensor([lead] + lengths).cumsum(0)
    want = ref.copy(cache)
    values = torch.zeros(2, T, heads, d, dtype=torch.float64)
    for b, (a, n) in enumerate(zip(starts, lengths)):
        for i in range(n):
            t, at = int(ptr[b]) + i, (int(table[b, (a + i) // page]), (a + i) % page)
            for m, (name, rows) in enumerate((("k", k), ("v", v))):
                ref.put(want, name, *at, rows[t])
                values[m, t] = ref.get(want, name, *at)
    args = table.to(dev), ptr.to(dev)
    start = torch.tensor(starts, device=dev)
    cache.write(k, v, *args, start)
    ref.same(cache, want)
    for out in {dtype, BF16 if stored in ref.MOST else dtype}:
        got = cache.read(*args, T, start=start, dtype=out)
        for m in range(2):
            assert torch.equal(got[m].cpu(), values[m].float().to(out)), (out, m)


@pytest.mark.parametrize("stored", [F16, I8, E4], ids=["f16", "i8", "e4m3"])
def test_tokens_without_a_page_are_left_out(dev, stored):
    gen = torch.Generator().manual_seed(3)
    cache = _cache(dev, 6, 2, 32, 64, stored, gen)
    want = ref.copy(cache)
    k, v = (torch.randn(360, 2, 32, generator=gen).half().to(dev) for _ in range(2))
    # stream 0: no second page; 1: beyond its table; 2: from before its first position; 3: far beyond anything
    table = torch.tensor([[1, -1, 2], [3, 4, 5], [0, 6, 1 << 30], [-5, 7, 9]], dtype=torch.int32)
    ptr, start = torch.tensor([0, 150, 250, 300, 360]), torch.tensor([0, 100, -20, 1 << 60])
    lost = torch.zeros(360, dtype=torch.bool)
    for b in range(4):
        for t in range(int(ptr[b]), int(ptr[b + 1])):
            at = int(start[b]) + t - int(ptr[b])
            page = int(table[b, at // 64]) if 0 <= at < 192 else -1
            if 0 <= page < 6:
                ref.put(want, "k", page, at % 64, k[t]), ref.put(want, "v", page, at % 64, v[t])
            else:
                lost[t] = True
    assert lost.any() and not lost.all()
    args = table.to(dev), ptr.to(dev)
    cache.write(k, v, *args, start.to(dev))
    ref.same(cache, want)
    for x in cache.read(*args, 360, start=start.to(dev), dtype=F16):
        assert torch.equal(x.isnan().all(-1).all(-1).cpu(), lost) and torch.equal(x.isnan().any(-1).any(-1).cpu(), lost)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("stored", [I8, E4], ids=["i8", "e4m3"])
def test_rows_at_the_ends_of_their_range(dev, dtype, stored):
    """Zeros, the type's least and largest values, infinities and NaN, and values on the borders of codes."""
    from gdl_amd.functional import PagedCache
    info, d = torch.finfo(dtype), 32
    rows = torch.randn(14, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    rows[0] = 0
    rows[1] *= info.tiny
    rows[2] = (rows[2].float() * 2.0 ** -101).to(dtype)
    rows[3] = (rows[3].float().clamp(-1, 1) * info.max).to(dtype)
    rows[3, 0] = info.max
    rows[4, 3] = math.inf
    rows[5, 31] = -math.inf
    rows[6, 7] = math.nan
    rows[7] = torch.arange(d).to(dtype) / 2  # many halves of a code
    rows[7, 0] = 127
    rows[8] = torch.arange(d).to(dtype) * 28 + 14
    rows[9] = -rows[8]
    rows[10] = (2.0 ** -torch.arange(d).float()).to(dtype)
    rows[11] = (1.5 * 2.0 ** -torch.arange(d).float()).to(dtype)
    rows[12] = -0.0
    rows[13, 1:] = 0
    k = rows.view(14, 1, d).to(dev)
    cache = PagedCache.empty(1, 1, d, dtype=stored, device=dev)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).zero_()
    cache.k_scale.zero_(), cache.v_scale.zero_()
    want = ref.copy(cache)
    for i in range(14):
        ref.put(want, "k", 0, i, k[i]), ref.put(want, "v", 0, i, k[i])
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    cache.write(k, k.clone(), table)
    for name in ("k_scale", "v_scale"):  # any NaN is one
        g, w = getattr(cache, name).cpu(), want.pop(name)
        assert torch.equal(g.isnan(), w.isnan()) and torch.equal(g.nan_to_num(9), w.nan_to_num(9))
    for name in ("k", "v"):  # -0 and 0 are one value
        assert torch.equal(getattr(cache, name).cpu().float(), want[name].float())
    for x in cache.read(table, None, 14, dtype=F32):
        got = x[:, 0].cpu()
        assert got[4:7].isnan().all() and got[0].eq(0).all() and got[12].eq(0).all()
        fine = [i for i in range(14) if i not in (4, 5, 6)]
        assert torch.equal(got[fine], ref.stored(rows, stored)[fine].float())


def test_shared_strides_and_other_streams(dev):
    """Rows that are not on 16 bytes, a table that is a slice of a wider one, offsets of other whole types, a
    side stream."""
    gen = torch.Generator().manual_seed(9)
    cache, other = (_cache(dev, 6, 2, 24, 64, F32, torch.Generator().manual_seed(4)) for _ in range(2))
    k, v = (torch.randn(100, 2, 24, generator=gen).to(dev) for _ in range(2))
    wide = torch.tensor([[9, 2, 0, 3], [9, 5, 1, 4]], dtype=torch.int32, device=dev)
    ptr = torch.tensor([0, 37, 100])
    cache.write(k, v, wide[:, 1:], ptr.to(dev))
    odd = torch.randn(100, 2, 25, generator=gen).to(dev)
    odd[..., 1:] = k
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other.write(odd[..., 1:], v.transpose(0, 1).contiguous().transpose(0, 1), wide.t().contiguous().t()[:, 1:], ptr.int().to(dev),
                    torch.zeros(2, dtype=torch.int32, device=dev))
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)


def test_beyond_32_bit_offsets(dev):
    """Pages whose elements lie beyond 2^31 of the pool."""
    from gdl_amd.functional import PagedCache
    heads, d, page = 8, 128, 256
    pages = (1 << 31) // (heads * d * page) + 40
    cache = PagedCache.empty(pages, heads, d, page=page, dtype=I8, device=dev)
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(600, heads, d, generator=gen).bfloat16().to(dev) for _ in range(2))
    table = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32, device=dev)
    cache.write(k, v, table)
    got = cache.read(table, None, 600, dtype=F32)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x.cpu(), ref.stored(y, I8).float())


def test_captured_and_replayed(dev):
    gen = torch.Generator().manual_seed(5)
    cache, eager = (_cache(dev, 9, 2, 64, 64, E4, torch.Generator().manual_seed(4)) for _ in range(2))
    k, v = (torch.randn(90, 2, 64, generator=gen).bfloat16().to(dev) for _ in range(2))
    table = torch.randperm(9, generator=gen).int().view(3, 3).to(dev)
    ptr, start = torch.tensor([0, 30, 31, 90], device=dev), torch.tensor([5, 60, 100], device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, table, ptr, start)
        out = cache.read(table, ptr, 90, start=start)
    for n in range(3):
        k.copy_(torch.randn(k.shape, generator=gen)), start.add_(n)
        graph.replay()
        eager.write(k, v, table, ptr, start)
        want = eager.read(table, ptr, 90, start=start)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        ref.same(cache, ref.copy(eager))
