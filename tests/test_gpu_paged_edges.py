"""GPU tests of calls at the edges of what paged caches take."""

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, I8), (F16, E4)], ids=["f32", "bf16-i8", "f16-e4m3"])
def test_no_streams(dev, dtype, stored):
    """A serving loop whose last stream has ended: an empty result, and the pool as it was."""
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    cache = PagedCache.empty(2, 2, 32, dtype=stored, device=dev)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            t.view(torch.uint8).fill_(7)
    want = ref.copy(cache)
    q, k = torch.empty(0, 4, 32, dtype=dtype, device=dev), torch.empty(0, 2, 32, dtype=dtype, device=dev)
    at = torch.empty(0, dtype=torch.int64, device=dev)
    for columns in (1, 5000):
        table = torch.empty(0, columns, dtype=torch.int32, device=dev)
        bias = torch.zeros(8, 4, dtype=dtype, device=dev)
        assert paged_attention_step(q, k, k, cache, table, at).shape == (0, 4, 32)
        assert paged_attention_step(q, k, k, cache, table, at, bias=bias, max_distance=20).shape == (0, 4, 32)
    table, ptr = torch.zeros(2, 3, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    cache.write(k, k, table, ptr)
    assert paged_attention(q, cache, table, ptr).shape == (0, 4, 32)
    assert all(x.shape == (0, 2, 32) for x in cache.read(table, ptr, 0, dtype=dtype))
    ref.same(cache, want)


@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, I8), (F16, E4)],
                         ids=["f32", "bf16", "f16", "f32-i8", "bf16-i8", "f16-e4m3"])
@pytest.mark.parametrize("d", [32, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_scores_far_out(dev, dtype, stored, d, bias):
    """Scores up to 2^37, where float32's steps are far above 1: which keys weigh most is up to the order of its sums (error
    bound e (d + 8) S), and a row still is a mean of the values that it sees, weights above 0 and a sum of 1."""
    from attention_ref import SPACING, UNIT
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(d)
    n, H, Hk = 300, 4, 2
    cache = PagedCache.empty(5, Hk, d, dtype=stored, device=dev)
    table = torch.tensor([[3, 1, 0, 4, 2]], dtype=torch.int32, device=dev)
    q = (6e4 * (0.1 + 0.9 * torch.rand(n, H, 1, generator=gen))).expand(n, H, d).to(dtype).to(dev)
    k = (6e4 * (0.1 + 0.9 * torch.rand(1, Hk, 1, generator=gen))).expand(n, Hk, d).to(dtype).to(dev)
    v = torch.randn(n, Hk, d, generator=gen).to(dtype).to(dev)
    cache.write(k, v, table)
    kw = dict(bias=torch.full((8, H), 0.5, dtype=dtype, device=dev), max_distance=20) if bias else {}
    V = ref.stored(v, stored).repeat_interleave(H // Hk, 1)
    lo, hi = V.cummin(0).values, V.cummax(0).values

    def check(out, lo, hi):
        x, size = out.double().cpu(), torch.maximum(lo.abs(), hi.abs())
        slack = SPACING[dtype] + (2 * UNIT[dtype] + (n + 8) * 2.0 ** -24) * size  # the weights' and the output's rounding
        assert x.isfinite().all(), int((~x.isfinite()).sum())
        assert (x >= lo - slack).all() and (x <= hi + slack).all()

    check(paged_attention(q, cache, table, **kw), lo, hi)
    at = torch.tensor([n - 1], device=dev)
    check(paged_attention_step(q[-1:], k[-1:], v[-1:], cache, table, at, **kw), lo[-1:], hi[-1:])


@pytest.mark.parametrize("dtype,stored,unit", [(BF16, BF16, 2.0 ** -16), (F16, F16, 2.0 ** -22), (BF16, I8, 2.0 ** -16), (BF16, E4, 2.0 ** -16)],
                         ids=["bf16", "f16", "bf16-i8", "bf16-e4m3"])
@pytest.mark.parametrize("columns", [12, 300, 9000])
@pytest.mark.parametrize("new", [5, 300])
def test_weights_of_short_prompts_do_not_hang_on_the_table(dev, dtype, stored, unit, columns, new):
    """Weights of a call of few queries over a short history are kept in two parts, however many tokens the table has room for."""
    from gdl_amd.functional import PagedCache, paged_attention
    gen = torch.Generator().manual_seed(new)
    n, H, Hk, d = 700, 6, 2, 64
    cache = PagedCache.empty(12, Hk, d, dtype=stored, device=dev)
    table = torch.full((1, columns), -1, dtype=torch.int32)
    table[0, :12] = torch.randperm(12, generator=gen).int()
    table = table.to(dev)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(dtype).to(dev) for h in (H, Hk, Hk))
    cache.write(k, v, table)
    out = paged_attention(q[-new:], cache, table, None, torch.tensor([n - new], device=dev))
    ref.assert_near(out, *ref.attend(q[-new:], ref.stored(k, stored), ref.stored(v, stored), n - new, stored, unit=unit))


@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, BF16), (F16, F16), (F16, I8)], ids=["f32", "bf16", "f16", "f16-i8"])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_every_size(dev, dtype, stored, sign):
    """Scores from 2^14 to 2^40 and their negatives, several in each power of two: rows are means of what they see."""
    from attention_ref import SPACING, UNIT
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(3)
    n, H, d = 200, 8, 32
    cache = PagedCache.empty(4, 1, d, dtype=stored, device=dev)
    table = torch.tensor([[3, 1, 0, 2]], dtype=torch.int32, device=dev)
    q = (0.5 + 0.5 * torch.rand(n, H, 1, generator=gen)).expand(n, H, d).to(dtype).to(dev)
    k, v = torch.ones(n, 1, d, dtype=dtype, device=dev), torch.randn(n, 1, d, generator=gen).to(dtype).to(dev)
    cache.write(k, v, table)
    V = ref.stored(v, stored).expand(n, H, d)
    lo, hi = V.cummin(0).values, V.cummax(0).values
    slack = SPACING[dtype] + (2 * UNIT[dtype] + (n + 8) * 2.0 ** -24) * torch.maximum(lo.abs(), hi.abs())
    at = torch.tensor([n - 1], device=dev)
    for e in range(14, 41):
        scale = sign * 2.0 ** e / d
        x = paged_attention(q, cache, table, scale=scale).double().cpu()
        assert x.isfinite().all(), (e, int((~x.isfinite()).sum()))
        assert (x >= lo - slack).all() and (x <= hi + slack).all(), e
        x = paged_attention_step(q[-1:], k[-1:], v[-1:], cache, table, at, scale=scale).double().cpu()
        assert x.isfinite().all() and (x >= lo[-1:] - slack[-1:]).all() and (x <= hi[-1:] + slack[-1:]).all(), e
