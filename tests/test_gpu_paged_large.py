"""Calls that fill the card: the kernels of prompts with more than 512 tiles of 128 queries (by heads), calls in which short
sequences have weights in two parts and long ones in one, and steps with more rows than workgroups (1024 at most)."""

import pytest
import torch

import paged_ref as ref
from test_gpu_paged_attention import _poisoned

pytestmark = pytest.mark.gpu
F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, I8), (BF16, E4), (F16, I8), (F16, E4)]
IDS = [f"{str(a)[6:]}-{str(b)[6:]}" for a, b in TYPES]


def _prompt(dev, dtype, stored, spans, H, Hk, d, buckets, spare):
    """Rows at the ends and on both sides of tiles and pages, against the definition."""
    from gdl_amd.functional import paged_attention
    gen = torch.Generator().manual_seed(d + H)
    ends = [a + n for a, n in spans]
    pages = sum(-(-n // 64) for n in ends) + 2
    table = ref.random_table(ends, 64, pages, gen, spare).to(dev)
    cache = _poisoned(dev, pages, Hk, d, 64, stored)
    k, v = ([torch.randn(n, Hk, d, generator=gen).to(dtype).to(dev) for n in ends] for _ in range(2))
    cache.write(torch.cat(k), torch.cat(v), table, torch.tensor([0] + ends).cumsum(0).to(dev))
    news = [n for _, n in spans]
    q = torch.randn(sum(news), H, d, generator=gen).to(dtype).to(dev)
    bias = torch.randn(buckets, H, generator=gen).to(dtype).to(dev) if buckets else None
    ptr, start = torch.tensor([0] + news).cumsum(0), torch.tensor([a for a, _ in spans])
    out = paged_attention(q, cache, table, ptr.to(dev), start.to(dev), bias=bias, max_distance=100)
    assert out.isfinite().all()
    for b, (a, n) in enumerate(spans):
        K, V = ref.stored(k[b], stored), ref.stored(v[b], stored)
        for i in sorted({0, 1, 15, 16, 31, 32, 63, 64, 127, 128, n // 2, n - 2, n - 1} & set(range(n))):
            row = slice(int(ptr[b]) + i, int(ptr[b]) + i + 1)
            want, tol = ref.attend(q[row], K[:a + i + 1], V[:a + i + 1], a + i, stored, None, bias, 100)
            ref.assert_near(out[row], want, tol, (b, a, i))
    return q, out


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("buckets", [0, 16])
def test_prompts_that_fill_the_card(dev, dtype, stored, d, buckets):
    q, _ = _prompt(dev, dtype, stored, [(1100, 900), (0, 1300), (333, 1)], 32, 4, d, buckets, 1)
    assert q.shape[0] * q.shape[1] / 128 > 512


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("d,spare", [(32, 1), (64, 500), (128, 1)])
@pytest.mark.parametrize("buckets", [0, 16])
def test_short_and_long_sequences_together(dev, dtype, stored, d, spare, buckets):
    """Sequences whose middle query sees at most 65,536 keys over the number of tiles, some 200 here, have weights in two parts."""
    q, _ = _prompt(dev, dtype, stored, [(0, 90), (2000, 400), (100, 5), (0, 600), (5, 70)], 32, 4, d, buckets, spare)
    assert 256 < q.shape[0] * q.shape[1] / 128 < 512


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("H,Hk,d,buckets", [(8, 4, 64, 0), (8, 4, 64, 16), (40, 2, 32, 0), (4, 4, 128, 16)])
def test_steps_with_more_rows_than_workgroups(dev, dtype, stored, H, Hk, d, buckets):
    """300 streams over a table of 100 pages: shares of several rows, rows of several shares.  Some streams are left
    alone, some lack a page, some have no place in the table for the new token."""
    from gdl_amd.functional import paged_attention_step
    gen = torch.Generator().manual_seed(H + d)
    B, columns = 300, 100
    lengths = [1 + (i * 37) % 150 for i in range(B)]  # the new token among them
    for i, n in ((3, 6400), (100, 2000), (101, 1999), (290, 4097), (299, 700)):
        lengths[i] = n
    pages = sum(-(-n // 64) for n in lengths) + 2
    table = torch.full((B, columns), -1, dtype=torch.int32)
    short = ref.random_table(lengths, 64, pages, gen)
    table[:, :short.shape[1]] = short[:, :columns]
    cache = _poisoned(dev, pages, Hk, d, 64, stored)
    k, v = ([torch.randn(n, Hk, d, generator=gen).to(dtype) for n in lengths] for _ in range(2))
    before = [n - 1 for n in lengths]
    cache.write(*(torch.cat([x[:-1] for x in y]).to(dev) for y in (k, v)), table.to(dev), torch.tensor([0] + before).cumsum(0).to(dev))
    at = torch.tensor(before)
    at[7::40], alone = -1 - torch.arange(len(at[7::40])), set(range(7, B, 40))
    gone = {11, 100}  # a page of the past, and of the new token
    table[11, 0], table[100, 1999 // 64] = pages + 5, -7
    at[50] = 6400  # beyond the table
    want_pool = ref.copy(cache)
    for b in range(B):
        if b not in alone and b != 50 and b != 100 and not (b == 11 and lengths[b] <= 64):
            page, slot = int(table[b, before[b] // 64]), before[b] % 64
            ref.put(want_pool, "k", page, slot, k[b][-1]), ref.put(want_pool, "v", page, slot, v[b][-1])
    if stored is E4:  # small negative values are kept as the code of 0, whose sign the rounding in the reference keeps
        for name in ("k", "v"):
            codes = want_pool[name].view(torch.uint8)
            codes[codes == 0x80] = 0
    q = torch.randn(B, H, d, generator=gen).to(dtype)
    bias = torch.randn(buckets, H, generator=gen).to(dtype) if buckets else None
    args = [x.to(dev) for x in (q, torch.stack([x[-1] for x in k]), torch.stack([x[-1] for x in v]))]
    out = paged_attention_step(*args, cache, table.to(dev), at.to(dev), bias=None if bias is None else bias.to(dev), max_distance=100)
    ref.same(cache, want_pool)
    for b in range(B):
        if b in alone:
            assert (out[b] == 0).all(), b
        elif b in gone or b == 50:
            assert out[b].isnan().all(), b
        else:
            assert out[b].isfinite().all(), b
    for b in [0, 1, 2, 3, 4, 63, 64, 99, 101, 102, 150, 200, 250, 289, 290, 291, 298, 299]:
        if b not in alone:
            want, tol = ref.attend(q[b:b + 1], ref.stored(k[b], stored), ref.stored(v[b], stored), before[b], stored, None, bias, 100)
            ref.assert_near(out[b:b + 1], want, tol, (b, lengths[b]))
    assert B * Hk * -(-(H // Hk) // 16) > 1024
