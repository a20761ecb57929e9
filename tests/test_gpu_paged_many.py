"""Thousands of short streams in one call, and streams that share the pages of a common past."""

import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _softmax_rows(q, K, V, seen):
    """float64 rows [B, H, D] of q [B, H, D] over K, V [B, n, 1, D], and the bounds of float32 sums over n keys."""
    s = torch.einsum("bhd,bnd->bhn", q.double(), K[:, :, 0].double()) / math.sqrt(q.shape[-1])
    p = s.masked_fill(~seen.unsqueeze(1), -math.inf).softmax(-1)
    size = torch.einsum("bhd,bnd->bhn", q.double().abs(), K[:, :, 0].double().abs()).amax(-1, keepdim=True) / math.sqrt(q.shape[-1])
    e, D, n = 2.0 ** -24, q.shape[-1], K.shape[1]
    w = 2 * e * ((D + 8) * size + 4) + e * n + 2 * e
    return torch.einsum("bhn,bnd->bhd", p, V[:, :, 0].double()), w * torch.einsum("bhn,bnd->bhd", p, V[:, :, 0].double().abs()) + 1e-30


@pytest.mark.parametrize("B", [65, 700, 5000])
@pytest.mark.parametrize("columns", [1, 40])
def test_many_streams(dev, B, columns):
    """Stream b holds b % 7 tokens, takes b % 4 as a packet and then one more; every eleventh is left alone by the step."""
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(B)
    H, D, most = 2, 16, 10
    cache = PagedCache.empty(B, 1, D, dtype=F32, device=dev)
    table = torch.full((B, columns), -1, dtype=torch.int32)
    table[:, 0] = torch.randperm(B, generator=gen).int()
    table = table.to(dev)
    K, V = (torch.randn(B, most, 1, D, generator=gen) for _ in range(2))
    q = torch.randn(B, most, H, D, generator=gen)
    i = torch.arange(B)
    held, new = i % 7, i % 4

    def packed(x, first, n):
        at = torch.arange(most).view(1, -1)
        return x[(at >= first.view(-1, 1)) & (at < (first + n).view(-1, 1))].to(dev)

    def ptr_of(n):
        return torch.cat([n.new_zeros(1), n.cumsum(0)]).to(dev)

    cache.write(packed(K, held * 0, held), packed(V, held * 0, held), table, ptr_of(held))
    cache.write(packed(K, held, new), packed(V, held, new), table, ptr_of(new), held.to(dev))
    out = paged_attention(packed(q, held, new), cache, table, ptr_of(new), held.to(dev)).cpu().double()
    owner = torch.repeat_interleave(i, new)
    place = torch.cat([torch.arange(n) for n in new.tolist()]) + held[owner]
    want, tol = _softmax_rows(q[owner, place], K[owner], V[owner], torch.arange(most) <= place.view(-1, 1))
    assert ((out - want).abs() <= tol).all()
    length = held + new
    for got, x in zip(cache.read(table, ptr_of(length), int(length.sum())), (K, V)):
        assert torch.equal(got.cpu(), packed(x, held * 0, length).cpu())
    p = torch.where(i % 11 == 3, -1, length)
    out = paged_attention_step(q[i, length].to(dev), K[i, length].to(dev), V[i, length].to(dev), cache, table, p.to(dev)).cpu().double()
    want, tol = _softmax_rows(q[i, length], K, V, torch.arange(most) <= length.view(-1, 1))
    assert (out[p < 0] == 0).all() and ((out - want).abs() <= tol)[p >= 0].all()


@pytest.mark.parametrize("stored", [BF16, torch.int8], ids=["bf16", "i8"])
def test_a_common_past(dev, stored):
    """Streams that share their first pages, by one table's rows and by a table without rows of its own."""
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    gen = torch.Generator().manual_seed(4)
    B, H, Hk, D, past = 3, 4, 2, 32, 128
    cache = PagedCache.empty(2 + B, Hk, D, dtype=stored, device=dev)
    k, v = (torch.randn(past + B, Hk, D, generator=gen).bfloat16().to(dev) for _ in range(2))
    table = torch.tensor([[1, 0, 2 + b] for b in range(B)], dtype=torch.int32, device=dev)
    cache.write(k[:past], v[:past], table[:1])
    q = torch.randn(past + B, H, D, generator=gen).bfloat16().to(dev)
    out = paged_attention_step(q[past:], k[past:], v[past:], cache, table, torch.full((B,), past, device=dev))
    for b in range(B):
        rows = torch.cat([torch.arange(past), torch.tensor([past + b])])
        want, tol = ref.attend(q[past + b:past + b + 1], ref.stored(k[rows], stored), ref.stored(v[rows], stored), past, stored)
        ref.assert_near(out[b:b + 1], want, tol, b)
    common = table[:1].expand(B, -1)  # no stream writes: each asks for the same past
    ptr, start = torch.tensor([0, 2, 2, 7], device=dev), torch.tensor([60, 0, 100], device=dev)
    out = paged_attention(q[:7], cache, common, ptr, start)
    for lo, hi, at in ((0, 2, 60), (2, 7, 100)):
        ref.assert_near(out[lo:hi], *ref.attend(q[lo:hi], ref.stored(k[:past], stored)[:at + hi - lo], ref.stored(v[:past], stored)[:at + hi - lo], at, stored))
