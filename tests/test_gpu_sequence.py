"""GPU tests of the sequence block (recurrence, window attention, relative bias together), of the order
that it takes clouds in, and of the operators at lengths beyond their chunks' rounds."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_serial_order_is_morton_order_of_each_cloud(dev):
    from gdl_amd.sequence import serial_order
    gen = torch.Generator().manual_seed(0)
    sizes = [50, 1, 0, 200]
    ptr = torch.tensor([0] + sizes).cumsum(0)
    pos = torch.randn(int(ptr[-1]), 3, generator=gen)
    order = serial_order(pos.to(dev), ptr.to(dev)).cpu()
    for a, b in zip(ptr[:-1].tolist(), ptr[1:].tolist()):
        p = pos[a:b]
        if not len(p):
            continue
        low, size = p.amin(0), (p.amax(0) - p.amin(0)).max().clamp(min=torch.finfo(torch.float32).tiny)
        cell = ((p - low) / size * 1024).long().clamp(0, 1023)

        def code(c):
            return sum((int(c[k]) >> n & 1) << (3 * n + k) for n in range(10) for k in range(3))

        want = sorted(range(len(p)), key=lambda i: (code(cell[i]), i))
        assert order[a:b].tolist() == [a + i for i in want]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_steps_are_the_forwards_rows(dev, dtype):
    from gdl_amd.sequence import PointSequenceBlock
    torch.manual_seed(1)
    block = PointSequenceBlock(64, 4, 9, kv_heads=2, sinks=2, buckets=16, max_distance=20).to(dev)
    with torch.no_grad():
        block.bias.normal_()
    block = block.to(dtype)
    block.decay.data = block.decay.data.float()
    B, T = 3, 40
    x = torch.randn(B, T, 64, device=dev).to(dtype)
    with torch.no_grad():
        rows = block(x.reshape(B * T, 64), torch.arange(0, B * T + 1, T, device=dev)).view(B, T, 64)
    cache = block.new_cache(B)
    # the two forms round the same values to the type once each; bfloat16 rows differ by its roundings
    tol = 2e-5 if dtype is torch.float32 else 6e-2
    for t in range(T):
        out = block.step(x[:, t], torch.full((B,), t, device=dev), cache)
        assert (out.float() - rows[:, t].float()).abs().max() <= tol * max(1.0, rows[:, t].float().abs().max().item())


def test_block_learns_both_ways(dev):
    """Every parameter gets a finite gradient, and a few steps lower the loss."""
    from gdl_amd.sequence import PointSequenceBlock
    torch.manual_seed(2)
    for causal in (True, False):
        block = PointSequenceBlock(32, 2, 8, causal=causal, buckets=8, max_distance=16).to(dev)
        x, y = torch.randn(300, 32, device=dev), torch.randn(300, 32, device=dev)
        ptr, mask = torch.tensor([0, 120, 300], device=dev), torch.rand(300, device=dev) < 0.9
        opt = torch.optim.Adam(block.parameters(), lr=3e-3)
        losses = []
        for _ in range(30):
            loss = (block(x, ptr, mask) - y).square().mean()
            opt.zero_grad(set_to_none=True)
            loss.backward()
            assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())
            opt.step()
            losses.append(loss.item())
        assert losses[-1] < 0.9 * losses[0]
    with pytest.raises(ValueError):
        block.new_cache(2)
    with pytest.raises(ValueError):
        PointSequenceBlock(30, 4, 8)


def test_recurrence_beyond_one_round_of_chunks(dev):
    """300,000 tokens in one scan are two scans, the second from the first's state: the same sums in
    another grouping, so equal to some units of float32 of the states' size."""
    from gdl_amd.functional import gated_recurrence
    gen = torch.Generator().manual_seed(3)
    T, C, cut = 300_000, 5, 150_016
    x, ga, gx = (torch.randn(T, C, generator=gen).to(dev) for _ in range(3))
    decay = torch.full((C,), -6.0, device=dev)
    for reverse in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, ga, gx)]
        h, last = gated_recurrence(*leaves, decay, reverse=reverse)
        dh = torch.randn(T, C, generator=gen).to(dev)
        grads = torch.autograd.grad(h, leaves, dh)
        parts = [t.clone().requires_grad_() for t in (x, ga, gx)]
        first, second = (slice(0, cut), slice(cut, T)) if not reverse else (slice(cut, T), slice(0, cut))
        h1, l1 = gated_recurrence(*(t[first] for t in parts), decay, reverse=reverse)
        h2, l2 = gated_recurrence(*(t[second] for t in parts), decay, state=l1, reverse=reverse)
        want = torch.autograd.grad([h1, h2], parts, [dh[first], dh[second]])
        size = h.abs().max().item()
        assert (h[first] - h1).abs().max() <= 1e-5 * size and (h[second] - h2).abs().max() <= 1e-5 * size
        assert (last - l2).abs().max() <= 1e-5 * size
        for g, w in zip(grads, want):
            assert (g - w).abs().max() <= 1e-5 * w.abs().max()


def test_leading_tokens_of_a_long_sequence(dev):
    """Gradients of leading tokens that 140,000 later ones see, against the definition over the window's
    and the leading keys in float64: a weight's relative error is some 30 units of float32 (8 products,
    34 keys), and the terms' errors have no common sign, so a sum is as exact as its terms."""
    from gdl_amd.functional import window_attention
    gen = torch.Generator().manual_seed(4)
    T, H, D, left, sinks = 140_000, 2, 8, 30, 3
    q = torch.randn(T, H, D, generator=gen).to(dev).requires_grad_()
    k, v = (torch.randn(T, 1, D, generator=gen).to(dev).requires_grad_() for _ in range(2))
    g = torch.randn(T, H, D, generator=gen).to(dev)
    out = window_attention(q, k, v, (left, 0), sinks=sinks)
    got = torch.autograd.grad(out, [q, k, v], g)
    i = torch.arange(T, device=dev).view(T, 1)
    j = torch.cat([torch.arange(sinks, device=dev).expand(T, sinks), i - left + torch.arange(left + 1, device=dev)], 1)
    seen = torch.cat([j[:, :sinks] < i - left, j[:, sinks:] >= 0], 1)
    qd, kd, vd = (t.detach().double().requires_grad_() for t in (q, k, v))
    jc = j.clamp(0)
    s = (qd.unsqueeze(2) * kd[jc].transpose(1, 2)).sum(-1) / D ** 0.5
    p = s.masked_fill(~seen.unsqueeze(1), -torch.inf).softmax(-1)
    o = (p.unsqueeze(-1) * vd[jc].transpose(1, 2)).sum(2)
    want = torch.autograd.grad(o, [qd, kd, vd], g.double())
    assert (out.double() - o).abs().max() <= 1e-5
    for a, b in zip(got, want):
        for rows in (slice(0, sinks), slice(sinks, T)):
            assert (a[rows].double() - b[rows]).abs().max() <= 2e-5 * b[rows].abs().max()


def test_many_short_sequences_with_leading_tokens(dev):
    """More sequences than pieces, some of which reach past theirs."""
    from attention_ref import assert_within, reference, visible
    from gdl_amd.functional import window_attention
    gen = torch.Generator().manual_seed(5)
    lengths = [1] * 40 + [700] + [3] * 30 + [600] + [2] * 20
    ptr = [0]
    for n in lengths:
        ptr.append(ptr[-1] + n)
    T, H, D = ptr[-1], 2, 16
    q, g = (torch.randn(T, H, D, generator=gen).to(dev) for _ in range(2))
    k, v = (torch.randn(T, 1, D, generator=gen).to(dev) for _ in range(2))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, (20, 0), sinks=5, ptr=torch.tensor(ptr, device=dev))
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g)), out=out)
    want, tol = reference(q, k, v, g, visible(T, 20, 0, 5, ptr))
    assert_within(got, want, tol)
