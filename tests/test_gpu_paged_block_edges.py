"""GPU tests of the sequence block's packets at negative positions, where no stream has tokens."""

import pytest
import torch

from test_gpu_paged_block import _block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stored", [torch.float32, torch.int8], ids=["f32", "i8"])
def test_packets_before_and_across_position_0(dev, stored):
    """A packet ahead of position 0 leaves its stream as it was, whatever its rows hold; one that crosses it begins the stream
    anew at position 0; the streams beside them go on."""
    block = _block(dev)
    T, lost = 40, 5
    x = torch.randn(4, T, 64, device=dev)

    def extend(cache, parts, start):
        ptr = torch.tensor([0] + [len(p) for p in parts]).cumsum(0)
        y = block.extend(torch.cat(parts), ptr.to(dev), torch.tensor(start, device=dev), cache)
        return [y[int(a):int(b)] for a, b in zip(ptr, ptr[1:])]

    cache, alone = (block.new_cache(4, stored, tokens=2 * T) for _ in range(2))
    for c in (cache, alone):
        extend(c, [x[0], x[1, :0], x[2], x[3]], [0, 0, 0, 0])
    def pages(c):
        """The bits of the second and the last stream's pages, two each."""
        return [t.view(4, 2, -1)[1::2].contiguous().view(torch.uint8) for t in (c.window.k, c.window.v)]

    before, held = cache.state.clone(), pages(cache)
    wild = torch.full((lost, 64), torch.nan, device=dev)
    news = torch.randn(4, T, 64, device=dev)
    far = [T, -3 - lost, -lost, -(1 << 63)]
    got = extend(cache, [news[0], wild, torch.cat([wild, news[2]]), news[3]], far)
    want = extend(alone, [news[0], news[1, :0], news[2], news[3, :0]], [T, 0, 0, 0])
    # rows and states of the same tokens in other places of the packet: sums in another order
    tol = 1e-5
    for b in (0, 2):
        assert (got[b][-T:] - want[b]).abs().max() <= tol * max(1.0, want[b].abs().max().item()), b
    assert torch.equal(cache.state[1::2], before[1::2])
    assert (cache.state - alone.state).abs().max() <= tol * max(1.0, alone.state.abs().max().item())
    for a, b in zip(held, pages(cache)):  # what packets at negative positions hold is nowhere in the pool
        assert torch.equal(a, b)
    y = torch.randn(4, 64, device=dev)
    at = torch.tensor([2 * T, -1, T, T], device=dev)
    rows = [block.step(y, at, c) for c in (cache, alone)]
    for b in (0, 2, 3):
        assert (rows[0][b] - rows[1][b]).abs().max() <= tol * max(1.0, rows[1][b].abs().max().item()), b


def test_packets_and_steps_agree_at_negative_positions(dev):
    """The same tokens in packets and one by one, from position -4 on: the same rows from 0 on, the same states."""
    block = _block(dev)
    x = torch.randn(2, 12, 64, device=dev)
    a, b = (block.new_cache(2, tokens=64) for _ in range(2))
    for c in (a, b):
        c.state.normal_(generator=torch.Generator(device=dev).manual_seed(5))
    start, sizes = -4, (3, 3, 2, 4)
    at, rows = start, []
    for n in sizes:
        part = x[:, at - start:at - start + n].reshape(2 * n, 64)
        rows.append(block.extend(part, torch.tensor([0, n, 2 * n], device=dev), torch.full((2,), at, device=dev), a).view(2, n, 64))
        at += n
    rows = torch.cat(rows, 1)
    for t in range(12):
        y = block.step(x[:, t], torch.full((2,), start + t, device=dev), b)
        if start + t >= 0:
            assert (y - rows[:, t]).abs().max() <= 2e-5 * max(1.0, y.abs().max().item()), t
    assert (a.state - b.state).abs().max() <= 2e-5
    assert a.state.is_contiguous() and b.state.is_contiguous()


@pytest.mark.parametrize("B,C", [(1, 1), (1, 64), (3, 5), (70, 33)])
@pytest.mark.parametrize("dtype,step", [(torch.float32, 1), (torch.float32, 2), (torch.bfloat16, 1)], ids=["f32", "rows-apart", "bf16"])
def test_packets_as_sequences(dev, B, C, dtype, step):
    """Offsets and states of streams whose packets lie before, across and behind position 0, some without tokens."""
    from gdl_amd.functional.recurrence import packets_as_sequences
    gen = torch.Generator().manual_seed(B + C)
    n = torch.randint(0, 4, (B,), generator=gen)
    ptr = 2 + torch.cat([n.new_zeros(1), n.cumsum(0)])
    start = torch.randint(-4, 3, (B,), generator=gen)
    ends = torch.tensor([-(1 << 63), (1 << 63) - 1, 1 - (1 << 63)])
    start[::5] = ends[torch.arange(len(start[::5])) % 3]
    state = torch.randn(step * B, C, generator=gen).to(dtype).to(dev)[::step]
    parts, before = packets_as_sequences(ptr.to(dev), start.to(dev), state)
    assert before.dtype is torch.float32 and before.shape == (2 * B - 1, C) and parts.shape == (2 * B,)
    for b in range(B):
        lo, hi, at = int(ptr[b]), int(ptr[b + 1]), int(start[b])
        assert parts.tolist()[2 * b:2 * b + 2] == [min(max(lo, lo - at), hi), hi], (b, lo, hi, at)
        anew = at <= 0 < at + hi - lo
        assert torch.equal(before[2 * b], torch.zeros_like(before[0]) if anew else state[b].float()), b
        assert b == B - 1 or (before[2 * b + 1] == 0).all()
