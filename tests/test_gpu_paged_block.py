"""GPU tests of the sequence block over whole histories: forward, packets and single tokens of one stream are the
same rows; streams that pause and begin anew; histories in 8 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _block(dev, dtype=torch.float32, heads=4, kv_heads=2, channels=64, **kw):
    from gdl_amd.sequence import PointSequenceBlock
    torch.manual_seed(1)
    block = PointSequenceBlock(channels, heads, None, kv_heads=kv_heads, buckets=16, max_distance=20, **kw).to(dev)
    with torch.no_grad():
        block.bias.normal_()
    block = block.to(dtype)
    block.decay.data = block.decay.data.float()
    return block


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_packets_and_steps_are_the_forward_s_rows(dev, dtype):
    block = _block(dev, dtype)
    B, T = 3, 150
    x = torch.randn(B, T, 64, device=dev).to(dtype)
    with torch.no_grad():
        rows = block(x.reshape(B * T, 64), torch.arange(0, B * T + 1, T, device=dev)).view(B, T, 64)
    cache = block.new_cache(B, tokens=T)
    cache.state.fill_(math.nan)  # what other streams left
    # the three forms round the same values to the type once each; bfloat16 rows differ by its roundings
    tol = 2e-5 if dtype is torch.float32 else 6e-2

    def check(got, want):
        assert (got.float() - want.float()).abs().max() <= tol * max(1.0, want.float().abs().max().item())

    at = [0] * B
    for sizes in ((70, 1, 5), (0, 40, 64), (3, 0, 20), (40, 60, 1)):
        ptr = torch.tensor([0, *sizes]).cumsum(0)
        part = torch.cat([x[b, at[b]:at[b] + n] for b, n in enumerate(sizes)])
        kept = cache.state.clone()
        got = block.extend(part, ptr.to(dev), torch.tensor(at, device=dev), cache)
        for b, n in enumerate(sizes):
            if n:
                check(got[int(ptr[b]):int(ptr[b + 1])], rows[b, at[b]:at[b] + n])
            else:
                assert torch.equal(cache.state[b].nan_to_num(7), kept[b].nan_to_num(7))
            at[b] += n
    for _ in range(20):
        got = block.step(torch.stack([x[b, at[b]] for b in range(B)]), torch.tensor(at, device=dev), cache)
        for b in range(B):
            check(got[b], rows[b, at[b]])
            at[b] += 1


def test_a_block_without_a_window_learns(dev):
    """Every parameter's gradient is that of finite differences along a random direction."""
    from gdl_amd.sequence import PointSequenceBlock
    torch.manual_seed(2)
    for causal in (True, False):
        block = PointSequenceBlock(32, 2, None, causal=causal, buckets=8, max_distance=16).to(dev)
        x, g = torch.randn(90, 32, device=dev), torch.randn(90, 32, device=dev)
        ptr = torch.tensor([0, 30, 90], device=dev)
        block(x, ptr).backward(g)
        for name, p in block.named_parameters():
            way = torch.randn_like(p)
            way /= way.norm()
            want = (p.grad * way).sum().item()
            with torch.no_grad():
                ends = []
                for h in (1e-2, -1e-2):
                    p.add_(way, alpha=h)
                    ends.append((block(x, ptr).double() * g).sum().item())
                    p.sub_(way, alpha=h)
            got = (ends[0] - ends[1]) / 2e-2
            # h^2 / 6 third derivatives of a sum of 2880 terms of size 1, and float32's rounding of it over 2 h
            assert abs(got - want) <= 2e-2 * max(1.0, p.grad.norm().item()), (name, got, want)


@pytest.mark.parametrize("stored", [torch.int8, torch.float8_e4m3fn], ids=["i8", "e4m3"])
def test_histories_in_8_bits(dev, stored):
    """Packets and steps over 8 bits are one another's rows, and the forward's as far as 8 bits allow."""
    block = _block(dev)
    B, T = 2, 100
    x = torch.randn(B, T, 64, device=dev)
    with torch.no_grad():
        rows = block(x.reshape(B * T, 64), torch.arange(0, B * T + 1, T, device=dev))
    a, b = (block.new_cache(B, stored, tokens=T) for _ in range(2))
    whole = block.extend(x.reshape(B * T, 64), torch.arange(0, B * T + 1, T, device=dev), torch.zeros(B, dtype=torch.int64, device=dev), a)
    for t in range(T):
        got = block.step(x[:, t], torch.full((B,), t, device=dev), b)
        want = whole.view(B, T, 64)[:, t]
        # float32 throughout; a row's code may fall to the other side of a border where its inputs differ in the last bits
        assert (got - want).abs().max() <= 1e-2 * max(1.0, want.abs().max().item())
    # a value is off by 1 / 254 of its row's largest (int8) or 1 / 16 of itself (e4m3); scores of size 1 and weights follow
    assert (whole - rows).abs().max() <= (0.05 if stored is torch.int8 else 0.3) * max(1.0, rows.abs().max().item())


def test_a_shared_pool(dev):
    """Streams of unequal lengths in one pool, two of which share the pages of a common past."""
    from gdl_amd.functional import PagedCache
    from gdl_amd.sequence import BlockCache
    block = _block(dev)
    past, tails = torch.randn(128, 64, device=dev), torch.randn(2, 50, 64, device=dev)
    pool = PagedCache.empty(6, 2, 16, device=dev)
    first = BlockCache(torch.zeros(1, 64, device=dev), pool, torch.tensor([[4, 1]], dtype=torch.int32, device=dev))
    block.extend(past, torch.tensor([0, 128], device=dev), torch.zeros(1, dtype=torch.int64, device=dev), first)
    both = BlockCache(first.state.repeat(2, 1), pool, torch.tensor([[4, 1, 0], [4, 1, 5]], dtype=torch.int32, device=dev))
    got = block.extend(tails.reshape(100, 64), torch.tensor([0, 50, 100], device=dev), torch.tensor([128, 128], device=dev), both)
    with torch.no_grad():
        for b in range(2):
            want = block(torch.cat([past, tails[b]]))[128:]
            assert (got[50 * b:50 * b + 50] - want).abs().max() <= 2e-5 * max(1.0, want.abs().max().item())


def test_refusals(dev):
    from gdl_amd.sequence import PointSequenceBlock
    block = _block(dev)
    with pytest.raises(ValueError):
        block.new_cache(2)  # no number of tokens
    with pytest.raises(ValueError):
        PointSequenceBlock(32, 2, None, sinks=1)
    windowed = PointSequenceBlock(32, 2, 8).to(dev)
    with pytest.raises(ValueError):
        windowed.new_cache(2, tokens=10)
    x = torch.randn(4, 32, device=dev)
    ptr, start = torch.tensor([0, 2, 4], device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError):
        windowed.extend(x, ptr, start, windowed.new_cache(2))
    cache = block.new_cache(3, tokens=10)
    with pytest.raises(ValueError):
        block.extend(torch.randn(4, 64, device=dev), ptr, start, cache)
    state = cache.state.normal_().clone()
    cache = block.new_cache(2, torch.bfloat16, tokens=10)  # not the block's type
    cache.state.copy_(state[:2])
    with pytest.raises(TypeError):
        block.extend(torch.randn(4, 64, device=dev), ptr, start, cache)
    assert torch.equal(cache.state, state[:2])
