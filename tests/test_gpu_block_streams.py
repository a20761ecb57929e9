"""GPU tests of streams that the sequence block and the recurrence's step are to leave alone or to begin
anew."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,C", [(5, 7), (6, 64), (2100, 2048)])
def test_step_at_positions(dev, dtype, B, C):
    from gdl_amd.functional import gated_recurrence_step
    gen = torch.Generator().manual_seed(C)
    x, ga, gx = (torch.randn(B, C, generator=gen).to(dev, dtype) for _ in range(3))
    decay, state = torch.randn(C, generator=gen).to(dev), torch.randn(B, C, generator=gen).to(dev)
    pos = torch.arange(B, device=dev) % 3 - 1  # -1, 0, 1
    h, new = gated_recurrence_step(x, ga, gx, decay, state)
    h0, new0 = gated_recurrence_step(x, ga, gx, decay, torch.zeros_like(state))
    junk = state.clone()
    junk[pos == 0] = math.nan
    idle = x.clone()
    idle[pos < 0] = math.nan
    got, after = gated_recurrence_step(idle, ga, gx, decay, junk, positions=pos)
    for n, (want, w) in enumerate(((torch.zeros_like(h), state), (h0, new0), (h, new))):
        rows = pos == n - 1
        assert torch.equal(got[rows], want[rows]) and torch.equal(after[rows], w[rows]), n
    same = gated_recurrence_step(idle, ga, gx, decay, junk, positions=pos.int())
    assert torch.equal(same[0], got) and torch.equal(same[1], after)
    for bad in (pos[:-1], pos.float(), pos.view(1, -1)):
        with pytest.raises(ValueError):
            gated_recurrence_step(x, ga, gx, decay, state, positions=bad)


def test_streams_that_pause_and_begin_anew(dev):
    """Streams of the block that start at different times, pause (with NaN in their rows) and are taken
    over by others: every row is the forward's for its own stream."""
    from gdl_amd.sequence import PointSequenceBlock
    torch.manual_seed(3)
    block = PointSequenceBlock(32, 2, 6, sinks=1, buckets=8, max_distance=9).to(dev)
    with torch.no_grad():
        block.bias.normal_()
    B, T = 4, 30
    sequences = [torch.randn(T, 32, device=dev) for _ in range(2 * B)]
    with torch.no_grad():
        rows = [block(s) for s in sequences]
    cache = block.new_cache(B)
    cache.state.fill_(math.nan)  # what another stream left
    gen = torch.Generator().manual_seed(0)
    now, at = list(range(B)), [0] * B
    for _ in range(70):
        go = (torch.rand(B, generator=gen) < 0.7).tolist()
        x = torch.stack([sequences[now[b]][at[b]] if go[b] else torch.full((32,), math.nan, device=dev) for b in range(B)])
        out = block.step(x, torch.tensor([at[b] if go[b] else -1 for b in range(B)], device=dev), cache)
        for b in range(B):
            if not go[b]:
                continue
            want = rows[now[b]][at[b]]
            assert (out[b] - want).abs().max() <= 2e-5 * max(1.0, want.abs().max().item())
            at[b] += 1
            if at[b] == T:
                now[b], at[b] = (now[b] + B) % (2 * B), 0


def test_a_refused_step_leaves_the_cache(dev):
    from gdl_amd.sequence import PointSequenceBlock
    block = PointSequenceBlock(32, 2, 6, buckets=8, max_distance=9).to(dev)
    cache = block.new_cache(3, dtype=BF16)  # not the block's type
    state = cache.state.normal_().clone()
    with pytest.raises(TypeError):
        block.step(torch.randn(3, 32, device=dev), torch.tensor([4, 5, 6], device=dev), cache)
    assert torch.equal(cache.state, state)
