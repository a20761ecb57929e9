"""GPU tests of the sequence block's mask: points that it hides count for nothing."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("junk", [5.0, math.nan, math.inf])
def test_hidden_points_reach_no_row_and_no_gradient(dev, causal, junk):
    from gdl_amd.sequence import PointSequenceBlock
    torch.manual_seed(4)
    block = PointSequenceBlock(32, 2, 8, sinks=1 if causal else 0, causal=causal, buckets=8, max_distance=16).to(dev)
    ptr = torch.tensor([0, 70, 71, 200], device=dev)
    mask = torch.rand(200, device=dev) < 0.7
    mask[:3], mask[70] = False, False
    x, y = torch.randn(200, 32, device=dev), torch.randn(200, 32, device=dev)
    results = []
    for value in (None, junk):
        z = x.clone()
        if value is not None:
            z[~mask] = value
        z.requires_grad_()
        out = block(z, ptr, mask)
        loss = (out[mask] * y[mask]).sum()
        results.append([out[mask]] + list(torch.autograd.grad(loss, [z] + list(block.parameters()))))
    for a, b in zip(*results):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert (results[0][1][~mask] == 0).all()


@pytest.mark.parametrize("causal", [True, False])
def test_the_recurrence_passes_hidden_points_by(dev, causal):
    """Without its attention the block gives the rows of the sequences of the other points alone, to
    the rounding of another order of the sums (64 channels, states of unit size)."""
    from gdl_amd.sequence import PointSequenceBlock
    torch.manual_seed(5)
    block = PointSequenceBlock(64, 2, 8, causal=causal, buckets=8, max_distance=16).to(dev)
    with torch.no_grad():
        block.attend_out.weight.zero_(), block.attend_out.bias.zero_()
    sizes = [150, 1, 90]
    ptr = torch.tensor([0] + sizes).cumsum(0)
    mask = torch.rand(241) < 0.5
    kept = torch.tensor([0] + [int(mask[a:b].sum()) for a, b in zip(ptr[:-1], ptr[1:])]).cumsum(0)
    x, mask = torch.randn(241, 64, device=dev), mask.to(dev)
    with torch.no_grad():
        rows = block(x, ptr.to(dev), mask)[mask]
        want = block(x[mask], kept.to(dev))
    assert (rows - want).abs().max() <= 1e-5 * want.abs().max()
