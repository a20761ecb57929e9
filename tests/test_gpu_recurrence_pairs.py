"""Large 16-bit recurrences put two channels on a lane where rows begin on multiples of 4 bytes.  A
channel's operations and their order are the same either way, so results equal those of the same
values in rows at odd places, bit by bit (these are checked against 64 bits elsewhere)."""

import pytest
import torch

from gdl_amd.functional import gated_recurrence, gated_recurrence_step

pytestmark = pytest.mark.gpu


def _twice(rows, channels, dtype, seed):
    """Three inputs in rows at even places, and the same in rows at odd places."""
    gen = torch.Generator("cuda").manual_seed(seed)
    even = [torch.randn(rows, channels, device="cuda", generator=gen).to(dtype) for _ in range(3)]
    odd = []
    for t in even:
        wide = torch.zeros(rows, channels + 1, device="cuda", dtype=dtype)
        wide[:, 1:] = t
        odd.append(wide[:, 1:])
    return even, odd


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("tokens, channels", [((1 << 17) + 77, 128), (43691, 384)])
def test_scan_of_pairs(dtype, reverse, tokens, channels):
    even, odd = _twice(tokens, channels, dtype, 1)
    decay = torch.linspace(-6.0, 2.0, channels, device="cuda")
    ptr = torch.tensor([3, 3, 4, 70, 5000, 5000, tokens // 2 + 1, tokens - 9], device="cuda")
    state = torch.randn(ptr.numel() - 1, channels, device="cuda")
    dh = torch.randn(tokens, channels, device="cuda").to(dtype)
    dlast = torch.randn_like(state)
    results = []
    for inputs in (even, odd):
        leaves = [t.detach().requires_grad_() for t in (*inputs, decay, state)]
        h, last = gated_recurrence(*leaves[:4], ptr=ptr, state=leaves[4], reverse=reverse)
        grads = torch.autograd.grad((h, last), leaves, (dh, dlast))
        results.append((h, last, *grads))
    for one, two in zip(*results):
        assert torch.equal(one, two)
        assert torch.isfinite(one).all()
    assert not results[0][0][:3].any() and not results[0][0][tokens - 9:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_step_of_pairs(dtype):
    even, odd = _twice(4099, 1026, dtype, 2)
    decay = torch.linspace(-6.0, 2.0, 1026, device="cuda")
    state = torch.randn(4099, 1026, device="cuda")
    for one, two in zip(gated_recurrence_step(*even, decay, state), gated_recurrence_step(*odd, decay, state)):
        assert torch.equal(one, two)
