"""GPU tests of a relative bias that holds its type's lowest and highest finite values, forward and step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def uniform(v, first, last):
    """The mean of v's rows first[i] .. last[i]: adding the lowest value leaves nothing of a score in
    32 or 64 bits, so keys that all have it weigh the same."""
    return torch.stack([v[a:b + 1].mean(0) for a, b in zip(first, last)])


@pytest.mark.parametrize("heads", [1, 48], ids=["few", "many"])
@pytest.mark.parametrize("table", [F32, BF16], ids=["t32", "t16"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_lowest_values_alone_and_beside_others(dev, dtype, table, heads):
    """Causal, buckets 0 .. 3 for the distances 0 .. 3 and more beyond.  With the lowest value in the
    first three, tokens 0 .. 2 see nothing else; later ones see such keys at the weight 0."""
    from gdl_amd.functional import WindowCache, window_attention, window_attention_step
    T, D, left = 800 if heads > 1 else 60, 32, 20
    gen = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(T, heads, D, generator=gen).to(dev, dtype) for _ in range(3))
    bias = torch.zeros(8, heads, dtype=table, device=dev)
    bias[:3] = torch.finfo(table).min
    out = window_attention(q, k, v, (left, 0), bias=bias, max_distance=16).double().cpu()
    vd = v.double().cpu()
    want = uniform(vd, [0, 0, 0], [0, 1, 2])
    u = UNIT[dtype]
    assert ((out[:3] - want).abs() <= (2 * u + 2.0 ** -20) * vd[:3].abs().amax(0)).all()
    # the others: the definition without the three nearest keys
    s = torch.einsum("ihd,jhd->hij", q.double().cpu(), k.double().cpu()) / D ** 0.5
    i, j = torch.arange(T).view(T, 1), torch.arange(T)
    seen = (j <= i - 3) & (j >= i - left)
    p = s.masked_fill(~seen, -torch.inf)[:, 3:].softmax(-1)
    rest = torch.einsum("hij,jhd->ihd", p, vd)
    size = torch.einsum("hij,jhd->ihd", p, vd.abs())
    assert ((out[3:] - rest).abs() <= (2 * u + 2.0 ** -17) * size + 2.0 ** -24).all()
    # a step over three tokens, and over more
    cache = WindowCache.empty(1, heads, D, left, dtype=dtype, device=dev)
    for t in (0, 1, 2, 3, 4, 5):
        row = window_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], cache, torch.tensor([t], device=dev), bias=bias,
                                    max_distance=16)
        assert ((row[0].double().cpu() - out[t]).abs() <= (2 * u + 2.0 ** -17) * vd[:6].abs().amax(0)).all(), t
    # the highest value takes all the weight
    bias[:3], bias[1] = 0, torch.finfo(table).max
    out = window_attention(q, k, v, (left, 0), bias=bias, max_distance=16)
    assert torch.equal(out[1:], v[:-1])
