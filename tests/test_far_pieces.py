"""Leading tokens' gradients are sums over pieces of their sequences: how much scratch the pieces take (on the
CPU), and that longer pieces and wide heads give the definition's gradients (on the GPU)."""

import pytest
import torch

from attention_ref import assert_within, reference, visible
from gdl_amd import _native

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _scratch(tokens, heads, kv_heads, head_dim, left, sinks, dtype=1):
    args = _native.pack_window_attention(4096, 4096, 4096, heads * head_dim, head_dim, kv_heads * head_dim, head_dim, kv_heads * head_dim,
                                         head_dim, 0, 0, 0, 0, tokens, 1, left, 0, sinks, dtype, 0, heads, kv_heads, head_dim, 0, 0, 0.1)
    return _native.lib().geo_window_attention_bwd_workspace_bytes(args)


@pytest.mark.parametrize("tokens", [1000, 131_072, 1 << 22, (1 << 30) - 1])
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (16, 4), (64, 64)])
@pytest.mark.parametrize("sinks", [1, 16, 256])
def test_scratch_is_bounded(tokens, heads, kv_heads, sinks):
    delta = 4 * heads * tokens
    need = _scratch(tokens, heads, kv_heads, 128, 300, sinks)
    assert delta <= need <= delta + (64 << 20) + 4096
    assert _scratch(tokens, heads, kv_heads, 128, tokens, sinks) <= delta + 4096  # nothing lies beyond the window


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [96, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_long_pieces_and_wide_heads(dev, dtype, D, bias):
    from gdl_amd.functional import window_attention
    T, H, sinks, left = 2000, 32, 200, 100
    print(dtype, D, bias, flush=True)
    gen = torch.Generator().manual_seed(D)
    q, k, v, g = (torch.randn(T, H, D, generator=gen).to(dev, dtype) for _ in range(4))
    table = torch.randn(8, H, generator=gen).to(dev, dtype) if bias else None
    ptr = [0, 1600, 2000]
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = window_attention(*leaves, (left, 0), sinks=sinks, ptr=torch.tensor(ptr, device=dev), bias=table, max_distance=30)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g)), out=out)
    seen = visible(T, left, 0, sinks, ptr)
    for h in (0, H - 1):
        one = slice(h, h + 1)
        want, tol = reference(q[:, one], k[:, one], v[:, one], g[:, one], seen, table=table[:, one] if bias else None, maxd=30,
                              two_sided=False)
        assert_within({n: x[:, one] for n, x in got.items()}, {n: want[n] for n in got}, tol, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [96, 128])
def test_pieces_of_one_wave_at_wide_heads(dev, dtype, D):
    """Few heads: every kernel by one wave, V of dk and dv in LDS, eight pieces of 256 tokens."""
    from gdl_amd.functional import window_attention
    T, H, sinks, left = 2000, 2, 40, 60
    gen = torch.Generator().manual_seed(D + 1)
    q, g = (torch.randn(T, H, D, generator=gen).to(dev, dtype) for _ in range(2))
    k, v = (torch.randn(T, 1, D, generator=gen).to(dev, dtype) for _ in range(2))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    ptr = [0, 30, 1700, 2000]
    out = window_attention(*leaves, (left, 0), sinks=sinks, ptr=torch.tensor(ptr, device=dev))
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g)), out=out)
    want, tol = reference(q, k, v, g, visible(T, left, 0, sinks, ptr))
    assert_within(got, want, tol, D)
