"""GPU tests of the attention's gradients where log-sums are too large for float32 to hold a sum of several
weights: biases of any size that all keys share, and large scores."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.mark.parametrize("heads", [2, 48], ids=["few", "many"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bias", [0.0, -1e4, 1e5, -1e6, -1e9, 1e20, torch.finfo(F32).min])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_the_weights_of_a_query_sum_to_one(dev, heads, dtype, bias, D):
    """Whatever a query's weights are, they sum to one, so the gradients of v sum to the output's over the
    queries.  Bound: each weight is rounded to the type, and so is the output's gradient times the row's
    factor, each result too, and the float32 sums, exponentials and reciprocals of at most 61 weights are
    off by less than 2^-16."""
    from gdl_amd.functional import window_attention
    T = 700 if heads > 2 else 150
    print(heads, dtype, bias, D, flush=True)
    gen = torch.Generator().manual_seed(D)
    q, k, v, g = (torch.randn(T, heads, D, generator=gen).to(dev, dtype) for _ in range(4))
    table = torch.full((8, heads), bias, device=dev)
    if bias == 0.0:  # scores of some 10^5
        q = (q.float() * 6e4 / D ** 0.5).to(dtype) if dtype is not F16 else q * 8192
    leaves = [x.requires_grad_() for x in (q, k, v, table)]
    out = window_attention(q, k, v, (40, 20), sinks=1, ptr=torch.tensor([0, 60, T], device=dev), bias=table, max_distance=9)
    grads = torch.autograd.grad(out, leaves, g)
    assert all(torch.isfinite(x).all() for x in grads)
    dv, gd, u = grads[2].double(), g.double(), UNIT[dtype]
    bound = (2 * u + 2.0 ** -16) * gd.abs().sum(0) + u * dv.abs().sum(0) + T * 2.0 ** -25
    off = (dv.sum(0) - gd.sum(0)).abs()
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_equal_weights(dev, dtype):
    """Biases of which a score is less than half a unit: equal weights, and gradients from them."""
    from gdl_amd.functional import window_attention
    T, H, D, left = 90, 3, 32, 25
    gen = torch.Generator().manual_seed(1)
    q, k, v, g = (torch.randn(T, H, D, generator=gen).to(dev, dtype).requires_grad_() for _ in range(4))
    table = torch.full((8, H), torch.finfo(F32).min, device=dev)
    out = window_attention(q, k, v, (left, 0), bias=table, max_distance=9)
    dq, dk, dv = torch.autograd.grad(out, [q, k, v], g)
    i, j = torch.arange(T).view(T, 1), torch.arange(T)
    p = ((j <= i) & (j >= i - left)).double()
    p = p / p.sum(1, keepdim=True)
    qd, kd, vd, gd = (x.detach().double().cpu().transpose(0, 1) for x in (q, k, v, g))
    o, u = p @ vd, UNIT[dtype]
    ds = p * (gd @ vd.transpose(1, 2) - (gd * o).sum(-1, keepdim=True))
    size = p * (gd.abs() @ vd.abs().transpose(1, 2) + (gd.abs() * o.abs()).sum(-1, keepdim=True))
    for got, want, term in ((out, o, p @ vd.abs()), (dv, p.t() @ gd, p.t() @ gd.abs()), (dq, ds @ kd / D ** 0.5, size @ kd.abs() / D ** 0.5),
                            (dk, ds.transpose(1, 2) @ qd / D ** 0.5, size.transpose(1, 2) @ qd.abs() / D ** 0.5)):
        bound = (3 * u + 2.0 ** -16) * term + u * want.abs() + 2.0 ** -20
        assert ((got.detach().double().cpu().transpose(0, 1) - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bias", [-2e7, 5e7, 1e8, -1.3e8])
def test_many_keys_and_large_gradients(dev, dtype, bias):
    """Log-sums whose units (4 to 16) are as large as log2 of the 4096 keys, output gradients of 4096: as above,
    with the spacing of float16 below its normal numbers, 2^-24, in the gradient times the factor, for every key."""
    from gdl_amd.functional import window_attention
    T, H, D = 4096, 2, 32
    gen = torch.Generator().manual_seed(2)
    q, k, v, g = (torch.randn(T, H, D, generator=gen).to(dev, dtype) for _ in range(4))
    g = (g.float() * 4096).to(dtype)
    table = torch.full((8, H), bias, device=dev)
    leaves = [x.requires_grad_() for x in (q, k, v, table)]
    out = window_attention(*leaves[:3], (None, 0), bias=table, max_distance=9)
    dv = torch.autograd.grad(out, leaves, g)[2]
    assert torch.isfinite(dv).all()
    dv, gd, u = dv.double(), g.double(), UNIT[dtype]
    bound = (2 * u + 2.0 ** -14) * gd.abs().sum(0) + u * dv.abs().sum(0) + T * T * 2.0 ** -25
    off = (dv.sum(0) - gd.sum(0)).abs()
    assert (off <= bound).all(), (off / bound).max()
