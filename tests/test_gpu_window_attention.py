"""GPU tests of window attention: output and gradients against the dense definition in float64 with
derived bounds, the gradient against differences, masks that leave rows empty, infinities and NaN in
places that are not seen, strides, streams, graph replays, refusals."""

import math

import pytest
import torch

from attention_ref import assert_within, bucket, reference, visible

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(dev, T, H, Hk, D, dtype, seed=0, fused=False):
    gen = torch.Generator().manual_seed(seed)
    if fused:
        x = torch.randn(T, H + 2 * Hk, D, generator=gen).to(dev, dtype)
        q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    else:
        q, k, v = (torch.randn(T, h, D, generator=gen).to(dev, dtype) for h in (H, Hk, Hk))
    return q, k, v, torch.randn(T, H, D, generator=gen).to(dev, dtype)


def attend(q, k, v, g, window, table=None, **kw):
    from gdl_amd.functional import window_attention
    leaves = [x.detach().requires_grad_() for x in (q, k, v) + ((table,) if table is not None else ())]
    out = window_attention(*leaves[:3], window, bias=leaves[3] if table is not None else None, **kw)
    got = dict(zip(("dq", "dk", "dv", "dbias"), torch.autograd.grad(out, leaves, g)))
    got["out"] = out
    return got


# (T, H, Hk, D, (left, right), sinks, sequences' lengths or None, share of masked keys, buckets, maxd)
CASES = [
    (1, 1, 1, 8, (0, 0), 0, None, 0, 0, 0),
    (1, 2, 1, 32, (5, 0), 3, None, 0, 16, 20),
    (2, 1, 1, 16, (1, 1), 0, None, 0, 0, 0),
    (31, 2, 2, 32, (3, 0), 0, None, 0, 0, 0),
    (33, 3, 1, 24, (40, 40), 0, None, 0.3, 8, 9),
    (64, 4, 4, 64, (0, 0), 0, None, 0, 0, 0),
    (65, 2, 2, 128, (64, 0), 1, None, 0, 32, 64),
    (127, 1, 1, 80, (31, 33), 0, [127], 0, 0, 0),
    (130, 2, 1, 5, (17, 4), 0, None, 0.2, 0, 0),
    (257, 4, 2, 32, (16, 16), 0, [1, 0, 100, 156], 0.1, 16, 30),
    (300, 2, 2, 48, (20, 0), 7, [3, 290, 0, 7], 0, 0, 0),
    (320, 6, 2, 64, (10, 2), 64, [200, 120], 0.5, 16, 12),
    (500, 2, 1, 96, (-1, 0), 0, [250, 250], 0, 32, 128),
    (700, 1, 1, 128, (-1, -1), 0, None, 0.95, 0, 0),
    (1100, 2, 1, 32, (30, 0), 40, [1090, 10], 0.1, 16, 100),
    (1500, 3, 1, 64, (100, 5), 9, [20, 1400, 80], 0, 32, 1024),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=[str(c[0]) + "x" + str(c[3]) for c in CASES])
def test_against_definition(dev, case, dtype):
    T, H, Hk, D, (left, right), sinks, lengths, masked, buckets, maxd = case
    print(case, dtype, flush=True)
    q, k, v, g = make(dev, T, H, Hk, D, dtype, seed=T, fused=T % 2 == 1 and D % 8 == 0)
    gen = torch.Generator().manual_seed(7)
    mask = (torch.rand(T, generator=gen) >= masked).to(dev) if masked else None
    table = torch.randn(buckets, H, generator=gen).to(dev, dtype) if buckets else None
    ptr = [0] if lengths else None
    for n in lengths or []:
        ptr.append(ptr[-1] + n)
    l, r = (x if x >= 0 else T for x in (left, right))
    want, tol = reference(q, k, v, g, visible(T, l, r, sinks, ptr, mask), table=table, maxd=maxd, two_sided=right != 0)
    got = attend(q, k, v, g, (left, right), table, sinks=sinks, mask=mask, max_distance=maxd or 128,
                 ptr=None if ptr is None else torch.tensor(ptr, device=dev))
    assert_within(got, want, tol, case)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D,H,Hk", [(64, 32, 8), (32, 40, 40), (128, 24, 12), (96, 16, 16)])
def test_shared_tiles(dev, dtype, D, H, Hk):
    """Enough heads and tokens for the four-wave workgroups of every kernel."""
    T = 2100
    print(D, H, Hk, dtype, flush=True)
    q, k, v, g = make(dev, T, H, Hk, D, dtype, seed=D)
    table = torch.randn(16, H, generator=torch.Generator().manual_seed(1)).to(dev, dtype)
    ptr = [0, 700, 701, 2100]
    mask = (torch.rand(T, generator=torch.Generator().manual_seed(2)) < 0.8).to(dev)
    # the definition on one group of heads at a time
    got = attend(q, k, v, g, (90, 33), table, sinks=5, mask=mask, max_distance=50, ptr=torch.tensor(ptr, device=dev))
    seen = visible(T, 90, 33, 5, ptr, mask)
    n = H // Hk
    for hk in (0, Hk - 1):
        a, b = hk * n, hk * n + n
        want, tol = reference(q[:, a:b], k[:, hk:hk + 1], v[:, hk:hk + 1], g[:, a:b], seen, table=table[:, a:b], maxd=50)
        part = {x: got[x][:, a:b] for x in ("out", "dq", "dbias")} | {x: got[x][:, hk:hk + 1] for x in ("dk", "dv")}
        assert_within(part, want, tol, (D, hk))


@pytest.mark.parametrize("bias", [False, True])
def test_gradient_against_differences(dev, bias):
    """Central differences of sum(out * g) in float32 along random directions, float64 sums.  A step
    h = 1/64 has a truncation error of h^2 / 6 times the third derivative (below 1e-3 of the sum's
    scale for scores of unit size) and a rounding error of 2e-7 |g| |out| sqrt(n) / h."""
    T, H, Hk, D = 90, 2, 1, 16
    q, k, v, g = make(dev, T, H, Hk, D, F32, seed=3)
    q, k = 0.5 * q, 0.5 * k
    table = 0.5 * torch.randn(16, H, device=dev) if bias else None
    kw = dict(sinks=2, ptr=torch.tensor([0, 60, 90], device=dev), max_distance=20)
    from gdl_amd.functional import window_attention
    grads = attend(q, k, v, g, (12, 3), table, **kw)
    gen = torch.Generator().manual_seed(5)
    inputs = {"dq": q, "dk": k, "dv": v} | ({"dbias": table} if bias else {})
    for name, x in inputs.items():
        step = torch.randn(x.shape, generator=gen).to(dev)
        h = 1 / 64

        def loss(sign):
            y = {n: t + sign * h * step if n == name else t for n, t in inputs.items()}
            o = window_attention(y["dq"], y["dk"], y["dv"], (12, 3), bias=y.get("dbias"), **kw)
            return (o.double() * g.double()).sum().item()

        slope = (loss(1) - loss(-1)) / (2 * h)
        want = (grads[name].double() * step.double()).sum().item()
        scale = (grads[name].double().abs() * step.double().abs()).sum().item()
        assert abs(slope - want) <= 1e-3 * scale + 2e-7 / h * math.sqrt(T * H * D) * 3, (name, slope, want, scale)


def test_rows_that_see_nothing(dev):
    """All keys masked, or none in the window: 0, and no gradient anywhere."""
    for dtype in (F32, BF16):
        q, k, v, g = make(dev, 70, 2, 2, 32, dtype)
        got = attend(q, k, v, g, (4, 0), torch.randn(8, 2, device=dev, dtype=dtype), max_distance=9, sinks=2,
                     mask=torch.zeros(70, dtype=torch.bool, device=dev))
        assert all((x == 0).all() for x in got.values())
        # tokens outside ptr's range see nothing and are seen by no one
        got = attend(q, k, v, g, (4, 0), ptr=torch.tensor([10, 30, 50], device=dev))
        for x in got.values():
            assert (x[:10] == 0).all() and (x[50:] == 0).all() and torch.isfinite(x).all()
            assert x[10:50].abs().sum() > 0
        # only the first 20 keys: queries 25 and on have none in reach
        mask = (torch.arange(70) < 20).to(dev)
        got = attend(q, k, v, g, (4, 0), mask=mask)
        assert (got["out"][24:] == 0).all() and (got["dq"][24:] == 0).all() and (got["dk"][20:] == 0).all()
        assert (got["out"][:24].abs().sum(-1) > 0).all()


@pytest.mark.parametrize("heads", [2, 40], ids=["few", "many"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "-inf"])
def test_places_that_are_not_seen_have_no_effect(dev, dtype, junk, heads):
    """NaN and infinities in masked keys, in another sequence and outside the window leave every
    other result as it is, bit by bit."""
    T, D = 1000 if heads > 2 else 300, 32
    q, k, v, g = make(dev, T, heads, heads, D, dtype, seed=9)
    ptr = torch.tensor([0, 100, 130, T], device=dev)
    table = torch.randn(8, heads, device=dev, dtype=dtype)
    mask = (torch.arange(T) % 7 != 3).to(dev)
    kw = dict(ptr=ptr, sinks=2, mask=mask, max_distance=9)
    clean = attend(q, k, v, g, (20, 4), table, **kw)

    def spoilt(rows, *which):
        x = [t.clone() for t in (q, k, v, g)]
        for n in which:
            x["qkvg".index(n)][rows] = junk
        got = attend(*x, (20, 4), table, **kw)
        return got

    masked = torch.nonzero(~mask).flatten()
    got = spoilt(masked, "k", "v")
    assert all(torch.equal(got[x], clean[x]) for x in clean)
    # the whole second sequence: the others' rows stay, in every output
    rest = torch.cat([torch.arange(100), torch.arange(130, T)]).to(dev)
    got = spoilt(torch.arange(100, 130, device=dev), "q", "k", "v", "g")
    for x in ("out", "dq", "dk", "dv"):
        assert torch.equal(got[x][rest], clean[x][rest]), x
    # one token of the third: queries that do not see it, keys that it does not see
    at = 200
    seen = visible(T, 20, 4, 2, ptr.tolist(), mask.cpu())
    assert seen[at].any() and mask[at]
    blind, unseen = ~seen[:, at].to(dev), ~seen[at].to(dev)
    got = spoilt(at, "k", "v")
    for x in ("out", "dq"):
        assert torch.equal(got[x][blind], clean[x][blind]), x
    assert not torch.isfinite(got["out"][~blind].float()).any()
    got = spoilt(at, "v")
    assert not torch.isfinite(got["out"][~blind].float()).any() and torch.equal(got["out"][blind], clean["out"][blind])
    got = spoilt(at, "g")
    for x in ("dk", "dv"):
        assert torch.equal(got[x][unseen], clean[x][unseen]), x
        assert not torch.isfinite(got[x][~unseen].float()).all(-1).any(), x
    got = spoilt(at, "q")
    for x in ("dk", "dv"):
        assert torch.equal(got[x][unseen], clean[x][unseen]), x


def test_large_scores(dev):
    """Scores of +-3000: the running maximum keeps every exponential at or below 1."""
    q, k, v, g = make(dev, 200, 2, 2, 32, F32, seed=4)
    q = q * 500
    got = attend(q, k, v, g, (60, 10))
    want, tol = reference(q, k, v, g, visible(200, 60, 10, 0))
    assert_within(got, want, tol)


def test_same_bits_every_time(dev):
    q, k, v, g = make(dev, 3000, 8, 2, 64, BF16, seed=11)
    table = torch.randn(32, 8, device=dev, dtype=BF16)
    kw = dict(ptr=torch.tensor([0, 1200, 3000], device=dev), sinks=16)
    one, two = (attend(q, k, v, g, (200, 0), table, **kw) for _ in range(2))
    assert all(torch.equal(one[x], two[x]) for x in one)


def test_strides_and_broadcast(dev):
    """Any strides give the contiguous result; a broadcast key head's gradient is the sum."""
    T, H, D = 150, 4, 32
    q, k, v, g = make(dev, T, H, H, D, F32, seed=12)
    base = attend(q, k, v, g, (30, 30))
    turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    odd = [torch.cat([x.new_zeros(T, H, 3), x], 2)[..., 3:] for x in (q, k, v)]  # rows off 16 bytes
    every = [x.repeat_interleave(2, 2)[..., ::2] for x in (q, k, v)]
    for views in (turned, odd, every):
        got = attend(*views, g.transpose(0, 1).contiguous().transpose(0, 1), (30, 30))
        assert all(torch.equal(got[x], base[x]) for x in base)
    from gdl_amd.functional import window_attention
    k1, v1 = (x[:, :1].detach().requires_grad_() for x in (k, v))
    out = window_attention(q, k1.expand(-1, H, -1), v1.expand(-1, H, -1), 30)
    grads = torch.autograd.grad(out, [k1, v1], g)
    shared = attend(q, k[:, :1], v[:, :1], g, 30)
    assert torch.equal(out, shared["out"])
    for x, y in zip(grads, (shared["dk"], shared["dv"])):
        torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-5)


def test_other_stream_and_graph_replay(dev):
    from gdl_amd.functional import window_attention
    q, k, v, g = make(dev, 600, 4, 2, 64, BF16, seed=13)
    ptr, mask = torch.tensor([0, 350, 600], device=dev), (torch.arange(600) % 5 != 0).to(dev)
    table = torch.randn(16, 4, device=dev, dtype=BF16)
    kw = dict(ptr=ptr, mask=mask, sinks=4, bias=table)
    want = window_attention(q, k, v, (50, 0), **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = window_attention(q, k, v, (50, 0), **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v, table)]

    def step():
        o = window_attention(*leaves[:3], (50, 0), ptr=ptr, mask=mask, sinks=4, bias=leaves[3])
        return [o] + list(torch.autograd.grad(o, leaves, g))

    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for n in range(4):
        with torch.no_grad():
            for x in leaves:
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_no_tokens(dev):
    for dtype in (F32, BF16):
        q, k, v, g = make(dev, 0, 2, 1, 16, dtype)
        table = torch.randn(8, 2, device=dev, dtype=dtype)
        got = attend(q, k, v, g, (4, 4), table, max_distance=16)
        assert got["out"].shape == (0, 2, 16) and (got["dbias"] == 0).all()


def test_refusals(dev):
    from gdl_amd.functional import window_attention
    q, k, v, _ = make(dev, 20, 4, 2, 16, F32)
    bad = [
        (ValueError, dict(q=q[:, :3])), (ValueError, dict(v=v[:19])), (ValueError, dict(q=q[0])),
        (TypeError, dict(k=k.bfloat16())), (TypeError, dict(q=q.double(), k=k.double(), v=v.double())),
        (RuntimeError, dict(k=k.cpu())), (ValueError, dict(window=(-2, 0))),
        (RuntimeError, dict(sinks=-1)), (RuntimeError, dict(sinks=257)),
        (ValueError, dict(mask=torch.ones(19, dtype=torch.bool, device=dev))),
        (ValueError, dict(mask=torch.ones(20, device=dev))),
        (ValueError, dict(ptr=torch.tensor([0], device=dev))),
        (ValueError, dict(bias=torch.zeros(8, 3, device=dev))), (ValueError, dict(bias=torch.zeros(7, 4, device=dev))),
        (ValueError, dict(bias=torch.zeros(512, 4, device=dev))),
        (ValueError, dict(bias=torch.zeros(32, 4, device=dev), max_distance=8)),
        (ValueError, dict(bias=torch.zeros(32, 4, device=dev), max_distance=2000)),
        (ValueError, dict(q=torch.zeros(20, 4, 136, device=dev), k=torch.zeros(20, 2, 136, device=dev),
                          v=torch.zeros(20, 2, 136, device=dev))),
    ]
    for error, change in bad:
        with pytest.raises(error):
            window_attention(**(dict(q=q, k=k, v=v, window=(4, 4)) | change))
    x = q.clone().requires_grad_()
    first = torch.autograd.grad(window_attention(x, k, v, 4).sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)


def test_bad_offsets_stay_in_bounds(dev):
    """Offsets outside the tokens, or not ascending, read nothing that is not there."""
    q, k, v, g = make(dev, 50, 1, 1, 16, F32)
    for ptr in ([-5, 20, 90], [30, 10, 50], [0, 0, 0], [60, 70, 80]):
        got = attend(q, k, v, g, (10, 10), ptr=torch.tensor(ptr, device=dev))
        assert got["out"].shape == q.shape


def test_buckets_of_distances(dev):
    from gdl_amd.functional import relative_buckets
    for buckets, maxd, two in ((32, 128, True), (32, 128, False), (8, 9, True), (5, 40, False), (64, 1000, True)):
        d = torch.arange(-1200, 1201)
        want = torch.tensor([bucket(int(x), buckets, maxd, two) for x in d])
        assert torch.equal(relative_buckets(d.to(dev), buckets, maxd, two).cpu(), want)
