"""GPU tests of the gated linear recurrence: outputs and gradients against the definition, token by
token in float64, with derived bounds; differences; sequence borders; refusals."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SPACING = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


def make(dev, T, C, dtype, B=1, seed=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x, ga, gx, dh = ((spread * torch.randn(T, C, generator=gen)).to(dev, dtype) for _ in range(4))
    a = 0.9 + 0.0999 * torch.rand(C, generator=gen, dtype=torch.float64)
    decay = torch.log(torch.expm1(-torch.log(a) / 4)).float().to(dev)
    state, dlast = (torch.randn(B, C, generator=gen).to(dev) for _ in range(2))
    return x, ga, gx, decay, state, dh, dlast


def definition(x, ga, gx, decay, state, dh, dlast, ptr, reverse, rate):
    """Values and error bounds.  e = 2^-24: a gate's factors and sums carry some 16 roundings, a
    decay's log is off by e (|log a| + 8 |log a|) at most, m by 16 e relatively (its argument's error
    is relative too), and the scan accumulates errors as it does values: bounds follow the same
    recurrences over absolute values, with 40 e per term."""
    u, e, z0 = UNIT[x.dtype], 2.0 ** -24, SPACING[x.dtype] / 2
    x64, ga64, gx64, dh64 = (t.detach().double().cpu() for t in (x, ga, gx, dh))
    dec, dl = decay.detach().double().cpu(), dlast.double().cpu()
    r, z = torch.sigmoid(ga64), torch.sigmoid(gx64)
    lr = -rate * torch.nn.functional.softplus(dec)
    la = lr * r
    a = torch.exp(la)
    m = torch.sqrt(-torch.expm1(2 * la))
    T, C = x.shape
    B = len(ptr) - 1
    h, before, G = (torch.zeros(T, C, dtype=torch.float64) for _ in range(3))
    ah, ab, aG = (torch.zeros(T, C, dtype=torch.float64) for _ in range(3))
    eh, eb, eG = (torch.zeros(T, C, dtype=torch.float64) for _ in range(3))
    st = state.detach().double().cpu() if state is not None else torch.zeros(B, C, dtype=torch.float64)
    last, dstate, elast, edstate = (torch.zeros(B, C, dtype=torch.float64) for _ in range(4))
    da = 40 * e * (1 + la.abs())  # relative error of a
    for b in range(B):
        order = list(range(ptr[b], ptr[b + 1]))
        order = order[::-1] if reverse else order
        now, mag, err = st[b], st[b].abs(), torch.zeros(C, dtype=torch.float64)
        for t in order:
            before[t], ab[t], eb[t] = now, mag, err
            add = m[t] * z[t] * x64[t]
            err = a[t] * err + da[t] * a[t] * mag + 40 * e * add.abs()
            now, mag = a[t] * now + add, a[t] * mag + add.abs()
            h[t], ah[t], eh[t] = now, mag, err
        last[b], elast[b] = now, err
        now, mag, err = dl[b], dl[b].abs(), torch.zeros(C, dtype=torch.float64)
        for t in reversed(order):
            G[t], aG[t], eG[t] = now + dh64[t], mag + dh64[t].abs(), err + 2 * e * (mag + dh64[t].abs())
            now, mag = a[t] * G[t], a[t] * aG[t]
            err = a[t] * eG[t] + da[t] * mag
        dstate[b], edstate[b] = now, err
    live = torch.zeros(T, 1, dtype=torch.float64)
    live[ptr[0]:ptr[-1]] = 1
    inn = z * x64
    slope = torch.where(m > 0, a * a * la / m.clamp(min=1e-300), torch.zeros_like(m))
    dla = G * (a * before * la - slope * inn)   # times log a
    edla = eG * ((a * ab * la).abs() + (slope * inn).abs()) + aG * (
        (a * la).abs() * (eb + da * ab) + 60 * e * (1 + la.abs()) * ((a * ab * la).abs() + (slope * inn).abs()))
    want = {"h": h, "last": last, "dx": G * m * z, "dgx": G * m * inn * (1 - z), "dga": dla * (1 - r),
            "ddecay": dla.sum(0) * torch.sigmoid(dec) / torch.nn.functional.softplus(dec), "dstate": dstate}
    tol = {"h": eh, "last": elast, "dx": (m * z).abs() * (eG + 40 * e * aG),
           "dgx": (m * inn).abs() * (1 - z) * (eG + 40 * e * aG) + 2 * e * aG * (m * inn).abs(),
           "dga": edla * (1 - r) + 2 * e * dla.abs(), "dstate": edstate}
    ratio = torch.sigmoid(dec) / torch.nn.functional.softplus(dec)
    tol["ddecay"] = (edla.sum(0) + e * (T / 16 + 64) * dla.abs().sum(0)) * ratio + 40 * e * want["ddecay"].abs()
    for n in ("h", "dx", "dgx", "dga"):
        want[n] = want[n] * live
        tol[n] = tol[n] + u * want[n].abs() + z0
    return want, {n: t + 1e-30 for n, t in tol.items()}


def run(x, ga, gx, decay, state, dh, dlast, **kw):
    from gdl_amd.functional import gated_recurrence
    leaves = {n: t.detach().requires_grad_() for n, t in dict(dx=x, dga=ga, dgx=gx, ddecay=decay, dstate=state).items()
              if t is not None}
    h, last = gated_recurrence(leaves["dx"], leaves["dga"], leaves["dgx"], leaves["ddecay"], state=leaves.get("dstate"), **kw)
    grads = torch.autograd.grad([h, last], list(leaves.values()), [dh, dlast])
    return {"h": h, "last": last, **dict(zip(leaves, grads))}


def check(got, want, tol, what):
    for n, g in got.items():
        off = (g.detach().double().cpu() - want[n]).abs()
        bad = ~(off <= tol[n])
        assert g.shape == want[n].shape and not bad.any(), (what, n, int(bad.sum()), bad.nonzero()[:4].tolist(),
                                                            off[bad][:4].tolist(), tol[n][bad][:4].tolist())


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("reverse", [False, True], ids=["ahead", "reverse"])
@pytest.mark.parametrize("lengths,C,state", [
    ([1], 1, False), ([31], 3, True), ([32], 64, False), ([33], 65, True), ([500], 130, True), ([3000], 7, False),
    ([1, 0, 5, 64, 0, 33, 2], 20, True), ([0, 0, 70], 128, True), ([40, 0], 6, True), ([1] * 100, 9, True),
    ([700, 1, 900], 200, False)])
def test_against_definition(dev, dtype, reverse, lengths, C, state):
    print(lengths[:5], C, dtype, reverse, flush=True)
    ptr = [0]
    for n in lengths:
        ptr.append(ptr[-1] + n)
    x, ga, gx, decay, st, dh, dlast = make(dev, ptr[-1], C, dtype, len(lengths), seed=C)
    st = st if state else None
    want, tol = definition(x, ga, gx, decay, st, dh, dlast, ptr, reverse, 8.0)
    got = run(x, ga, gx, decay, st, dh, dlast, reverse=reverse,
              ptr=torch.tensor(ptr, device=dev) if len(lengths) > 1 or C == 3 else None)
    check(got, want, tol, (lengths[:4], C))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_extreme_gates(dev, dtype):
    """Gates of +-60 and decays of +-30 (a = 1 and a = 0 to the last bit), odd rate."""
    T, C = 200, 40
    x, ga, gx, decay, st, dh, dlast = make(dev, T, C, dtype, seed=5, spread=20.0)
    decay = torch.linspace(-30, 30, C, device=dev)
    want, tol = definition(x, ga, gx, decay, st, dh, dlast, [0, T], False, 0.37)
    got = run(x, ga, gx, decay, st, dh, dlast, rate=0.37)
    assert all(torch.isfinite(v).all() for v in got.values())
    check(got, want, tol, "extreme")


def test_tokens_outside_sequences_and_bad_values(dev):
    x, ga, gx, decay, st, dh, dlast = make(dev, 300, 16, F32, 3, seed=6)
    ptr = [20, 100, 130, 260]
    want, tol = definition(x, ga, gx, decay, st, dh, dlast, ptr, False, 8.0)
    p = torch.tensor(ptr, device=dev)
    got = run(x, ga, gx, decay, st, dh, dlast, ptr=p)
    check(got, want, tol, "outside")
    for junk in (math.nan, math.inf):
        y = [t.clone() for t in (x, ga, gx)]
        for t in y:
            t[:20], t[100:130], t[260:] = junk, junk, junk  # outside, and the second sequence
        for reverse in (False, True):
            clean = run(x, ga, gx, decay, st, dh, dlast, ptr=p, reverse=reverse)
            bad = run(*y, decay, st, dh, dlast, ptr=p, reverse=reverse)
            rest = torch.ones(300, dtype=torch.bool)
            rest[100:130] = False
            for n in ("h", "dx", "dga", "dgx"):
                assert torch.equal(bad[n][rest.to(dev)], clean[n][rest.to(dev)]), n
            for n in ("last", "dstate"):
                assert torch.equal(bad[n][::2], clean[n][::2]), n


def test_gradient_against_differences(dev):
    """Central differences in float32 with a step of 1/64: truncation below 1e-3 of the sum's scale,
    rounding 2e-7 times the outputs' size over the step."""
    from gdl_amd.functional import gated_recurrence
    T, C = 120, 8
    x, ga, gx, decay, st, dh, dlast = make(dev, T, C, F32, 2, seed=8)
    ptr = torch.tensor([0, 50, 120], device=dev)
    got = run(x, ga, gx, decay, st, dh, dlast, ptr=ptr)
    inputs = dict(dx=x, dga=ga, dgx=gx, ddecay=decay, dstate=st)
    gen, step_size = torch.Generator().manual_seed(9), 1 / 64
    for name, t in inputs.items():
        step = torch.randn(t.shape, generator=gen).to(dev)

        def loss(sign):
            y = {n: s + sign * step_size * step if n == name else s for n, s in inputs.items()}
            h, last = gated_recurrence(y["dx"], y["dga"], y["dgx"], y["ddecay"], state=y["dstate"], ptr=ptr)
            return ((h.double() * dh.double()).sum() + (last.double() * dlast.double()).sum()).item()

        slope = (loss(1) - loss(-1)) / (2 * step_size)
        want, scale = ((f(got[name].double()) * f(step.double())).sum().item() for f in (lambda q: q, torch.abs))
        assert abs(slope - want) <= 1e-3 * scale + 2e-7 / step_size * math.sqrt(T * C) * 3, (name, slope, want)


def test_partial_gradients_and_types(dev):
    from gdl_amd.functional import gated_recurrence
    x, ga, gx, decay, st, dh, dlast = make(dev, 90, 12, BF16, seed=10)
    both = run(x, ga, gx, decay, st, dh, dlast)
    for use_h, use_last in ((True, False), (False, True)):
        leaf = x.detach().requires_grad_()
        h, last = gated_recurrence(leaf, ga, gx, decay, state=st)
        got, = torch.autograd.grad([h] if use_h else [last], leaf, [dh] if use_h else [dlast])
        zero = run(x, ga, gx, decay, st, dh if use_h else torch.zeros_like(dh), dlast if use_last else torch.zeros_like(dlast))
        assert torch.equal(got, zero["dx"])
    low = run(x, ga, gx, decay.bfloat16(), st.bfloat16(), dh, dlast)
    assert low["ddecay"].dtype is BF16 and low["dstate"].dtype is BF16 and low["last"].dtype is F32
    assert both["ddecay"].dtype is F32


def test_strides_streams_graph_and_same_bits(dev):
    from gdl_amd.functional import gated_recurrence
    T, C = 2000, 96
    wide = torch.randn(T, 3 * C + 1, device=dev).to(BF16)
    for parts in ((wide[:, :C], wide[:, C:2 * C], wide[:, 2 * C:3 * C]), tuple(wide[:, n + 1:n + 1 + C] for n in (0, C, 2 * C)),
                  tuple(wide.t().contiguous().t()[:, n:n + C] for n in (0, C, 2 * C))):
        decay = torch.zeros(C, device=dev)
        one, two = gated_recurrence(*parts, decay), gated_recurrence(*(t.contiguous() for t in parts), decay)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    x, ga, gx, decay, st, dh, dlast = make(dev, T, C, BF16, 2, seed=11)
    ptr = torch.tensor([0, 900, T], device=dev)
    want = run(x, ga, gx, decay, st, dh, dlast, ptr=ptr)
    again = run(x, ga, gx, decay, st, dh, dlast, ptr=ptr)
    assert all(torch.equal(want[n], again[n]) for n in want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(x, ga, gx, decay, st, dh, dlast, ptr=ptr)
    torch.cuda.synchronize()
    assert all(torch.equal(want[n], other[n]) for n in want)
    inputs = [t.clone() for t in (x, ga, gx)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*inputs, decay, st, dh, dlast, ptr=ptr)
    for n in range(4):
        for t in inputs:
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        eager = run(*inputs, decay, st, dh, dlast, ptr=ptr)
        assert all(torch.equal(out[k], eager[k]) for k in out)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,C", [(1, 1), (3, 65), (40, 128), (7, 1000)])
def test_step(dev, dtype, B, C):
    """A stream stepped token by token ends where the scan ends, and each step is the definition."""
    from gdl_amd.functional import gated_recurrence, gated_recurrence_step
    x, ga, gx, decay, st, dh, dlast = make(dev, 5 * B, C, dtype, B, seed=B)
    state = st
    for n in range(5):
        rows = slice(n * B, n * B + B)
        want, tol = definition(x[rows], ga[rows], gx[rows], decay, state, dh[rows], dlast, list(range(B + 1)), False, 8.0)
        h, new = gated_recurrence_step(x[rows], ga[rows], gx[rows], decay, state)
        check({"h": h, "last": new}, want, tol, n)
        state = new
    order = torch.arange(5 * B, device=dev).view(5, B).t().reshape(-1)
    _, last = gated_recurrence(x[order], ga[order], gx[order], decay, ptr=torch.arange(0, 5 * B + 1, 5, device=dev), state=st)
    torch.testing.assert_close(state, last, rtol=1e-5, atol=1e-6)


def test_no_tokens(dev):
    x, ga, gx, decay, st, dh, dlast = make(dev, 0, 5, F32, 2)
    got = run(x, ga, gx, decay, st, dh, dlast, ptr=torch.tensor([0, 0, 0], device=dev))
    assert torch.equal(got["last"], st) and torch.equal(got["dstate"], dlast) and (got["ddecay"] == 0).all()
    assert got["h"].shape == (0, 5)


def test_refusals(dev):
    from gdl_amd.functional import gated_recurrence, gated_recurrence_step
    x, ga, gx, decay, st, _, _ = make(dev, 10, 4, F32)
    bad = [(ValueError, dict(gate_a=ga[:9])), (ValueError, dict(decay=decay[:3])), (TypeError, dict(gate_x=gx.bfloat16())),
           (TypeError, dict(x=x.double(), gate_a=ga.double(), gate_x=gx.double())), (ValueError, dict(rate=0.0)),
           (ValueError, dict(state=st[:, :2])), (ValueError, dict(ptr=torch.tensor([0], device=dev))),
           (RuntimeError, dict(decay=decay.cpu())), (TypeError, dict(decay=decay.long()))]
    for error, change in bad:
        with pytest.raises(error):
            gated_recurrence(**(dict(x=x, gate_a=ga, gate_x=gx, decay=decay) | change))
    state = torch.zeros(10, 4, device=dev)
    for error, change in [(ValueError, dict(state=state.half())), (ValueError, dict(state=state[:4])), (ValueError, dict(rate=-1)),
                          (RuntimeError, dict(x=x.clone().requires_grad_()))]:
        with pytest.raises(error):
            gated_recurrence_step(**(dict(x=x, gate_a=ga, gate_x=gx, decay=decay, state=state) | change))
