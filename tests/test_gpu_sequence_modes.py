"""GPU tests of the sequence operators in modes that see no raw pointers: traced and compiled programs
compute what the eager calls do, gradients too."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from test_sequence_modes import CALLS

pytestmark = pytest.mark.gpu


def _args(name, dev, seed=0):
    torch.manual_seed(seed)
    return [t.to(dev) for t in CALLS[name][1]()]


def _equal(a, b):
    a, b = ([x] if torch.is_tensor(x) else x for x in (a, b))
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("name", CALLS)
def test_traces_compute(dev, name):
    """Traced with one set of inputs, run with another."""
    call = CALLS[name][0]
    want = call(*_args(name, dev, 1))
    assert _equal(torch.jit.trace(call, _args(name, dev), check_trace=False)(*_args(name, dev, 1)), want)
    assert _equal(make_fx(call)(*_args(name, dev))(*_args(name, dev, 1)), want)
    torch._dynamo.reset()
    compiled = torch.compile(call, backend="aot_eager", fullgraph=True)
    compiled(*_args(name, dev))
    assert _equal(compiled(*_args(name, dev, 1)), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", ["window_attention", "gated_recurrence"])
def test_compiled_gradients(dev, name, dtype):
    call = CALLS[name][0]
    torch.manual_seed(2)
    args = [t.to(dev) for t in CALLS[name][1](dtype)]
    results = []
    torch._dynamo.reset()
    for f in (call, torch.compile(call, backend="aot_eager", fullgraph=True)):
        leaves = [t.detach().clone().requires_grad_() if t.is_floating_point() else t for t in args]
        out = f(*leaves)
        out = [out] if torch.is_tensor(out) else list(out)
        g = [torch.linspace(-1, 1, o.numel(), device=dev).view(o.shape).to(o.dtype) for o in out]
        results.append([o.detach() for o in out] + list(torch.autograd.grad(out, [t for t in leaves if t.is_floating_point()], g)))
    assert _equal(*results)


@pytest.mark.parametrize("name", ["window_attention", "gated_recurrence"])
def test_second_derivatives_are_refused(dev, name):
    call = CALLS[name][0]
    args = _args(name, dev)
    args[0].requires_grad_()
    out = call(*args)
    out = out if torch.is_tensor(out) else out[0]
    first, = torch.autograd.grad(out.sum(), args[0], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), args[0])
    # forward over reverse
    x = args[0].detach()
    with torch.autograd.forward_ad.dual_level():
        leaf = x.clone().requires_grad_()
        args[0] = leaf
        out = call(*args)
        out = out if torch.is_tensor(out) else out[0]
        g = torch.autograd.forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, leaf, g)
