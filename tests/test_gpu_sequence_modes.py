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


OPS = {"window_attention": lambda a: (*a, 5, 0, 2, 9, 0.25), "gated_recurrence": lambda a: (*a, True, 8.0),
       "window_attention_step": lambda a: (*a, 1, 9, 0.25), "window_cache_fill": lambda a: (*a[:4], 0, a[4], None),
       "gated_recurrence_step": lambda a: (*a, None, 8.0)}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("bias", [True, False])
def test_the_ops_are_what_they_say(dev, name, bias):
    """Schemas, registered gradients and shapes against what the ops do, all their outputs."""
    args = _args(name, dev)
    if not bias and name.startswith("window_attention"):
        args[3 if name == "window_attention" else 6] = None
    if name in ("window_attention", "gated_recurrence"):
        args = [t.requires_grad_() if t is not None and t.is_floating_point() else t for t in args]
    torch.library.opcheck(getattr(torch.ops.geoembodied, name).default, OPS[name](args))


def test_batches(dev):
    """vmap, and gradients of several vectors at once: a call each, or the same."""
    from gdl_amd.functional import gated_recurrence, window_attention
    torch.manual_seed(3)
    q, k, v = (torch.randn(3, 20, 2, 16, device=dev) for _ in range(3))
    out = torch.func.vmap(lambda a, b, c: window_attention(a, b, c, 4))(q, k, v)
    assert torch.equal(out, torch.stack([window_attention(a, b, c, 4) for a, b, c in zip(q, k, v)]))
    x = q[0].clone().requires_grad_()
    g = torch.randn(3, 20, 2, 16, device=dev)
    for f in (lambda y: window_attention(y, k[0], v[0], 4), lambda y: gated_recurrence(y[:, 0], k[0, :, 0], v[0, :, 0], v[0, 0, 0])[0]):
        out = f(x)
        rows = g if out.dim() == 3 else g[:, :, 0]
        many, = torch.autograd.grad(out, x, rows, is_grads_batched=True, retain_graph=True)
        assert torch.equal(many, torch.stack([torch.autograd.grad(out, x, r, retain_graph=True)[0] for r in rows]))


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
