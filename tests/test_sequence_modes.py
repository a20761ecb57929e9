"""CPU tests of the sequence operators in modes that see no raw pointers: tracing records ops that compute
the results, compilation takes them whole, forward-mode differentiation is refused."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from gdl_amd import functional as F

T, H, HK, D, C, B = 24, 4, 2, 16, 12, 3


def _attention(q, k, v, bias, ptr, mask):
    return F.window_attention(q, k, v, (5, 0), sinks=2, ptr=ptr, mask=mask, bias=bias, max_distance=9)


def _attention_args(dtype=torch.float32):
    return (torch.randn(T, H, D, dtype=dtype), *(torch.randn(T, HK, D, dtype=dtype) for _ in range(2)),
            torch.randn(8, H, dtype=dtype), torch.tensor([0, 10, T]), torch.ones(T, dtype=torch.bool))


def _recurrence(x, ga, gx, decay, state, ptr):
    return F.gated_recurrence(x, ga, gx, decay, state=state, ptr=ptr, reverse=True)


def _recurrence_args(dtype=torch.float32):
    return (*(torch.randn(T, C, dtype=dtype) for _ in range(3)), torch.randn(C), torch.randn(B, C), torch.tensor([0, 10, 10, T]))


def _step(q, k, v, kc, vc, pos, bias):
    return F.window_attention_step(q, k, v, F.WindowCache(kc, vc, sinks=1), pos, bias=bias, max_distance=9)


def _step_args():
    return (torch.randn(B, H, D), *(torch.randn(B, HK, D) for _ in range(2)), *(torch.zeros(B, HK, 8, D) for _ in range(2)),
            torch.arange(B), torch.randn(8, H))


def _fill(k, v, kc, vc, ptr):
    F.WindowCache(kc, vc).fill(k, v, ptr)
    return kc + vc


def _fill_args():
    return (*(torch.randn(T, HK, D) for _ in range(2)), *(torch.zeros(B, HK, 8, D) for _ in range(2)), torch.tensor([0, 10, 10, T]))


def _recurrence_step(x, ga, gx, decay, state):
    return F.gated_recurrence_step(x, ga, gx, decay, state)


def _recurrence_step_args():
    return (*(torch.randn(B, C) for _ in range(3)), torch.randn(C), torch.randn(B, C))


CALLS = {"window_attention": (_attention, _attention_args), "gated_recurrence": (_recurrence, _recurrence_args),
         "window_attention_step": (_step, _step_args), "window_cache_fill": (_fill, _fill_args),
         "gated_recurrence_step": (_recurrence_step, _recurrence_step_args)}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("mode", ["fake", "symbolic"])
def test_a_trace_holds_the_op(name, mode):
    call, args = CALLS[name]
    graph = make_fx(call, tracing_mode=mode)(*args())
    assert f"geoembodied.{name}." in graph.code


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["window_attention", "gated_recurrence"])
def test_a_trace_holds_the_backward(name, dtype):
    call, args = CALLS[name]
    args = args(dtype)

    def grads(*inputs):
        leaves = [t.detach().requires_grad_() if t.is_floating_point() else t for t in inputs]
        out = call(*leaves)
        out = out if torch.is_tensor(out) else out[0]
        wanted = [t for t in leaves if t.is_floating_point()]
        return torch.autograd.grad(out.float().sum(), wanted)

    graph = make_fx(grads, tracing_mode="fake")(*args)
    assert f"geoembodied.{name}." in graph.code and f"geoembodied.{name}_backward." in graph.code


@pytest.mark.parametrize("name", CALLS)
def test_compilation_takes_the_call_whole(name):
    call, args = CALLS[name]
    seen = []

    def backend(module, inputs):
        seen.append(module.print_readable(print_output=False))
        raise _Done

    class _Done(Exception):
        pass

    torch._dynamo.reset()
    with pytest.raises(Exception):  # the backend stops before anything runs
        torch.compile(call, backend=backend, fullgraph=True)(*args())
    assert len(seen) == 1 and name in seen[0]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad):
    call, args = CALLS[name]
    inputs = list(args())
    if grad and name in ("window_attention", "gated_recurrence"):
        inputs[1].requires_grad_()
    with torch.autograd.forward_ad.dual_level():
        inputs[0] = torch.autograd.forward_ad.make_dual(inputs[0], torch.ones_like(inputs[0]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*inputs)
    if name != "window_cache_fill":
        rest = args()[1:]
        x = args()[0]
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(lambda y: call(y, *rest), (x,), (torch.ones_like(x),))


def test_bucket_configurations_are_checked_when_traced():
    q, k, v, bias, ptr, mask = _attention_args()
    with pytest.raises(ValueError):
        make_fx(lambda q, k, v, b: F.window_attention(q, k, v, 3, bias=b, max_distance=2000), tracing_mode="fake")(q, k, v, bias)
