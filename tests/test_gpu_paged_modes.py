"""GPU tests of the paged caches in modes that see no raw pointers: traced and compiled programs compute what the eager
calls do."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from test_paged_host import CALLS

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


OPS = {"paged_write": lambda a: a, "paged_read": lambda a: (*a[:5], a[5], None, 20, torch.float32),
       "paged_attention": lambda a: (*a, 9, 0.25), "paged_attention_step": lambda a: (*a, 9, 0.25)}


@pytest.mark.parametrize("name", CALLS)
def test_the_ops_are_what_they_say(dev, name):
    """Schemas, aliasing and fake kernels against what the ops do."""
    args = OPS[name](_args(name, dev))
    checks = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    torch.library.opcheck(getattr(torch.ops.geoembodied, name).default, tuple(args), test_utils=checks)
