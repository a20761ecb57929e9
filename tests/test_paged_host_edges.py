"""CPU tests of calls at the edges of what paged caches take: no streams, and what their entries do before any launch."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from gdl_amd import _native
from gdl_amd.functional.recurrence import packets_as_sequences


def _pool(table=4096):
    return _native.pack_paged(4096, 1 << 20, 0, 0, table, 2, 6, 2, 0, 2, 16, 64)


def _step(pool, batch):
    return _native.pack_paged_step(pool, 0, 0, 0, 64, 16, 32, 16, 32, 16, 0, 0, 0, batch, 0, 0, 4, 0, 0, 0.25)


def test_no_streams_need_no_table():
    """Tensors without elements have no address: nothing of theirs is asked for."""
    lib = _native.lib()
    assert lib.geo_paged_attention_step(_step(_pool(0), 0), None, None, 0, None) == 0
    assert lib.geo_paged_attention_step(_step(_pool(0), 1), None, None, 0, None) != 0
    assert "null table" in lib.geo_last_error().decode()


def test_packets_are_refused():
    lib = _native.lib()
    for args, part in (((0, 4096, 4096, 8, 2, 8, 4096, 4096), "null tensor"), ((4096, 0, 4096, 8, 2, 8, 4096, 4096), "null tensor"),
                       ((4096, 4096, 0, 8, 2, 8, 4096, 4096), "null tensor"), ((4096, 4096, 4096, 8, 2, 8, 0, 4096), "null tensor"),
                       ((4096, 4096, 4096, 8, 2, 8, 4096, 0), "null tensor"), ((4096, 4096, 4096, 8, 0, 8, 4096, 4096), "0 streams"),
                       ((4096, 4096, 4096, 8, 1 << 30, 8, 4096, 4096), "streams"), ((4096, 4096, 4096, 8, 2, -1, 4096, 4096), "-1 channels"),
                       ((4096, 4096, 4096, 8, 1 << 29, 1 << 10, 4096, 4096), "too many workgroups")):
        assert lib.geo_recurrence_packets(*args, None) != 0, args
        assert part in lib.geo_last_error().decode(), (args, lib.geo_last_error())


def test_a_trace_holds_the_packets_op():
    args = torch.tensor([0, 3, 3, 9]), torch.tensor([0, 5, -2]), torch.zeros(3, 8)
    for mode in ("fake", "symbolic"):
        assert "geoembodied.recurrence_packets." in make_fx(packets_as_sequences, tracing_mode=mode)(*args).code


def test_packets_of_other_shapes_are_refused():
    ptr, start, state = torch.tensor([0, 3, 9]), torch.tensor([0, -2]), torch.zeros(2, 8)
    for bad in ((ptr[:2], start, state), (ptr, start[:1], state), (ptr, start, state[:1]), (ptr[:1], start[:0], state[:0]),
                (ptr, start, state[0]), (ptr, start.view(1, 2), state)):
        with pytest.raises(ValueError, match="packets_as_sequences"):
            packets_as_sequences(*bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        packets_as_sequences(ptr, start, state)


@pytest.mark.parametrize("kw", [dict(page=0), dict(page=-64), dict(page=32), dict(page=100), dict(tokens=0), dict(tokens=None), dict(batch=0)])
def test_caches_of_a_block_are_refused(kw):
    from gdl_amd.sequence import PointSequenceBlock
    args = {"batch": 2, "dtype": torch.int8, "tokens": 10, **kw}
    with pytest.raises(ValueError):
        PointSequenceBlock(32, 2, None).new_cache(args.pop("batch"), args.pop("dtype"), **args)
