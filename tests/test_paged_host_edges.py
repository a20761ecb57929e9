"""CPU tests of calls at the edges of what paged caches take: no streams, and what their entries do before any launch."""

from gdl_amd import _native


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
