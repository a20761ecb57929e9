"""CPU tests of the sequence operators' largest sizes: what a launch cannot hold (2^32 threads) is refused by the
C entries with the reason, ahead of any launch."""

import pytest

from gdl_amd import _native


def _refused(status):
    assert status != 0 and "too many workgroups" in _native.lib().geo_last_error().decode()


@pytest.mark.parametrize("tokens, channels", [(1 << 29, 4), (1 << 28, 65), (1 << 20, 64 << 9)])
def test_recurrence(tokens, channels):
    lib = _native.lib()

    def args(n):
        return _native.pack_recurrence(4096, 4096, 4096, channels, channels, channels, 4096, 0, 0, n, channels, 1, 1, 0, 8.0)

    _refused(lib.geo_recurrence_fwd(args(tokens), 4096, 4096, 4096, 4096, 0, None))
    _refused(lib.geo_recurrence_bwd(args(tokens), 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 0, None))
    # one chunk fewer is looked at further
    assert lib.geo_recurrence_fwd(args(tokens - 64), 4096, 4096, 4096, 4096, 0, None) != 0
    assert "workspace" in lib.geo_last_error().decode()


@pytest.mark.parametrize("tokens, heads", [((1 << 30) - 1, 3), (1 << 28, 16)])
def test_attention(tokens, heads):
    lib = _native.lib()
    args = _native.pack_window_attention(4096, 4096, 4096, *[heads * 8, 8] * 3, 0, 0, 0, 0, tokens, 1, 2000, 0, 0, 1, 0, heads, heads, 8, 0, 0, 0.3)
    _refused(lib.geo_window_attention_fwd(args, 4096, None, None, None))
    need = lib.geo_window_attention_bwd_workspace_bytes(args)
    _refused(lib.geo_window_attention_bwd(args, 4096, None, 4096, 4096, 4096, 4096, 4096, None, None, 4096, need, None))


def test_steps():
    lib = _native.lib()
    batch, slots, d = 1 << 23, 16, 8
    step = _native.pack_window_step(4096, 4096, 4096, 1 << 20, 1 << 40, *[2 * d, d] * 3, *[2 * slots * d, slots * d] * 2, 4096, 0, 0,
                                    batch, slots, 1, 1, 0, 2, 2, d, 0, 0, 0.3)
    _refused(lib.geo_window_attention_step(step, 4096, None, 0, None))
    _refused(lib.geo_window_cache_fill(1, 4096, 4096, 2 * d, d, 2 * d, d, 4096, None, 1 << 31, 4, 2, d, 1 << 20, 1 << 40,
                                       *[2 * slots * d, slots * d] * 2, slots, 1, None))
    args = _native.pack_recurrence(4096, 4096, 4096, 256, 256, 256, 4096, 0, 4096, 1 << 24, 257, 1 << 24, 0, 0, 8.0)
    _refused(lib.geo_recurrence_step(args, 4096, 4096, None))
