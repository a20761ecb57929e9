"""CPU tests of the memory that a window cache may have: streams and heads that share some would be
written and read without order, so they are refused, by the class and by the C entries."""

import pytest
import torch

from gdl_amd import _native
from gdl_amd.functional import WindowCache

B, H, S, D = 3, 2, 6, 16


def _good():
    buffer = torch.zeros(B, 2, H, S, D)
    return [torch.zeros(B, H, S, D), buffer[:, 0], torch.zeros(H, B, S, D).transpose(0, 1), torch.zeros(B, H, S + 2, D)[:, :, :S],
            torch.zeros(1, H, S, D), torch.zeros(H, S, D).unsqueeze(0).expand(1, H, S, D), torch.zeros(B, 1, S, D), torch.zeros(0, H, S, D)]


def _bad():
    row = torch.zeros(B * H * S * D)
    return [torch.zeros(1, H, S, D).expand(B, H, S, D), torch.zeros(B, 1, S, D).expand(B, H, S, D),
            row.as_strided((B, H, S, D), (S * D, S * D, D, 1)), row.as_strided((B, H, S, D), (2 * D, S * D, D, 1)),
            row.as_strided((B, H, S, D), (S * D, 2 * S * D, D, 1))]


@pytest.mark.parametrize("n", range(8))
def test_caches_that_lie_apart(n):
    WindowCache(_good()[n], _good()[n].clone(memory_format=torch.preserve_format), sinks=1)


@pytest.mark.parametrize("n", range(5))
def test_shared_memory_is_refused(n):
    good = torch.zeros(B, H, S, D)
    for k, v in ((_bad()[n], good), (good, _bad()[n])):
        with pytest.raises(ValueError, match="share memory"):
            WindowCache(k, v)


def test_one_tensor_for_both_is_refused():
    x = torch.zeros(B, H, S, D)
    with pytest.raises(ValueError, match="same memory"):
        WindowCache(x, x)


@pytest.mark.parametrize("n", range(5))
def test_the_entries_refuse_it(n):
    lib = _native.lib()
    st, sh = _bad()[n].stride()[:2]
    args = _native.pack_window_step(4096, 4096, 4096, 1 << 20, 1 << 24, H * D, D, H * D, D, H * D, D, st, sh, H * S * D, S * D, 4096, 0, 0,
                                    B, S, 1, 0, 0, H, H, D, 0, 0, 0.25)
    assert lib.geo_window_attention_step(args, 4096, None, 0, None) != 0
    assert "share memory" in lib.geo_last_error().decode()
    assert lib.geo_window_cache_fill(0, 4096, 4096, H * D, D, H * D, D, 4096, None, 20, B, H, D, 1 << 20, 1 << 24, H * S * D, S * D, st, sh,
                                     S, 1, None) != 0
    assert "share memory" in lib.geo_last_error().decode()
