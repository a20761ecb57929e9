"""CPU tests of the sequence operators' host side: the C entries refuse bad arguments before they touch
a GPU, sizes and packed structures agree with the header, buckets and module paths."""

import math

import pytest
import torch

from gdl_amd import _native
from gdl_amd.functional import relative_buckets


def _attention(dtype=0, q=4096, tokens=8, heads=4, kv_heads=2, head_dim=16, left=4, right=0, sinks=0, strides=None, bias=0,
               lut=0, buckets=0, max_distance=0):
    strides = strides or [64, 16, 32, 16, 32, 16]
    return _native.pack_window_attention(q, q, q, *strides, 0, 0, bias, lut, tokens, 1, left, right, sinks, dtype, 0, heads,
                                         kv_heads, head_dim, buckets, max_distance, 0.25)


def _refused(status, part):
    assert status != 0
    assert part in _native.lib().geo_last_error().decode()


def test_structures_fill_the_header_s():
    assert len(_attention()) == 176
    assert len(_native.pack_window_step(*[0] * 28, 0.0)) == 200
    assert len(_native.pack_recurrence(*[0] * 14, 0.0)) == 112


@pytest.mark.parametrize("change, part", [
    (dict(dtype=2), "dtype code 2"),
    (dict(tokens=-1), "tokens"),
    (dict(tokens=1 << 30), "tokens"),
    (dict(heads=5), "no multiple"),
    (dict(head_dim=12), "head size 12"),
    (dict(head_dim=136), "head size 136"),
    (dict(left=-1), "window of -1"),
    (dict(sinks=257), "257 first tokens"),
    (dict(q=0), "null q, k or v"),
    (dict(q=4100), "multiples of 16 bytes"),
    (dict(strides=[63, 16, 32, 16, 32, 16]), "multiples of 16 bytes"),
    (dict(strides=[64, 16, 8, 16, 32, 16]), "below the head size"),
    (dict(bias=4096, lut=4096, buckets=257, max_distance=128), "257 buckets"),
    (dict(bias=4096, lut=4096, buckets=32, max_distance=1025), "distance 1025"),
])
def test_attention_refuses(change, part):
    args = _attention(**change)
    _refused(_native.lib().geo_window_attention_fwd(args, 4096, 0, 0, 0), part)
    assert _native.lib().geo_window_attention_bwd_workspace_bytes(args) == 0


def test_attention_of_no_tokens_is_done():
    assert _native.lib().geo_window_attention_fwd(_attention(tokens=0, q=0), 0, 0, 0, 0) == 0


def test_attention_backward_refuses_a_small_workspace():
    lib, args = _native.lib(), _attention()
    need = lib.geo_window_attention_bwd_workspace_bytes(args)
    assert need >= 8 * 4 * 4  # a float for each token and head
    _refused(lib.geo_window_attention_bwd(args, 4096, 0, 4096, 4096, 4096, 4096, 4096, 0, 0, 4096, need - 1, 0), "needed")


def test_recurrence_refuses():
    lib = _native.lib()

    def args(dtype=0, tokens=8, channels=4, sequences=1, x=4096):
        return _native.pack_recurrence(x, x, x, channels, channels, channels, x, 0, 0, tokens, channels, sequences, dtype, 0, 8.0)

    assert lib.geo_recurrence_carry_size(0, 4) == 0 and lib.geo_recurrence_carry_size(65, 4) == 2 * lib.geo_recurrence_carry_size(64, 4)
    for bad, part in ((dict(dtype=2), "dtype code 2"), (dict(tokens=-1), "-1 tokens"), (dict(tokens=(1 << 31) - 64), "tokens"),
                      (dict(sequences=0), "0 sequences"), (dict(x=0), "null tensor")):
        _refused(lib.geo_recurrence_fwd(args(**bad), 4096, 4096, 4096, 4096, 1 << 20, 0), part)
    _refused(lib.geo_recurrence_fwd(args(), 4096, 4096, 4096, 4096, 8, 0), "needed")
    _refused(lib.geo_recurrence_step(args(), 4096, 4096, 0), "one token for each")
    assert lib.geo_recurrence_fwd(args(tokens=0), 0, 0, 0, 0, 0, 0) == 0


@pytest.mark.parametrize("buckets, max_distance, two_sided", [(32, 128, True), (32, 128, False), (8, 16, True), (2, 2, False)])
def test_buckets(buckets, max_distance, two_sided):
    d = torch.arange(-3 * max_distance, 3 * max_distance + 1)
    got = relative_buckets(d, buckets, max_distance, two_sided)
    assert got.min() >= 0 and got.max() < buckets
    side = buckets // 2 if two_sided else buckets
    exact = side // 2
    for x, y in zip(d.tolist(), got.tolist()):
        far = abs(x) if two_sided else max(-x, 0)
        if far < exact:
            want = far
        else:
            want = min(side - 1, exact + int(math.log(far / exact) / math.log(max_distance / exact) * (side - exact) + 1e-9))
        assert y == want + (side if two_sided and x > 0 else 0), x


def test_module_paths():
    import geoembodied  # noqa: F401
    from geoembodied.functional.attention import window_attention
    from geoembodied.functional.recurrence import gated_recurrence
    import gdl_amd.functional as F

    assert window_attention is F.window_attention and gated_recurrence is F.gated_recurrence


def test_cpu_tensors_are_refused():
    from gdl_amd.functional import gated_recurrence, window_attention

    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError):
        window_attention(x, x, x, 2)
    with pytest.raises(RuntimeError):
        gated_recurrence(x[:, 0], x[:, 0], x[:, 0], torch.zeros(8))
