"""GPU tests of calls at the edges of what paged caches take."""

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, I8), (F16, E4)], ids=["f32", "bf16-i8", "f16-e4m3"])
def test_no_streams(dev, dtype, stored):
    """A serving loop whose last stream has ended: an empty result, and the pool as it was."""
    from gdl_amd.functional import PagedCache, paged_attention, paged_attention_step
    cache = PagedCache.empty(2, 2, 32, dtype=stored, device=dev)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            t.view(torch.uint8).fill_(7)
    want = ref.copy(cache)
    q, k = torch.empty(0, 4, 32, dtype=dtype, device=dev), torch.empty(0, 2, 32, dtype=dtype, device=dev)
    at = torch.empty(0, dtype=torch.int64, device=dev)
    for columns in (1, 5000):
        table = torch.empty(0, columns, dtype=torch.int32, device=dev)
        bias = torch.zeros(8, 4, dtype=dtype, device=dev)
        assert paged_attention_step(q, k, k, cache, table, at).shape == (0, 4, 32)
        assert paged_attention_step(q, k, k, cache, table, at, bias=bias, max_distance=20).shape == (0, 4, 32)
    table, ptr = torch.zeros(2, 3, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    cache.write(k, k, table, ptr)
    assert paged_attention(q, cache, table, ptr).shape == (0, 4, 32)
    assert all(x.shape == (0, 2, 32) for x in cache.read(table, ptr, 0, dtype=dtype))
    ref.same(cache, want)
