"""Attention of prompts with any number of query heads to a key head: whole groups, parts of them and single heads
to a workgroup, whose tiles of tokens are of any size."""

import pytest
import torch

from test_gpu_paged_attention import _check

pytestmark = pytest.mark.gpu
F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, BF16), (F16, I8), (BF16, E4)]
IDS = ["f32", "bf16", "f16-i8", "bf16-e4m3"]


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("group", [3, 5, 7, 12, 19, 20, 31, 67, 130, 160])
def test_groups(dev, dtype, stored, group):
    _check(dev, dtype, stored, [(0, 1), (70, 2), (0, 45), (13, 130), (0, 0), (250, 7)], group, 1, 32, 64, lead=3, tail=4)


@pytest.mark.parametrize("dtype,stored", [(F32, F32), (BF16, E4)], ids=["f32", "bf16-e4m3"])
@pytest.mark.parametrize("H,Hk,buckets,maxd", [(20, 1, 32, 128), (20, 1, 16, 400), (10, 2, 32, 64), (9, 3, 32, 1024), (40, 2, 32, 17), (4, 1, 32, 1024)])
def test_groups_with_a_bias(dev, dtype, stored, H, Hk, buckets, maxd):
    _check(dev, dtype, stored, [(0, 40), (300, 3), (5, 1), (1200, 9)], H, Hk, 16, 64, buckets=buckets, maxd=maxd)


@pytest.mark.parametrize("dtype,stored", TYPES, ids=IDS)
@pytest.mark.parametrize("H,Hk", [(6, 2), (20, 1), (16, 1)])
def test_groups_in_pieces(dev, dtype, stored, H, Hk):
    _check(dev, dtype, stored, [(2600, 3), (0, 5), (900, 1)], H, Hk, 64, 64, lead=1, tail=2)
