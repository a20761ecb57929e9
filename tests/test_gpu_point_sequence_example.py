"""The example on point sequences: its blocks without a window answer packets as their forward does."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_packets_over_an_8_bit_history(dev):
    spec = importlib.util.spec_from_file_location("point_sequence", Path(__file__).parents[1] / "examples" / "point_sequence.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(0)
    # values are off by at most half a step of 1 / 127 of their row's largest, weights by as much of the scores: the
    # attention's share of a row is a fraction of it, through two blocks
    assert example.packets(dev) < 2 / 127
