"""Tests of a bias configuration's first call inside a graph capture: refused with the reason, since its
table is copied to the device, and captured after a call outside."""

import pytest
import torch

from gdl_amd.functional import relative_bias


def test_the_first_call_of_a_configuration_is_refused_in_a_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        relative_bias.bucket_plan(14, 77, True, torch.device("cuda", 0))
    lut, spans = relative_bias.bucket_plan(14, 77, True, torch.device("cpu"))
    assert lut.shape == (155,) and spans.shape == (14, 2)


@pytest.mark.gpu
def test_captured_after_a_call(dev):
    from gdl_amd.functional import window_attention
    q, k, v = (torch.randn(200, 2, 32, device=dev) for _ in range(3))
    table = torch.randn(12, 2, device=dev)

    def call():
        return window_attention(q, k, v, 20, bias=table, max_distance=79)

    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    torch.cuda.synchronize()
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
