"""A step of BeamSearch leaves new scores and tokens each time: a graph that holds one would
start from the same ones at every replay, so a capture is refused."""
import pytest
import torch

from _util import pkg


def test_a_step_in_a_capture_is_refused(monkeypatch):
    search = object.__new__(pkg("integration.beam").BeamSearch)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        search.step(torch.zeros((2, 4)))


@pytest.mark.gpu
def test_a_search_goes_on_after_a_refused_capture():
    ops, tab = pkg("native.torch_ops"), pkg("integration.block_table")
    tables = tab.DeviceBlockTables(8, 32, 2, 4, 64, "cuda")
    cache = ops.q4_kv_cache(8, 32, 1, 64, "cuda")
    search = pkg("integration.beam").BeamSearch(tables, ops.PageSet(cache.planes()), 2)
    tables.step(torch.tensor([40, 0], dtype=torch.int32, device="cuda"))
    logits = torch.zeros((2, 50), device="cuda")
    logits[0, 3], logits[0, 4] = 5.0, 4.0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            search.step(logits)
        logits.mul_(1.0)
    assert search.step(logits).tolist() == [3, 4]
    assert search.sequences().tolist() == [[[3], [4]]]
