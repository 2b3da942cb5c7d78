"""The word that the books' launches count on: zero and in place before the first call, and
the handle's alone for good."""
import contextlib

import pytest
import torch

import flash_deepseek_amd as fdm


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on the first GPU."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", 0))

    def get_device(self):
        return 0


def on_gpu(*shape):
    return torch.Tensor._make_subclass(OnGpu, i32(*shape))


def test_no_handle_is_made_during_a_capture(monkeypatch):
    """Its word would be zero from the graph's first replay on only, and a call before it would count on anything."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    with pytest.raises(fdm.FdmError, match="captured"):
        fdm.KvPages(on_gpu(3, 8), on_gpu(3), on_gpu(40), on_gpu(1), 16)
    with pytest.raises(fdm.FdmError, match="captured"):
        fdm.kv_pages(3, 8, 40, 16)


@pytest.mark.gpu
def test_no_handle_is_made_inside_a_graph(fdm):
    tensors = [torch.zeros(*k, dtype=torch.int32, device="cuda") for k in ((3, 8), (3,), (40,), (1,))]
    x, stream, graph = torch.zeros(1, device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        x.add_(1)
        with pytest.raises(fdm.FdmError, match="captured"):
            fdm.KvPages(*tensors, 16)
        with pytest.raises(fdm.FdmError, match="captured"):
            fdm.kv_pages(3, 8, 40, 16)
    graph.replay()
    torch.cuda.synchronize()
    assert x.item() == 1 and fdm.kv_pages(3, 8, 40, 16).n_free.item() == 40
