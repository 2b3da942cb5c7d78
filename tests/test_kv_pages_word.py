"""The word that the books' launches count on: zero and in place before the first call, and
the handle's alone for good."""
import contextlib
import threading

import pytest
import torch

import flash_deepseek_amd as fdm
from tests.test_gpu_step import books, ints, rng


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


def test_a_word_is_handed_out_once(monkeypatch):
    """A queued launch, or a graph, counts on it when its handle is gone: not even another handle gets it."""
    monkeypatch.setattr(fdm, "_on_device", lambda *a: None)
    at = []

    def make(count):
        for _ in range(count):
            p = fdm.KvPages(i32(3, 8), i32(3), i32(40), i32(1), 16)
            assert p._turn.item() == 0 and p._turn.data_ptr() == p.desc.turn
            at.append(p.desc.turn)

    make(2100)
    threads = [threading.Thread(target=make, args=(200,)) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(at)) == len(at) == 3300
    held = [(w.data_ptr(), w.data_ptr() + 4 * w.numel()) for w in fdm._all_words if not w.is_cuda]
    assert all(any(lo <= a < hi for lo, hi in held) for a in at)


@pytest.mark.gpu
def test_a_graph_outlives_its_handle(fdm):
    """The caller keeps the tensors and the graph; the handle goes, and others use the memory that is free."""
    b = books(rng(9), 20, 400, 8100, 16, 3000)
    tensors = ints(b.pages), ints(b.kv_len), ints(b.free), ints([b.n_free])
    new, keep, N = [700] * 20, [500 + 100 * i for i in range(20)], 14003
    dn, dk = ints(new), ints(keep)
    q, pos, slots = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (21, N, N))
    p = fdm.KvPages(*tensors, 16)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        fdm.kv_trim(p, dk)
        fdm.kv_grow(p, dn, q, pos, slots)
    del p
    others = [torch.full((1,), 1000 + i, dtype=torch.int32, device="cuda") for i in range(3000)]
    for _ in range(3):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        b.trim(keep)
        want = b.grow(new, N)
        assert [q.tolist(), pos.tolist(), slots.tolist()] == list(want[:3])
    assert [t.tolist() for t in tensors] == [b.pages, b.kv_len, b.free, [b.n_free]]
    assert torch.equal(torch.cat(others).cpu(), torch.arange(1000, 4000, dtype=torch.int32))
