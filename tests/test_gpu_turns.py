"""One-launch kernels of several streams: calls that are all under way give the bits
of the same calls made alone, and a capture is refused."""
import numpy as np
import pytest

from tests._helpers import empty_f32, say, to_dev, to_host

pytestmark = pytest.mark.gpu

L = 16
K = 8


@pytest.fixture(scope="module")
def layer(fdm):
    from flash_deepseek_amd.synthetic import make_layer
    say(f"building layer L={L}")
    lay = make_layer(3000 + L)
    fdm.attach_layer(L, lay.experts, lay.expert_size, lay.Wg, lay.bias, lay.shared)
    yield lay
    fdm.release_layer(L)


@pytest.fixture(scope="module")
def data(oracle):
    import torch
    x = [to_dev(oracle.synth_normal(7168, 0.0, 1.0, 44000 + i)) for i in range(3)]
    # random blocks of 256 weights whose two fp16 scales (Q4_K) are small normal numbers
    g = torch.Generator().manual_seed(5)
    blob = torch.randint(0, 256, (3 * 8257536 // 144, 144), dtype=torch.uint8, generator=g)
    blob[:, 1] &= 0x03
    blob[:, 3] &= 0x03
    return x, blob.reshape(-1).cuda()


def calls(fdm, data, s):
    """The layer, an expert and a matvec by column parts on stream s."""
    x, blob = data
    out = [empty_f32(7168), empty_f32(7168), empty_f32(4096)]
    fdm.moe_layer(L, x[0], x[1], K, out[0], stream=s)
    fdm.expert_ffn(blob, 24772608, x[2], out[1], stream=s)
    fdm.matvec_q4k(blob, x[1], out[2], 4096, 5 * 1024, stream=s)
    return out


def test_streams_in_turn(fdm, layer, data):
    import torch
    say("reference calls on the null stream")
    want = [to_host(o).view(np.uint32) for o in calls(fdm, data, 0)]
    assert all(np.isfinite(w.view(np.float32)).all() and w.any() for w in want)
    streams = [0] + [torch.cuda.Stream().cuda_stream for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for r in range(25):
        for s in streams:
            got.append(calls(fdm, data, s))
    say("100 rounds of three kernels over four streams are queued")
    for s in streams:
        fdm.sync(s)
    for r, out in enumerate(got):
        for name, o, w in zip(("layer", "expert", "matvec"), out, want):
            assert np.array_equal(to_host(o).view(np.uint32), w), (r, name)
    say("one stream is released, another goes on")
    fdm.stream_release(streams[-1])
    for s in (streams[1], 0, streams[-1]):
        for o, w in zip(calls(fdm, data, s), want):
            assert np.array_equal(to_host(o).view(np.uint32), w)
    for s in streams[1:]:
        fdm.stream_release(s)


def test_a_capture_is_refused(fdm, layer, data):
    import torch
    x, blob = data
    s = torch.cuda.Stream()
    out = empty_f32(7168)
    with torch.cuda.stream(s):
        fdm.moe_layer(L, x[0], x[1], K, out)
    fdm.sync(s.cuda_stream)
    want = out.clone()
    other = torch.zeros(16, device="cuda")
    g = torch.cuda.CUDAGraph()
    say("capture")
    with torch.cuda.graph(g, stream=s):
        other += 1.0
        for call in (lambda: fdm.moe_layer(L, x[0], x[1], K, out), lambda: fdm.expert_ffn(blob, 24772608, x[2], out),
                     lambda: fdm.matvec_q4k(blob, x[1], out, 4096, 5 * 1024)):
            with pytest.raises(fdm.FdmError, match="captured"):
                call()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(other, torch.ones_like(other)) and torch.equal(out, want)
    with torch.cuda.stream(s):
        fdm.moe_layer(L, x[0], x[1], K, out)
    fdm.sync(s.cuda_stream)
    assert torch.equal(out, want)
    fdm.stream_release(s)
