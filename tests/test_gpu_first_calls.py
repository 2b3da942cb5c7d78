"""The first calls of a stream, which make its workspace: the words that the
one-launch kernels rely on are zero before the first of them starts, whatever
the null stream is busy with."""
import numpy as np
import pytest

from tests._helpers import empty_f32, say, to_dev, to_host

pytestmark = pytest.mark.gpu

L = 15
K = 8


@pytest.fixture(scope="module")
def layer(fdm):
    from flash_deepseek_amd.synthetic import make_layer
    say(f"building layer L={L}")
    lay = make_layer(3000 + L)
    fdm.attach_layer(L, lay.experts, lay.expert_size, lay.Wg, lay.bias, lay.shared)
    yield lay
    fdm.release_layer(L)


def test_first_calls_while_the_null_stream_is_busy(fdm, oracle, layer):
    """A clear that waited for the null stream's work would land among these calls and
    take their arrivals and tags away."""
    import torch
    h, h_in = (to_dev(oracle.synth_normal(7168, 0.0, 1.0, 43000 + i)) for i in range(2))
    want = empty_f32(7168)
    say(f"moe_layer L={L} on the null stream")
    fdm.moe_layer(L, h, h_in, K, want)
    want = to_host(want).view(np.uint32)
    a = torch.randn(4096, 4096, device="cuda")
    for turn in range(2):
        s = torch.cuda.Stream()
        fdm.stream_release(s)
        out = [empty_f32(7168) for _ in range(400)]
        torch.cuda.synchronize()
        say(f"400 calls of moe_layer on a stream without a workspace, the null stream multiplying ({turn})")
        for _ in range(20):
            torch.mm(a, a)
        with torch.cuda.stream(s):
            for o in out:
                fdm.moe_layer(L, h, h_in, K, o, stream=s.cuda_stream)
        fdm.sync(s.cuda_stream)
        for i, o in enumerate(out):
            assert np.array_equal(to_host(o).view(np.uint32), want), (turn, i)
        fdm.stream_release(s)
