"""The latent attention where its numbers or its work are extreme, against
float64 (tests/latent_case.py) and against itself."""
import math

import pytest
import torch

from tests import latent_case as C
from tests._helpers import say

pytestmark = pytest.mark.gpu
SCALE = (0.1 * math.log(40.0) + 1.0) ** 2 / math.sqrt(192.0)


def rng(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g) * std


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_tables_of_2_to_31_positions(fdm):
    """Tables that could hold more than 2^31 units of work are counted in 64 bits, with the same bits as the narrow count."""
    g = rng(5)
    page, B, H = 1 << 20, 40, 16
    cache = fdm.kv_cache("bf16", 1, page)
    cache.latent[0, :4096].copy_(normal(g, 4096, C.LAT))
    cache.rope[0, :4096].copy_(normal(g, 4096, C.ROT))
    n = torch.tensor([b % 4 for b in range(B)])
    n[7] = 600  # tokens in order over several tiles
    start = torch.zeros(B + 1, dtype=torch.int32)
    start[1:] = n.cumsum(0)
    N = int(start[-1])
    length = torch.tensor([700 + 83 * b for b in range(B)], dtype=torch.int32).clamp(max=4096)
    q_lat, q_rope = normal(g, N, H, C.LAT, std=0.6).bfloat16().cuda(), normal(g, N, H, C.ROT, std=0.6).bfloat16().cuda()
    pages = torch.zeros(B, 2048, dtype=torch.int32, device="cuda")
    for mask in (None, torch.randint(-2 ** 63, 2 ** 63 - 1, (N, 10), generator=g).cuda()):
        got = []
        for p in (pages, pages[:, :1].contiguous()):
            out = torch.full((N, H, C.LAT), 7.0, dtype=torch.bfloat16, device="cuda")
            lse = torch.full((N, H), 7.0, device="cuda")
            say(f"mla_attend of {B} sequences, tables of {p.shape[1]} pages of {page} rows, mask {mask is not None}")
            fdm.mla_attend(cache, q_lat, q_rope, start.cuda(), length.cuda(), p, SCALE, out, mask=mask, lse=lse)
            torch.cuda.synchronize()
            got.append((out.cpu(), lse.cpu()))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
        b = 5
        at, k = slice(int(start[b]), int(start[b + 1])), C.widened(cache.latent[:, :4096].cpu(), cache.rope[:, :4096].cpu())
        want = C.attend(k, 4096, q_lat.cpu()[at], q_rope.cpu()[at], torch.tensor([0, int(n[b])]), [int(length[b])], torch.zeros(1, 1, dtype=torch.int32),
                        SCALE, None if mask is None else mask.cpu()[at])
        C.check(got[0][0][at], want[0], want[2], "out")
        C.check(got[0][1][at], want[1], want[3], "lse")
