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


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("strong", [0, 5000, 32768])
def test_one_strong_position_among_many_weak_ones(fdm, fmt, strong):
    """Weights of 2^-25 of the row's largest, 32768 of them: 1e-3 of the values, all of
    those that the strong position has none of.  The tolerance is C.attend's, and
    for F16 weights half a step of its smallest numbers, 2^-25, where the row's
    largest weight is at least 2^7: 2^-32 a position.  512 sequences of one token
    share the pages, so that a workgroup walks each from end to end."""
    g = rng(6)
    page, L, H, B = 64, 32769, 4, 512
    t = C.DTYPES[fmt]
    rows = torch.rand(L, C.LAT, generator=g) + 0.5
    rows[:, 0] = 0.0
    rows[strong] = normal(g, C.LAT)
    rows[strong, 1:256] = 0.0
    rows[strong, 0] = 4.34375  # with q 4 and scale 1: 17.375, or 2^25.07
    cache = fdm.kv_cache(fmt, -(-L // page), page)
    cache.latent.flatten(0, 1)[:L].copy_(rows)
    q_lat, q_rope = torch.zeros(1, H, C.LAT, dtype=t), torch.zeros(1, H, C.ROT, dtype=t)
    q_lat[:, :, 0] = 4.0
    pages = torch.arange(cache.n_pages, dtype=torch.int32)[None]
    out, lse = torch.empty(B, H, C.LAT, dtype=t, device="cuda"), torch.empty(B, H, device="cuda")
    say(f"mla_attend {fmt}, the strong position at {strong} of {L}")
    fdm.mla_attend(cache, q_lat.expand(B, -1, -1).cuda(), q_rope.expand(B, -1, -1).cuda(), i32(*range(B + 1)), i32(*[L] * B),
                   pages.expand(B, -1).contiguous().cuda(), 1.0, out, lse=lse)
    torch.cuda.synchronize()
    assert torch.equal(out, out[:1].expand_as(out)) and torch.equal(lse, lse[:1].expand_as(lse))
    k = C.widened(cache.latent.cpu(), cache.rope.cpu())
    want, wlse, tol, ltol = C.attend(k, page, q_lat, q_rope, [0, 1], [L], pages, 1.0)
    tail = want[0, 0, 1:256].mean()
    assert 8e-4 < tail < 1.1e-3
    if fmt == "f16":
        tol = tol + 2.0 ** -32 * k[:L, :C.LAT].abs().sum(0)
    C.check(out[:1].cpu(), want, tol, "out")
    C.check(lse[:1].cpu(), wlse, ltol, "lse")


@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
@pytest.mark.parametrize("step", [0.3, 3.0])
def test_scores_that_grow_along_the_sequence(fdm, fmt, step):
    """Every 32 positions have a larger maximum than all before them, by `step` in
    log2 a position: the running maximum moves again and again in every row."""
    g = rng(7)
    page, L, H, n = 16, 700, 24, 5
    t = torch.float16 if fmt == "f16" else torch.bfloat16
    cache = fdm.kv_cache(fmt, -(-L // page), page)
    kv = normal(g, L, C.LAT + C.ROT)
    kv[:, C.LAT] = torch.arange(L) * step * math.log(2.0) / 2.0  # rotary parts keep 16 bits in every format
    fdm.kv_write(cache, kv.cuda(), torch.arange(L, dtype=torch.int32, device="cuda"))
    q_lat, q_rope = normal(g, n, H, C.LAT, std=0.02).to(t), torch.zeros(n, H, C.ROT, dtype=t)
    q_rope[:, :, 0] = 2.0
    pages = torch.arange(cache.n_pages, dtype=torch.int32)[None]
    out, lse = torch.empty(n, H, C.LAT, dtype=t, device="cuda"), torch.empty(n, H, device="cuda")
    say(f"mla_attend {fmt}, scores growing by 2^{step} a position")
    fdm.mla_attend(cache, q_lat.cuda(), q_rope.cuda(), i32(0, n), i32(L), pages.cuda(), 1.0, out, lse=lse)
    torch.cuda.synchronize()
    k = C.widened(cache.latent.cpu(), cache.rope.cpu(), None if cache.scale is None else cache.scale.cpu())
    score = k[:, C.LAT] * 2.0 / math.log(2.0)
    assert (score[32::32] - score[:-32:32][:score[32::32].numel()] > 8.0).all() or step < 1.0  # past what a weight may grow by
    want, wlse, tol, ltol = C.attend(k, page, q_lat, q_rope, [0, n], [L], pages, 1.0)
    C.check(out.cpu(), want, tol + (2.0 ** -32 * k[:L, :C.LAT].abs().sum(0) if fmt == "f16" else 0.0), "out")
    C.check(lse.cpu(), wlse, ltol, "lse")


@pytest.mark.parametrize("n,L,H", [(300, 70, 40), (260, 0, 16), (150, 149, 128), (40, 33, 7)])
def test_more_tokens_than_positions(fdm, n, L, H):
    """Tokens in order that stand before the first position see nothing, over several tiles."""
    g = rng(n)
    page = 8
    cache = fdm.kv_cache("bf16", 16 * 2, page)
    cache.latent.copy_(normal(g, *cache.latent.shape))
    cache.rope.copy_(normal(g, *cache.rope.shape))
    q_lat, q_rope = normal(g, n + 3, H, C.LAT, std=0.6).bfloat16(), normal(g, n + 3, H, C.ROT, std=0.6).bfloat16()
    pages = torch.randperm(32, generator=g)[:19 + 3].to(torch.int32)[None].expand(2, -1).contiguous()
    out, lse = torch.full((n + 3, H, C.LAT), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full((n + 3, H), 7.0, device="cuda")
    say(f"mla_attend of {n} tokens in order over {L} positions, {H} heads, beside three over 170")
    fdm.mla_attend(cache, q_lat.cuda(), q_rope.cuda(), i32(0, n, n + 3), i32(L, 170), pages.cuda(), SCALE, out, lse=lse)
    torch.cuda.synchronize()
    want, wlse, tol, ltol = C.attend(C.widened(cache.latent.cpu(), cache.rope.cpu()), page, q_lat, q_rope, [0, n, n + 3], [L, 170], pages, SCALE)
    assert (wlse[:n - L] == -math.inf).all() and (want[:n - L] == 0).all()
    C.check(out.cpu(), want, tol, "out")
    C.check(lse.cpu(), wlse, ltol, "lse")


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("grow,scale", [(1, 2.0794), (2, 2.0794), (1, 0.75), (5, 0.5123)])
def test_scores_of_2_to_25(fdm, fmt, grow, scale):
    """Scores whose fp32 neighbours are 4 apart (exact sums: 2^25 and multiples of 4): the
    reference of a row is rounded by up to 4 in log2, and no weight may pass the type's
    range for it.  With (1, 2.0794) a comparison of rounded maxima let one reach 2^20.
    Weights round by half a step of the type, exponents by 2^-18 with the exponential's own."""
    g = rng(8)
    page, L, H, B = 32, 128, 2, 512
    t, step = C.DTYPES[fmt], C.HALF_STEP[C.DTYPES[fmt]]
    scale = float(torch.tensor(scale, dtype=torch.float32))
    rows = normal(g, L, C.LAT)
    rows[:, 0], rows[:, 1] = 8192.0, 4.0 * grow * (torch.arange(L) // 32)
    cache = fdm.kv_cache(fmt, L // page, page)
    cache.latent.flatten(0, 1).copy_(rows)
    q_lat, q_rope = torch.zeros(B, H, C.LAT, dtype=t), torch.zeros(B, H, C.ROT, dtype=t)
    q_lat[:, :, 0], q_lat[:, :, 1] = 4096.0, 1.0
    pages = torch.arange(L // page, dtype=torch.int32)[None].expand(B, -1).contiguous()
    out = torch.empty(B, H, C.LAT, dtype=t, device="cuda")
    say(f"mla_attend {fmt}, scores of 2^25 growing by {4 * grow} times {scale}")
    fdm.mla_attend(cache, q_lat.cuda(), q_rope.cuda(), i32(*range(B + 1)), i32(*[L] * B), pages.cuda(), scale, out)
    torch.cuda.synchronize()
    k = cache.latent.cpu().flatten(0, 1).double()
    p = torch.softmax(k[:, 1] * scale, 0)  # the 2^25 is the same in all
    want = p @ k
    tol = p @ k.abs() * (step + 2.0 ** -18) + (2.0 ** -32 * k.abs().sum(0) if fmt == "f16" else 0.0) + want.abs() * step
    C.check(out.cpu(), want.expand(B, H, -1), tol, "out")


def test_two_threads_on_one_stream_share_a_workspace(fdm):
    """Calls on one stream run in its order, from whichever thread they come: a call's
    two launches follow each other."""
    import threading
    g = rng(9)
    page, H = 64, 128
    cache = fdm.kv_cache("bf16", 64, page)
    cache.latent.copy_(normal(g, *cache.latent.shape))
    cache.rope.copy_(normal(g, *cache.rope.shape))
    pages = torch.randperm(64, generator=g).to(torch.int32)[None].cuda()
    space = fdm.mla_workspace(4, H)
    sizes = [(1, 4000), (3, 2100)]  # one tile of many parts; three tiles
    args = []
    for n, L in sizes:
        q_lat, q_rope = normal(g, n, H, C.LAT, std=0.6).bfloat16().cuda(), normal(g, n, H, C.ROT, std=0.6).bfloat16().cuda()
        args.append((cache, q_lat, q_rope, i32(0, n), i32(L), pages, SCALE))
    want = [torch.empty_like(a[1]) for a in args]
    for a, o in zip(args, want):
        fdm.mla_attend(*a, o, workspace=space)
    torch.cuda.synchronize()
    say("two threads x 300 calls on the null stream, one workspace")
    got = [[torch.empty_like(w) for _ in range(300)] for w in want]
    errors = []

    def worker(i):
        try:
            for o in got[i]:
                fdm.mla_attend(*args[i], o, workspace=space, stream=0)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    torch.cuda.synchronize()
    assert not errors, errors
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)
