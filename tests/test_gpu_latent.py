"""Rotary positions, the paged latent cache and the attention of drafted tokens
over it, against their float64 forms (tests/latent_case.py), through the
package's entry points."""
import math

import numpy as np
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


# ---- rotary positions ------------------------------------------------------------------
@pytest.mark.parametrize("T,H,D,R,offset,layout,scaling,factor,tx,ty", [
    (1, 1, 64, 64, 0, "interleaved", "none", 1.0, "f32", "f32"),
    (5, 128, 192, 64, 128, "interleaved", "yarn", 40.0, "f32", "bf16"),
    (3, 7, 128, 128, 0, "half", "linear", 4.0, "bf16", "bf16"),
    (33, 2, 96, 48, 0, "half", "yarn", 8.0, "f16", "f32"),
    (17, 3, 101, 34, 13, "interleaved", "none", 1.0, "f32", "f16"),
    (9, 5, 77, 18, 59, "half", "linear", 2.0, "bf16", "f16"),
    (2, 1, 256, 256, 0, "half", "none", 1.0, "f16", "f16"),
    (700, 16, 64, 2, 8, "interleaved", "none", 1.0, "f32", "f32"),
    (4, 130, 40, 24, 16, "interleaved", "yarn", 2.0, "bf16", "f32"),
])
def test_rope_matches_definition(fdm, T, H, D, R, offset, layout, scaling, factor, tx, ty):
    g = rng(T * 1000 + D)
    x = normal(g, T, H, D).to(C.DTYPES[tx])
    pos = torch.randint(0, 1 << 20, (T,), generator=g, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1 if T > 1 else 0
    pos[-1] = -7 if T > 2 else pos[-1]
    table = fdm.rope_table(R, layout=layout, scaling=scaling, factor=factor, mul=1.25 if scaling == "yarn" else 1.0)
    out = torch.full((T, H, D), 9.0, dtype=C.DTYPES[ty], device="cuda")
    say(f"rope T={T} H={H} D={D} R={R} {layout} {scaling} {tx} -> {ty}")
    fdm.rope(table, x.cuda(), pos.cuda(), out, offset=offset)
    want = x.double()
    freq = C.frequencies(R, scaling=scaling, factor=factor)
    part, size = C.turned(want[..., offset:offset + R], pos, freq, layout, 1.25 if scaling == "yarn" else 1.0)
    tol = torch.zeros_like(want)
    # the reference's own frequency is a double: 2^-52 of itself, times the position
    tol[..., offset:offset + R] = size * (C.TURN_TOL + 2.0 ** 31 * 2.0 ** -51)
    want = want.clone()
    want[..., offset:offset + R] = part
    # half a step of the result, or of the smallest numbers of f16
    C.check(out.cpu(), want, tol + want.abs() * C.HALF_STEP[out.dtype] + (2.0 ** -25 if ty == "f16" else 0.0), "rope")


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("part", ["f32", "bf16"])
def test_rope_in_place_and_strided(fdm, layout, part):
    """In place: the same bits as out of place, the rest untouched.  Strided: a head's
    part out of a wider row, into a tensor of its own."""
    g = rng(5)
    x = normal(g, 6, 4, 200).to(C.DTYPES[part]).cuda()
    pos = torch.arange(6, dtype=torch.int32).cuda() * 1000
    table = fdm.rope_table(64, layout=layout)
    view = x[:, :, 8:184]  # [6, 4, 176], rotated at 40 .. 104 of it
    out = torch.empty(6, 4, 176, dtype=x.dtype, device="cuda")
    say("rope strided, then in place")
    fdm.rope(table, view, pos, out, offset=40)
    before = x.clone()
    fdm.rope(table, view, pos, view, offset=40)
    assert torch.equal(view, out)
    assert torch.equal(x[:, :, :48], before[:, :, :48]) and torch.equal(x[:, :, 112:], before[:, :, 112:])
    # heads and tokens swapped in memory, odd element offset: the element path
    y = torch.zeros(4, 6, 177, dtype=x.dtype, device="cuda")[:, :, 1:].transpose(0, 1)
    fdm.rope(table, before[:, :, 8:184], pos, y, offset=40)
    assert torch.equal(y, out)
    # one row for every token
    one = before[:1, :, 8:184].expand(6, 4, 176)
    fdm.rope(table, one, pos, out, offset=40)
    for t in range(6):
        single = torch.empty(1, 4, 176, dtype=x.dtype, device="cuda")
        fdm.rope(table, before[:1, :, 8:184], pos[t:t + 1], single, offset=40)
        assert torch.equal(single[0], out[t])


def test_rope_empty(fdm):
    table = fdm.rope_table(64)
    x = torch.empty(0, 4, 64, device="cuda")
    fdm.rope(table, x, torch.empty(0, dtype=torch.int32, device="cuda"), x)


# ---- the paged cache ---------------------------------------------------------------------
def planes(cache):
    return [p.cpu() for p in (cache.latent, cache.rope, cache.scale) if p is not None]


@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
@pytest.mark.parametrize("T,page,tx,stride", [(1, 1, "f32", 576), (7, 16, "bf16", 576), (130, 64, "f16", 584), (33, 4, "f32", 579)])
def test_write_and_read_back_exact(fdm, fmt, T, page, tx, stride):
    """Without norm and rotation every step is exact but the one rounding."""
    g = rng(T)
    n_pages = -(-T // page) + 2
    cache = fdm.kv_cache(fmt, n_pages, page)
    x = torch.zeros(T, stride).to(C.DTYPES[tx])
    x[:, :576] = (normal(g, T, 576) * torch.exp2(torch.randint(-12, 12, (T, 1), generator=g).float())).to(x.dtype)
    x[0, :128] = 0.0
    x[-1, 128] = 448.0  # a group's largest at the edge of its exponent
    x[-1, 129:256] = 1.0
    slots = torch.randperm(n_pages * page, generator=g)[:T].to(torch.int32)
    dead = T > 4
    if dead:
        slots[2], slots[3] = -1, n_pages * page  # padding, and past the cache
    say(f"kv_write {fmt} T={T} page={page} {tx}")
    xd = x.cuda()[:, :576]
    fdm.kv_write(cache, xd, slots.cuda())
    x = x[:, :576].float()
    live = [t for t in range(T) if not (dead and t in (2, 3))]
    at = slots[live].long()
    got = planes(cache)
    lat = got[0].reshape(-1, 512)
    untouched = torch.ones(n_pages * page, dtype=torch.bool)
    untouched[at] = False
    for p in got:
        assert not p.view(torch.uint8).reshape(n_pages * page, -1)[untouched].any()
    if fmt == "fp8":
        codes, e = C.quantised(x[live, :512])
        assert torch.equal(lat[at].view(torch.uint8) & 0x7F, codes.view(torch.uint8) & 0x7F)
        assert torch.equal(lat[at].float(), codes.float())
        assert torch.equal(got[2].view(torch.uint8).reshape(-1, 4)[at].int() - 127, e.int())
    else:
        assert torch.equal(lat[at], x[live, :512].to(lat.dtype))
    assert torch.equal(got[1].reshape(-1, 64)[at], x[live, 512:].to(got[1].dtype))
    rows = C.widened(*got)
    for ty, s in (("f32", 576), ("bf16", 576), ("f16", 600), ("f32", 577)):
        out = torch.full((T, s), 3.0, dtype=C.DTYPES[ty], device="cuda")
        fdm.kv_read(cache, slots.cuda(), out[:, :576])
        assert torch.equal(out[live, :576].cpu(), rows[at].to(out.dtype)), (ty, s)
        assert (out[:, 576:] == 3.0).all() and (not dead or (out[2:4] == 3.0).all())


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
def test_write_norms_and_turns(fdm, fmt, layout):
    T, page = 37, 16
    g = rng(3)
    x, w = normal(g, T, 576, std=2.0), 1.0 + normal(g, 512, std=0.2)
    pos = torch.randint(0, 1 << 18, (T,), generator=g, dtype=torch.int32)
    cache = fdm.kv_cache(fmt, 4, page)
    table = fdm.rope_table(64, scaling="yarn", factor=40.0, layout=layout)
    slots = torch.randperm(4 * page, generator=g)[:T].to(torch.int32)
    say(f"kv_write {fmt} normed and turned")
    fdm.kv_write(cache, x.cuda(), slots.cuda(), norm_w=w.cuda(), table=table, pos=pos.cuda())
    rows = C.widened(*planes(cache))[slots.long()]
    want = C.normed(x[:, :512].double(), w.double())
    # fp32: 8 + 6 sums of squares, the root, two products: 20 roundings at most
    tol = want.abs() * 20 * 2.0 ** -24
    if fmt == "fp8":
        # half a step: 2^-4 of the value, or 2^-10 of 2^e < max / 224 for the smallest
        big = want.unflatten(-1, (-1, 128)).abs().amax(-1, keepdim=True).expand(T, 4, 128).flatten(-2)
        tol = tol + torch.maximum(want.abs() * 2.0 ** -4, big / 224 * 2.0 ** -10) * (1 + 2.0 ** -19)
        half = torch.bfloat16
    else:
        half = C.DTYPES[fmt]
        tol = tol + want.abs() * C.HALF_STEP[half] + 2.0 ** -25
    C.check(rows[:, :512], want, tol, "latent")
    part, size = C.turned(x[:, None, 512:].double(), pos, C.frequencies(64, scaling="yarn", factor=40.0), layout)
    tol = size * (C.TURN_TOL + 2.0 ** 18 * 2.0 ** -51) + part.abs() * C.HALF_STEP[half] + 2.0 ** -25
    C.check(rows[:, None, 512:], part, tol, "rope")


def test_write_edges(fdm):
    """Infinities and NaN stay inside their group; the exponent's ends."""
    x = torch.ones(6, 576)
    x[0, 5] = math.inf
    x[1, 140] = math.nan
    x[2, :128] = 2.0 ** -140  # a subnormal of fp32
    x[3, :128] = torch.finfo(torch.float32).max
    x[4, :128] = 2.0 ** -105
    x[5, 300] = -math.inf
    cache = fdm.kv_cache("fp8", 1, 8)
    slots = torch.arange(6, dtype=torch.int32).cuda()
    out = torch.empty(6, 576, device="cuda")
    say("kv_write edges")
    fdm.kv_write(cache, x.cuda(), slots)
    fdm.kv_read(cache, slots, out)
    out, byte = out.cpu(), cache.scale.view(torch.uint8).cpu().reshape(8, 4)
    for row, group in ((0, 0), (1, 1), (5, 2)):
        nan = torch.zeros(576, dtype=torch.bool)
        nan[128 * group:128 * group + 128] = True
        assert torch.equal(out[row].isnan(), nan) and byte[row, group] == 255
        assert (out[row][~nan] == 1.0).all()
    assert (out[2, :128] == 0.0).all() and byte[2, 0] == 27  # 2^-100: below its smallest code
    assert (out[3, :128] == 448.0 * 2.0 ** 119).all() and byte[3, 0] == 246  # saturated
    assert (out[4, :128] == 2.0 ** -105).all() and byte[4, 0] == 27
    assert (out[2:5, 128:] == 1.0).all()


def test_cache_past_4_gib(fdm):
    """Rows whose bytes lie past 2^32."""
    page, n_pages = 64, 70000  # 4.48 M rows: 4.6 GB of latents
    latent = torch.empty(n_pages, page, 512, dtype=torch.bfloat16, device="cuda")
    rope = torch.empty(n_pages, page, 64, dtype=torch.bfloat16, device="cuda")
    cache = fdm.KvCache(latent, rope)
    g = rng(8)
    L, H = 70, 4
    pages = torch.tensor([[n_pages - 1, 3]], dtype=torch.int32)
    slots = torch.tensor([int(pages[0, j // page]) * page + j % page for j in range(L)], dtype=torch.int32)
    x = normal(g, L, 576).bfloat16()
    say("kv_write, kv_read, mla_attend past 4 GiB")
    fdm.kv_write(cache, x.cuda(), slots.cuda())
    out = torch.empty(L, 576, dtype=torch.bfloat16, device="cuda")
    fdm.kv_read(cache, slots.cuda(), out)
    assert torch.equal(out.cpu(), x)
    q = normal(g, 1, H, 576, std=0.6).bfloat16()
    o = torch.empty(1, H, 512, dtype=torch.bfloat16, device="cuda")
    fdm.mla_attend(cache, q[..., :512].contiguous().cuda(), q[..., 512:].contiguous().cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(),
                   torch.tensor([L], dtype=torch.int32).cuda(), pages.cuda(), SCALE, o)
    rows = torch.zeros(2 * page, 576, dtype=torch.float64)
    rows[:L] = x.double()
    want = C.attend(rows, page, q[..., :512], q[..., 512:], [0, 1], [L], [[0, 1]], SCALE)
    C.check(o.cpu(), want[0], want[2], "out")


# ---- attention -----------------------------------------------------------------------------
def filled(fdm, fmt, n_pages, page, g, std=1.0):
    """A cache of written rows, and its rows in float64."""
    cache = fdm.kv_cache(fmt, n_pages, page)
    x = normal(g, n_pages * page, 576, std=std)
    fdm.kv_write(cache, x.cuda(), torch.arange(n_pages * page, dtype=torch.int32).cuda())
    return cache, C.widened(*planes(cache))


def tree(g, counts, words=1, own_bit=True):
    """Random branches: each token sees some of the ones before it and itself."""
    rows = []
    for n in counts:
        for i in range(n):
            bits = [0] * words
            for d in range(min(i + 1, 64 * words)):
                if (d == i and own_bit) or (d < i and torch.rand(1, generator=g).item() < 0.4):
                    bits[d // 64] |= 1 << (d % 64)
            rows.append([b - (1 << 64) if b >> 63 else b for b in bits])
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, words)


def run_attend(fdm, cache, rows, page, q_lat, q_rope, q_start, kv_len, pages, mask=None, scale=SCALE, **kw):
    N, H, _ = q_lat.shape
    out = torch.full((N, H, 512), 7.0, dtype=q_lat.dtype, device="cuda")
    lse = torch.full((N, H), 7.0, device="cuda")
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    fdm.mla_attend(cache, q_lat.cuda(), q_rope.cuda(), i32(q_start), i32(kv_len), i32(pages), scale, out,
                   mask=None if mask is None else mask.cuda(), lse=lse, **kw)
    want, wlse, tol, ltol = C.attend(rows, page, q_lat, q_rope, q_start, kv_len, pages, scale, mask)
    inside = ~wlse.isnan().all(1)
    out, lse = out.cpu(), lse.cpu()
    C.check(out[inside], want[inside], tol[inside], "out")
    C.check(lse[inside], wlse[inside], ltol[inside], "lse")
    assert (out[~inside] == 7.0).all() and (lse[~inside] == 7.0).all()
    return out, lse


def queries(g, fmt, N, H, std=0.6):
    t = torch.float16 if fmt == "f16" else torch.bfloat16
    return normal(g, N, H, 512, std=std).to(t), normal(g, N, H, 64, std=std).to(t)


@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
@pytest.mark.parametrize("H,page,lens,counts,kind", [
    (128, 64, [1], [1], "order"),
    (128, 64, [31, 32, 33, 97], [1, 1, 1, 1], "order"),
    (16, 16, [200, 5, 64], [3, 1, 4], "tree"),
    (3, 1, [40, 7], [2, 5], "order"),
    (128, 32, [150, 129], [4, 7], "tree"),
    (40, 8, [70, 90, 300], [9, 3, 1], "order"),
    (1, 128, [500], [70], "order"),
    (64, 2, [65], [65], "tree2"),
    (33, 64, [260], [130], "order"),
])
def test_attend_matches_float64(fdm, fmt, H, page, lens, counts, kind):
    g = rng(H * 100 + len(lens))
    per = -(-max(lens) // page) + 1
    cache, rows = filled(fdm, fmt, len(lens) * per + 1, page, g)
    pages = torch.randperm(len(lens) * per + 1, generator=g)[:len(lens) * per].reshape(len(lens), per).tolist()
    start = [0] + np.cumsum(counts).tolist()
    mask = None if kind == "order" else tree(g, counts, 2 if kind == "tree2" else 1)
    say(f"mla_attend {fmt} H={H} page={page} lens={lens} counts={counts} {kind}")
    run_attend(fdm, cache, rows, page, *queries(g, fmt, start[-1], H), start, lens, pages, mask)


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_attend_long_and_split(fdm, fmt):
    """Few long sequences of uneven lengths, as the work is cut into parts that are put together again."""
    g = rng(17)
    page, lens, counts = 64, [3001, 40, 1500], [2, 1, 3]
    per = -(-max(lens) // page)
    cache, rows = filled(fdm, fmt, 3 * per, page, g)
    pages = torch.randperm(3 * per, generator=g).reshape(3, per).tolist()
    start = [0, 2, 3, 6]
    say(f"mla_attend {fmt} long")
    # scores that grow along the sequence: the running maximum moves again and again
    q = queries(g, fmt, 6, 24, std=0.6)
    run_attend(fdm, cache, rows, page, *q, start, lens, pages, tree(g, counts))
    q = queries(g, fmt, 6, 24, std=6.0)  # sharp: a few positions carry each row
    run_attend(fdm, cache, rows, page, *q, start, lens, pages)


@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
@pytest.mark.parametrize("H,B,L,most,kind", [(128, 24, 1500, 4, "tree"), (16, 400, 260, 3, "order"), (96, 5, 700, 70, "order"), (64, 512, 150, 1, "order")])
def test_attend_many_steps_a_workgroup(fdm, fmt, H, B, L, most, kind):
    """Enough work that every workgroup walks many steps of one tile, and several tiles; a
    sample of the sequences is checked."""
    g = rng(B)
    page = 32
    per = -(-L // page)
    cache, rows = filled(fdm, fmt, B * per, page, g)
    pages = torch.randperm(B * per, generator=g).reshape(B, per)
    counts = torch.randint(1, most + 1, (B,), generator=g).tolist()
    lens = torch.randint(L // 3, L + 1, (B,), generator=g).tolist()
    lens[B // 2], counts[B // 3] = L, most
    start = [0] + np.cumsum(counts).tolist()
    mask = None if kind == "order" else tree(g, counts)
    q = queries(g, fmt, start[-1], H)
    out = torch.full((start[-1], H, 512), 7.0, dtype=q[0].dtype, device="cuda")
    lse = torch.full((start[-1], H), 7.0, device="cuda")
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    say(f"mla_attend {fmt} H={H} B={B} L={L} up to {most} {kind}")
    fdm.mla_attend(cache, q[0].cuda(), q[1].cuda(), i32(start), i32(lens), pages.to(torch.int32).cuda(), SCALE, out,
                   mask=None if mask is None else mask.cuda(), lse=lse)
    out, lse = out.cpu(), lse.cpu()
    for b in sorted({0, 1, B // 3, B // 2, B - 1, *torch.randint(0, B, (6,), generator=g).tolist()}):
        t0, t1 = start[b], start[b + 1]
        want = C.attend(rows, page, q[0][t0:t1], q[1][t0:t1], [0, t1 - t0], [lens[b]], [pages[b].tolist()], SCALE,
                        None if mask is None else mask[t0:t1])
        C.check(out[t0:t1], want[0], want[2], f"out of {b}")
        C.check(lse[t0:t1], want[1], want[3], f"lse of {b}")


def test_attend_empty_rows_and_unseen_values(fdm):
    """A mask that leaves a row nothing, a sequence without positions, more tokens than
    positions, no tokens at all; NaN and infinity where no token looks, or only others do."""
    g = rng(23)
    page, H = 16, 32
    cache, rows = filled(fdm, "bf16", 8, page, g)
    pages = torch.arange(8).reshape(4, 2).tolist()
    lens, counts = [3, 0, 2, 20], [3, 1, 4, 0]
    start = [0, 3, 4, 8, 8]
    mask = torch.tensor([[0], [0b010], [0b101], [1], [0b1], [0], [0b1100], [0b1111]], dtype=torch.int64)
    q = queries(g, "bf16", 10, H)  # two rows behind the last sequence
    mask10 = torch.cat((mask, torch.zeros(2, 1, dtype=torch.int64)))
    say("mla_attend empty rows")
    out, lse = run_attend(fdm, cache, rows, page, *q, start, lens, pages, mask10)
    assert (lse[0] == -math.inf).all() and (out[0] == 0).all() and (lse[3] == -math.inf).all()
    run_attend(fdm, cache, rows, page, *q, start, lens, pages)  # in order: tokens before the first position
    # positions 1 and 2 of sequence 0: the one not finite, seen by token 1 alone, the other's seen by token 2
    bad = cache.latent.view(8 * page, 512)
    bad[1] = math.nan
    bad[2, 7] = math.inf
    bad[3:16] = math.nan  # behind the sequence, in its page
    cache.rope.view(8 * page, 64)[3:16] = -math.inf
    say("mla_attend values that are no numbers")
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    got = torch.empty(10, H, 512, dtype=torch.bfloat16, device="cuda")
    glse = torch.empty(10, H, device="cuda")
    fdm.mla_attend(cache, q[0].cuda(), q[1].cuda(), i32(start), i32(lens), i32(pages), SCALE, got, mask=mask10.cuda(), lse=glse)
    got, glse = got.cpu(), glse.cpu()
    assert (got[0] == 0).all() and (glse[0] == -math.inf).all()  # sees nothing
    assert got[1].isnan().all() and glse[1].isnan().all()  # sees the NaN
    assert torch.equal(got[4:8], out[4:8]) and torch.equal(glse[4:8], lse[4:8])
    # token 2 sees positions 0 and 2 (an infinity): no number, or the weights of an infinite score; never the NaN of 1
    mask10[2, 0] = 0b001
    fdm.mla_attend(cache, q[0].cuda(), q[1].cuda(), i32(start), i32(lens), i32(pages), SCALE, got := torch.empty_like(out).cuda(),
                   mask=mask10.cuda())
    assert torch.equal(got[2].cpu(), cache.latent.view(-1, 512)[0].cpu().expand(H, 512))  # sees position 0 alone


@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
@pytest.mark.parametrize("page", [1, 4, 8, 16, 32, 128])
def test_attend_among_rows_that_are_no_numbers(fdm, fmt, page):
    """Every row that belongs to no position of a sequence is NaN, the workspace full of ones."""
    g = rng(1000 + page)
    lens, counts = [1, 7, 33, 64, 95, 161], [1, 2, 1, 5, 3, 1]
    per = -(-max(lens) // page) + 1
    n_pages = len(lens) * per
    cache, _ = filled(fdm, fmt, n_pages, page, g)
    pages = torch.randperm(n_pages, generator=g).reshape(len(lens), per)
    used = torch.zeros(n_pages * page, dtype=torch.bool)
    for b, n in enumerate(lens):
        j = torch.arange(n)
        used[pages[b, j // page] * page + j % page] = True
    for plane, none in ((cache.latent, 0x7F if fmt == "fp8" else 0xFF), (cache.rope, 0xFF), (cache.scale, 0xFF)):
        if plane is not None:
            raw = plane.view(torch.uint8)
            raw.view(n_pages * page, -1)[~used.cuda()] = none
    rows = C.widened(*planes(cache))
    assert rows[~used].isnan().all() and rows[used].isfinite().all()
    workspace = fdm.mla_workspace(sum(counts), 16).fill_(0xFF)
    start = [0] + np.cumsum(counts).tolist()
    say(f"mla_attend {fmt} page={page} among NaN")
    run_attend(fdm, cache, rows, page, *queries(g, fmt, sum(counts), 16), start, lens, pages.tolist(), tree(g, counts), workspace=workspace)


def test_attend_as_many_sequences_as_a_call_takes(fdm):
    """512 of them: without tokens, without positions, and one that is longer than all others together."""
    g = rng(512)
    B, page = 512, 8
    counts = [i % 3 for i in range(B)]
    lens = [0 if i % 7 == 3 else max(counts[i], i % 11) for i in range(B)]
    counts[300], lens[300] = 2, 4000
    per = [max(1, -(-n // page)) for n in lens]
    cache, rows = filled(fdm, "bf16", sum(per), page, g)
    pages = torch.full((B, max(per)), -1, dtype=torch.int64)
    at = 0
    for b in range(B):
        pages[b, :per[b]] = torch.arange(at, at + per[b])
        at += per[b]
    start = [0] + np.cumsum(counts).tolist()
    say("mla_attend 512 sequences")
    run_attend(fdm, cache, rows, page, *queries(g, "bf16", start[-1], 5), start, lens, pages.tolist())


def test_attend_pages_outside_the_cache(fdm):
    """A page number that is none of the cache's: its positions are unseen, nothing is read."""
    g = rng(29)
    page = 16
    cache, rows = filled(fdm, "fp8", 6, page, g)
    pages = [[0, -1, 2], [6, 1, 2 ** 31 - 1], [-5, 77, 6]]
    say("mla_attend pages outside")
    out, lse = run_attend(fdm, cache, rows, page, *queries(g, "fp8", 4, 16), [0, 2, 3, 4], [48, 40, 37], pages)
    assert (lse[3] == -math.inf).all()


def test_attend_cuts_what_the_table_does_not_hold(fdm):
    """kv_len past the table or negative, q_start past N: cut."""
    g = rng(31)
    cache, rows = filled(fdm, "f16", 4, 16, g)
    pages = [[0, 1], [2, 3]]
    q = queries(g, "f16", 3, 8)
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    say("mla_attend cut lengths")
    got = [torch.full((3, 8, 512), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    lse = [torch.full((3, 8), 7.0, device="cuda") for _ in range(2)]
    for k, (start, lens) in enumerate([([-4, 2, 90], [1000, -3]), ([0, 2, 3], [32, 0])]):
        fdm.mla_attend(cache, q[0].cuda(), q[1].cuda(), i32(start), i32(lens), i32(pages), SCALE, got[k], lse=lse[k])
    assert torch.equal(got[0], got[1]) and torch.equal(lse[0], lse[1])


def test_attend_strides(fdm):
    """Queries out of wider rows, heads before tokens, an output with gaps: the same bits."""
    g = rng(37)
    page, H = 64, 24
    cache, rows = filled(fdm, "bf16", 4, page, g)
    q = queries(g, "bf16", 5, H)
    a = (torch.tensor([0, 2, 5], dtype=torch.int32).cuda(), torch.tensor([100, 77], dtype=torch.int32).cuda(),
         torch.tensor([[3, 1], [0, 2]], dtype=torch.int32).cuda())
    out = torch.empty(5, H, 512, dtype=torch.bfloat16, device="cuda")
    say("mla_attend strides")
    fdm.mla_attend(cache, q[0].cuda(), q[1].cuda(), *a, SCALE, out)
    wide = torch.cat((q[0], q[1]), -1).transpose(0, 1).contiguous().cuda().transpose(0, 1)  # [5, H, 576], heads outside
    gaps = torch.full((5, H, 640), 5.0, dtype=torch.bfloat16, device="cuda")
    fdm.mla_attend(cache, wide[..., :512], wide[..., 512:], *a, SCALE, gaps[..., 64:576])
    assert torch.equal(gaps[..., 64:576], out) and (gaps[..., :64] == 5.0).all() and (gaps[..., 576:] == 5.0).all()


def test_attend_streams_and_graph(fdm):
    """Two calls on two streams at once, each with its workspace, and a captured call
    replayed with other inputs between: the eager call's bits every time."""
    g = rng(41)
    page, H, lens = 64, 128, [700, 333]
    per = 11
    cache, rows = filled(fdm, "fp8", 2 * per, page, g)
    a = (torch.tensor([0, 2, 3], dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
         torch.arange(2 * per, dtype=torch.int32).reshape(2, per).cuda())
    q = [tuple(t.cuda() for t in queries(g, "fp8", 3, H)) for _ in range(3)]
    want = []
    for k in range(3):
        o = torch.empty(3, H, 512, dtype=torch.bfloat16, device="cuda")
        fdm.mla_attend(cache, *q[k], *a, SCALE, o)
        want.append(o)
    torch.cuda.synchronize()
    say("mla_attend on two streams")
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(want[0]) for _ in range(2)]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[k].zero_()
                fdm.mla_attend(cache, *q[k], *a, SCALE, outs[k])
    fdm.mla_attend(cache, *q[2], *a, SCALE, o := torch.empty_like(want[0]), stream=streams[0])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(o, want[2])
    say("mla_attend captured")
    ws = fdm.mla_workspace(3, H)
    held = [t.clone() for t in q[0]]
    out, row, back = torch.empty_like(want[0]), torch.randn(4, 576, device="cuda"), torch.empty(4, 576, device="cuda")
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    spare = fdm.kv_cache("fp8", 1, 4)
    table = fdm.rope_table(64)
    turned = torch.empty(3, H, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s, capture_error_mode="global"):
        fdm.mla_attend(cache, *held, *a, SCALE, out, workspace=ws)
        fdm.kv_write(spare, row, slots, table=table, pos=slots)
        fdm.kv_read(spare, slots, back)
        fdm.rope(table, held[1], pos, turned)
    eager = torch.empty_like(turned)
    for k in (0, 1, 2, 0):
        for h, t in zip(held, q[k]):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[k]), k
        fdm.rope(table, q[k][1], pos, eager)
        assert torch.equal(turned, eager)
        out.zero_()
        turned.zero_()


def test_attend_is_repeatable(fdm):
    g = rng(43)
    cache, rows = filled(fdm, "bf16", 40, 64, g)
    pages = torch.arange(40).reshape(1, 40).tolist()
    q = queries(g, "bf16", 1, 128)
    say("mla_attend repeated")
    first = run_attend(fdm, cache, rows, 64, *q, [0, 1], [2500], pages)
    again = run_attend(fdm, cache, rows, 64, *q, [0, 1], [2500], pages)
    assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("H,counts,extra", [(128, [37, 2], 70), (64, [81, 3], 31), (32, [150, 1], 5), (16, [300, 9], 33), (8, [200, 17], 64),
                                            (4, [333, 33], 1), (2, [400, 65], 40), (1, [300, 129], 0), (40, [90, 7], 50), (127, [25, 3], 64)])
def test_attend_prompts(fdm, H, counts, extra):
    """Many tokens in order, so that the tiles of one sequence differ in length and are found by their units, for heads that divide a tile and not."""
    g = rng(91 + H)
    page, lens = 32, [counts[0] + extra, counts[1] + 3 * extra]
    per = -(-max(lens) // page)
    cache, rows = filled(fdm, "bf16", 2 * per, page, g)
    pages = torch.randperm(2 * per, generator=g).reshape(2, per).tolist()
    say(f"mla_attend prompts H={H} {counts} {lens}")
    run_attend(fdm, cache, rows, page, *queries(g, "bf16", sum(counts), H), [0, counts[0], sum(counts)], lens, pages)


def test_refusals(fdm):
    """What the wrappers cannot take as it is, refused before a launch."""
    table = fdm.rope_table(64)
    cuda = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    i32 = dict(dtype=torch.int32)
    pos = cuda(2, **i32)
    cache = fdm.kv_cache("bf16", 2, 16)
    fp8 = fdm.kv_cache("fp8", 2, 16)
    q, r, o = cuda(2, 4, 512, dtype=torch.bfloat16), cuda(2, 4, 64, dtype=torch.bfloat16), cuda(2, 4, 512, dtype=torch.bfloat16)
    a = (cuda(2, **i32), cuda(1, **i32), cuda(1, 2, **i32))
    x = cuda(2, 4, 64)
    for call in (
        lambda: fdm.rope(table, x, pos, cuda(2, 4, 65)),
        lambda: fdm.rope(table, x[:, :, ::2], pos, x[:, :, ::2]),
        lambda: fdm.rope(table, x, pos.long(), x),
        lambda: fdm.rope(table, x, pos[:1], x),
        lambda: fdm.rope(table, x, pos, x, offset=1),
        lambda: fdm.rope(table, x.cpu(), pos, x),
        lambda: fdm.rope(table, x.double(), pos, x),
        lambda: fdm.rope(table, x, pos, x[:1].expand(2, 4, 64)),
        lambda: fdm.rope(table, cuda(2, 4, 63), pos, cuda(2, 4, 63)),
        lambda: fdm.kv_write(cache, cuda(2, 575), pos),
        lambda: fdm.kv_write(cache, cuda(2, 576), pos, table=table),
        lambda: fdm.kv_write(cache, cuda(2, 576), pos, table=fdm.rope_table(32), pos=pos),
        lambda: fdm.kv_write(cache, cuda(2, 576), pos, norm_w=cuda(511)),
        lambda: fdm.kv_read(cache, pos, cuda(3, 576)),
        lambda: fdm.kv_read(cache, pos, cuda(1, 576).expand(2, 576)),
        lambda: fdm.kv_cache("int4", 1),
        lambda: fdm.kv_cache("bf16", 4, 24),
        lambda: fdm.KvCache(cache.latent, fp8.rope[:1]),
        lambda: fdm.KvCache(cache.latent, cache.rope, fp8.scale),
        lambda: fdm.KvCache(fp8.latent, fp8.rope),
        lambda: fdm.mla_attend(cache, q.half(), r, *a, 1.0, o),
        lambda: fdm.mla_attend(cache, q, r, *a, 1.0, o.float()),
        lambda: fdm.mla_attend(cache, q, r[:1], *a, 1.0, o),
        lambda: fdm.mla_attend(cache, q, r, a[0][:1], a[1], a[2], 1.0, o),
        lambda: fdm.mla_attend(cache, q, r, *a, math.nan, o),
        lambda: fdm.mla_attend(cache, q, r, *a, 1.0, o, mask=cuda(1, 1, dtype=torch.int64)),
        lambda: fdm.mla_attend(cache, q, r, *a, 1.0, o, lse=cuda(2, 3)),
        lambda: fdm.mla_attend(cache, q, r, *a, 1.0, o, workspace=cuda(8, dtype=torch.uint8)),
        lambda: fdm.mla_attend(cache, q, r, *a, 1.0, o[:, :1].expand(2, 4, 512)),
        lambda: fdm.mla_attend(cache, cuda(2, 129, 512, dtype=torch.bfloat16), cuda(2, 129, 64, dtype=torch.bfloat16), *a, 1.0,
                               cuda(2, 129, 512, dtype=torch.bfloat16)),
    ):
        with pytest.raises(fdm.FdmError):
            call()


# ---- together --------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
def test_drafting_over_two_sequences(fdm, fmt):
    """A serving program's use: prompts written, a tree of drafted tokens written behind them
    and attended, the accepted branch moved to its places, the next token attended in order;
    against the attention of the exact rows, in float64."""
    g = rng(53)
    page, H, n_pages = 16, 8, 12
    table = fdm.rope_table(64, scaling="yarn", factor=40.0)
    cache = fdm.kv_cache(fmt, n_pages, page)
    pages = torch.randperm(n_pages, generator=g).reshape(2, 6).tolist()
    w = 1.0 + normal(g, 512, std=0.1)
    slot = lambda b, j: pages[b][j // page] * page + j % page  # noqa: E731
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    half = torch.float16 if fmt == "f16" else torch.bfloat16

    def put(x, slots, pos):
        fdm.kv_write(cache, x.cuda(), i32(slots), norm_w=w.cuda(), table=table, pos=i32(pos))

    def ask(pos):
        """Queries of tokens at pos: the rotary part turned out of the heads' fp32 rows."""
        heads = normal(g, len(pos), H, 192, std=0.6).cuda()
        q_rope = torch.empty(len(pos), H, 64, dtype=half, device="cuda")
        fdm.rope(table, heads[:, :, 128:], i32(pos), q_rope)
        part, size = C.turned(heads[:, :, 128:].cpu().double(), torch.tensor(pos), C.frequencies(64, scaling="yarn", factor=40.0), "interleaved")
        C.check(q_rope.cpu(), part, size * C.TURN_TOL + part.abs() * C.HALF_STEP[half] + 2.0 ** -25, "q_rope")
        return normal(g, len(pos), H, 512, std=0.6).to(half), q_rope.cpu()

    lens = [37, 52]
    for b, L in enumerate(lens):
        put(normal(g, L, 576), [slot(b, j) for j in range(L)], list(range(L)))
    # four drafted tokens each: 0 - 1 - 3 and 0 - 2; a token's position is its depth
    branch = [0b0001, 0b0011, 0b0101, 0b1011]
    depth = [0, 1, 1, 2]
    put(normal(g, 8, 576), [slot(b, lens[b] + i) for b in range(2) for i in range(4)], [lens[b] + d for b in range(2) for d in depth])
    q = ask([lens[b] + d for b in range(2) for d in depth])
    say(f"drafting {fmt}")
    run_attend(fdm, cache, C.widened(*planes(cache)), page, *q, [0, 4, 8], [L + 4 for L in lens], pages,
               torch.tensor(branch * 2, dtype=torch.int64)[:, None])
    # the branch 0 - 2 of the first is accepted: row 2 moves to place 1 (quantised rows move exactly)
    moved = torch.empty(1, 576, device="cuda")
    fdm.kv_read(cache, i32([slot(0, lens[0] + 2)]), moved)
    fdm.kv_write(cache, moved, i32([slot(0, lens[0] + 1)]))
    rows = C.widened(*planes(cache))
    assert torch.equal(rows[slot(0, lens[0] + 1)], rows[slot(0, lens[0] + 2)])
    lens = [lens[0] + 2, lens[1] + 1]
    put(normal(g, 2, 576), [slot(b, lens[b]) for b in range(2)], lens)
    q = ask(lens)
    run_attend(fdm, cache, C.widened(*planes(cache)), page, *q, [0, 1, 2], [L + 1 for L in lens], pages)


def test_agrees_with_the_single_sequence_layer(fdm, oracle):
    """The same tokens through fdm_attn_forward's parts in float64 and through these operators:
    the rotation of both uses the layer's YaRN frequencies."""
    freq = np.asarray(oracle.yarn_freq(), dtype=np.float64)
    mine = C.frequencies(64, scaling="yarn", factor=40.0).numpy()
    # the reference computes them in float: a handful of roundings
    assert np.max(np.abs(freq / mine - 1.0)) < 8 * 2.0 ** -23
