"""The cache's books, the residual's norm and projections with adapters against
their plain forms (tests/step_case.py), through the package's entry points."""
import math

import pytest
import torch

from tests import step_case as C
from tests._helpers import say

pytestmark = pytest.mark.gpu


def rng(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g) * std


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- the cache's books -------------------------------------------------------------------
def books(g, B, P, n_pages, page, longest):
    """Sequences of 0 .. longest positions on scattered pages, the rest free."""
    lens = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    order = torch.randperm(n_pages, generator=g).tolist()
    pages = []
    for n in lens:
        used = -(-n // page)
        pages.append([order.pop() for _ in range(used)] + [-7] * (P - used))
    return C.Books(pages, lens, order + [-9] * (n_pages - len(order)), len(order), page)


def on_gpu(fdm, b):
    return fdm.KvPages(ints(b.pages), ints(b.kv_len), ints(b.free), ints([b.n_free]), b.page)


def same(p, b):
    assert p.n_free.item() == b.n_free
    assert p.kv_len.tolist() == b.kv_len
    assert p.pages.tolist() == b.pages
    assert p.free.tolist() == b.free  # what lies above the stack's top too
    assert p._turn.item() == 0


def grow(fdm, p, b, new, N, seen=True):
    q, pos, slots, refused = (torch.full((k,), 77, dtype=torch.int32, device="cuda") for k in (b_len(b) + 1, N, N, 1))
    fdm.kv_grow(p, ints(new), q, pos, slots, refused=refused if seen else None)
    want = b.grow(new, N)
    assert q.tolist() == want[0]
    assert pos.tolist() == want[1]
    assert slots.tolist() == want[2]
    assert refused.item() == (want[3] if seen else 77)
    same(p, b)
    return want


def b_len(b):
    return len(b.kv_len)


@pytest.mark.parametrize("B,P,page,longest,most", [(1, 1, 1, 1, 1), (1, 40, 16, 300, 200), (3, 9, 64, 500, 4), (64, 8, 4, 20, 9), (300, 12, 16, 100, 60),
                                                   (1025, 6, 8, 30, 12), (4096, 5, 2, 6, 3), (7, 700, 1, 400, 250), (2, 3, 4096, 9000, 3000)])
def test_books_step_by_step(fdm, B, P, page, longest, most):
    """Steps of growth (from no token to many) and rollback."""
    g = rng(B * 7 + page)
    b = books(g, B, P, B * P + 5, page, min(longest, P * page))
    p = on_gpu(fdm, b)
    for step in range(4):
        new = torch.randint(-1 if step == 2 else 0, most + 1, (B,), generator=g).tolist()
        say(f"grow B={B} P={P} page={page} step {step}")
        N = sum(max(n, 0) for n in new) + step  # padded but for the first
        grow(fdm, p, b, new, N, seen=step != 1)
        keep = [int(torch.randint(-1, max(n, 0) + 3, (1,), generator=g)) if i % 5 else 0 for i, n in enumerate(b.kv_len)]
        fdm.kv_trim(p, ints(keep))
        b.trim(keep)
        same(p, b)


def test_a_growth_taken_back_leaves_the_stack(fdm):
    g = rng(3)
    b = books(g, 33, 20, 700, 16, 200)
    p = on_gpu(fdm, b)
    before = p.free.clone(), p.n_free.clone(), p.kv_len.clone()
    new = torch.randint(0, 100, (33,), generator=g).tolist()
    grow(fdm, p, b, new, 5000)
    fdm.kv_trim(p, before[2])
    assert all(torch.equal(x, y) for x, y in zip(before, (p.free, p.n_free, p.kv_len)))


def test_many_places_in_several_workgroups(fdm):
    """More places than a workgroup gives, more pages given back than one takes."""
    g = rng(4)
    b = books(g, 50, 700, 35100, 8, 3000)
    p = on_gpu(fdm, b)
    new = torch.randint(0, 2500, (50,), generator=g).tolist()
    for shift in (0, 1):  # 16-byte aligned, and not
        N = sum(new) + 1027
        q = torch.zeros(51, dtype=torch.int32, device="cuda")
        whole = torch.full((2, N + 4), 5, dtype=torch.int32, device="cuda")
        pos, slots = whole[0, shift:shift + N], whole[1, shift:shift + N]
        fdm.kv_grow(p, ints(new), q, pos, slots)
        want = b.grow(new, N)
        assert [q.tolist(), pos.tolist(), slots.tolist()] == list(want[:3])
        assert (whole[:, :shift] == 5).all() and (whole[:, shift + N:] == 5).all()
        same(p, b)
        keep = [n // 3 for n in b.kv_len]
        fdm.kv_trim(p, ints(keep))
        b.trim(keep)
        same(p, b)
        new = [100] * 50


def test_sequences_that_are_not_served(fdm):
    """Rows without room, too few free pages, too few places; no sequence takes what one before it lacked."""
    make = lambda: C.Books([[0, 1, -7], [2, -7, -7], [3, 4, 5], [6, -7, -7], [-7, -7, -7]], [7, 3, 12, 1, 0], [9, 8, 7, -9, -9, -9, -9, -9, -9, -9], 3, 4)
    for new, N in (([1, 9, 0, 3, 4], 50), ([5, 1, 1, 3, 1], 50), ([6, 1, 0, 3, 1], 50), ([1, 1, 0, 1, 4], 2), ([1, 1, 0, 1, 4], 3), ([9, 9, 9, 9, 9], 50),
                   ([2 ** 31 - 1] * 5, 50), ([-5, 1, -2 ** 31, 0, 13], 50), ([5, 5, 0, 3, 0], 13), ([0] * 5, 0), ([1] * 5, 0)):
        b = make()
        grow(fdm, on_gpu(fdm, b), b, new, N)


def test_numbers_that_are_none(fdm):
    """Lengths, free counts and pages outside their range are cut or leave slots empty; nothing is read or written elsewhere."""
    b = C.Books([[0, 99, -7], [-3, 1, 2], [3, -7, -7]], [6, 40, -4], [5, 4, 1000, -1, 0, 0], 4, 4)
    p = on_gpu(fdm, b)
    grow(fdm, p, b, [2, 0, 9], 20)
    b = C.Books([[0, 99, -7], [-3, 1, 2], [3, -7, -7]], [6, 40, -4], [5, 4, 1000, -1, 0, 0], 77, 4)
    p = on_gpu(fdm, b)
    grow(fdm, p, b, [2, 0, 9], 20)
    fdm.kv_trim(p, ints([0, 0, 0]))
    b.trim([0, 0, 0])
    same(p, b)


def test_books_in_a_graph_and_on_a_stream(fdm):
    """A captured step replayed: each replay is the next step."""
    g = rng(6)
    b = books(g, 9, 30, 300, 16, 100)
    p = on_gpu(fdm, b)
    new, keep = [3] * 9, [-1, 5] + [-1] * 7
    dn, dk = ints(new), ints(keep)
    q, pos, slots = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (10, 30, 30))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        fdm.kv_trim(p, dk)
        fdm.kv_grow(p, dn, q, pos, slots)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        b.trim(keep)
        want = b.grow(new, 30)
        assert [q.tolist(), pos.tolist(), slots.tolist()] == list(want[:3])
        same(p, b)
    with torch.cuda.stream(stream):
        fdm.kv_trim(p, dk)
    fdm.kv_grow(p, dn, q, pos, slots, stream=stream)
    torch.cuda.synchronize()
    b.trim(keep)
    assert list(b.grow(new, 30)[:3]) == [q.tolist(), pos.tolist(), slots.tolist()]
    same(p, b)


# ---- the residual's norm -----------------------------------------------------------------
@pytest.mark.parametrize("T,d,tx,ta,ty,w", [
    (1, 1, "f32", "f32", "f32", True), (3, 7, "bf16", "f16", "f16", True), (5, 128, "f32", None, "fp8", True), (2, 130, "f16", "f16", "fp8", False),
    (16, 7168, "f32", "f32", "fp8", True), (9, 7168, "bf16", "bf16", "fp8", True), (4, 7168, "f32", "bf16", "bf16", True), (33, 1536, "bf16", None, "bf16", True),
    (7, 512, "f16", "bf16", "f32", True), (2, 2048, "f16", "f32", "f16", False), (3, 2056, "bf16", "bf16", "f32", True), (2, 4104, "f32", "f32", "f16", True),
    (2, 16384, "bf16", "bf16", "fp8", True), (1, 16392, "f32", "bf16", "fp8", True), (2, 32768, "f32", "f32", "bf16", True), (3, 32767, "bf16", "f16", "fp8", True),
    (2, 1001, "f32", "f32", "fp8", True), (70, 64, "f32", "f32", "fp8", True)])
def test_norm_matches_definition(fdm, T, d, tx, ta, ty, w):
    g = rng(T * d)
    x = (normal(g, T, d) * torch.exp2(torch.randint(-8, 8, (T, 1), generator=g).float())).to(C.DTYPES[tx])
    add = None if ta is None else normal(g, T, d).to(C.DTYPES[ta])
    wt = 1.0 + 0.2 * normal(g, d) if w else None
    fp8 = ty == "fp8"
    out = torch.full((T, d), 3.0, device="cuda").to(torch.float8_e4m3fn if fp8 else C.DTYPES[ty])
    scale = torch.full((T, -(-d // 128)), 9, dtype=torch.uint8, device="cuda") if fp8 else None
    total = torch.empty(T, d, dtype=x.dtype, device="cuda")
    on = [None if t is None else t.cuda() for t in (x, add, wt)]
    say(f"add_rms_norm T={T} d={d} {tx}+{ta}->{ty}")
    fdm.add_rms_norm(on[0], on[1], on[2], out, scale=scale, sum=total, eps=1e-5)
    s, y = C.normed(x, add, wt, 1e-5)
    C.check(total.cpu(), s, s.abs() * (C.HALF_STEP[x.dtype] + 2.0 ** -24) + (2.0 ** -25 if tx == "f16" else 0.0), "sum")
    if fp8:
        C.check_codes(out.cpu(), scale.cpu(), y, C.NORM_TOL)
    else:
        C.check(out.cpu(), y, y.abs() * (C.NORM_TOL + C.HALF_STEP[out.dtype]) + (2.0 ** -25 if ty == "f16" else 0.0), "y")
    # without a sum to keep, and in the residual's own place: the same bits
    again = torch.zeros_like(out.view(torch.uint8)).view(out.dtype)
    fdm.add_rms_norm(on[0], on[1], on[2], again, scale=scale, eps=1e-5)
    assert torch.equal(again.view(torch.uint8), out.view(torch.uint8))
    fdm.add_rms_norm(on[0], on[1], on[2], again, scale=scale, sum=on[0], eps=1e-5)
    assert torch.equal(again.view(torch.uint8), out.view(torch.uint8)) and torch.equal(on[0], total)


@pytest.mark.parametrize("ty", ["bf16", "fp8"])
def test_norm_of_strided_rows(fdm, ty):
    """Rows inside wider ones, aligned and not; what lies beside them stays."""
    g = rng(8)
    T, d = 5, 1536
    x, add, w = normal(g, T, d).cuda(), normal(g, T, d).bfloat16().cuda(), (1 + normal(g, d) * 0.1).cuda()
    t = torch.float8_e4m3fn if ty == "fp8" else torch.bfloat16
    want, ws = torch.empty(T, d, device="cuda").to(t), torch.empty(T, 12, dtype=torch.uint8, device="cuda")
    fdm.add_rms_norm(x, add, w, want, scale=ws if ty == "fp8" else None)
    for off in (0, 8, 3):
        wide = [torch.full((T, d + 24), 2.0, device="cuda").to(k) for k in (x.dtype, add.dtype, t)]
        scales = torch.full((T, 16), 7, dtype=torch.uint8, device="cuda")
        at = [v[:, off:off + d] for v in wide]
        at[0].copy_(x)
        at[1].copy_(add)
        fdm.add_rms_norm(at[0], at[1], w, at[2], scale=scales[:, 1:13] if ty == "fp8" else None, sum=at[0])
        assert torch.equal(at[2].contiguous().view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(at[0], x + add.float())
        for v in wide:
            assert (v[:, :off].float() == 2).all() and (v[:, off + d:].float() == 2).all()
        if ty == "fp8":
            assert torch.equal(scales[:, 1:13], ws) and (scales[:, :1] == 7).all() and (scales[:, 13:] == 7).all()
    # one row for every token, tokens last to first
    one = x[:1].expand(T, d)
    out = torch.empty(T, d, device="cuda").to(t)
    sc = torch.empty(T, 12, dtype=torch.uint8, device="cuda")
    fdm.add_rms_norm(one, None, w, out, scale=sc if ty == "fp8" else None)
    assert all(torch.equal(out[i].view(torch.uint8), out[0].view(torch.uint8)) for i in range(T))
    y = torch.empty_like(x)
    fdm.add_rms_norm(x, None, w, y)
    in_place = x.clone()
    fdm.add_rms_norm(in_place, None, w, in_place)
    assert torch.equal(in_place, y)


def test_norm_of_zeros_and_of_no_numbers(fdm):
    """Zeros give zeros (scale byte 27); a row with an infinity or NaN has NaN there and leaves the others alone."""
    x = torch.ones(4, 300, device="cuda")
    x[1] = 0.0
    x[2, 150] = math.inf
    x[3, 10] = math.nan
    out, scale = torch.empty(4, 300, device="cuda").to(torch.float8_e4m3fn), torch.empty(4, 3, dtype=torch.uint8, device="cuda")
    fdm.add_rms_norm(x, None, None, out, scale=scale)
    got = out.float().cpu()
    assert (scale[1] == 27).all() and (got[1] == 0).all()
    assert scale[2].tolist()[1] == 255 and (got[2, 128:256]).isnan().all() and (got[2, :128] == 0).all() and (got[2, 256:] == 0).all()
    assert (scale[3] == 255).all() and got[3].isnan().all()
    assert (got[0] == 256).all() and (scale[0] == 119).all()  # 1 = 256 * 2^-8


# ---- projections ---------------------------------------------------------------------------
def project_case(g, fmt, T, inner, out, n=0, rank=0, counts=None, std=1.0):
    half = torch.float16 if fmt == "f16" else torch.bfloat16
    x, w = normal(g, T, inner, std=std), normal(g, out, inner, std=inner ** -0.5)
    s = {"half": half}
    if fmt == "fp8":
        (s["x"], s["x_scale"]), (s["w"], s["w_scale"]) = C.quantised_rows(x), C.quantised_matrix(w)
        s["wide"] = C.widened_rows(s["x"], s["x_scale"]), C.widened_matrix(s["w"], s["w_scale"])
    else:
        s["x"], s["w"], s["x_scale"], s["w_scale"] = x.to(half), w.to(half), None, None
        s["wide"] = s["x"].double(), s["w"].double()
    if n:
        s["a"] = normal(g, n, rank, inner, std=inner ** -0.5).to(half)
        s["b"] = normal(g, n, out, rank, std=rank ** -0.5).to(half)
        s["times"] = torch.rand(n, generator=g) * 2 - 0.5
        counts = counts or [T]
        s["q_start"] = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
        s["adapter"] = torch.randint(-1, n + 1, (len(counts),), generator=g).to(torch.int32)
        s["adapter"][0] = n - 1
    return s


def run_project(fdm, s, out, workspace=None, stream=None):
    gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    more = {}
    if "a" in s:
        more = dict(adapters=fdm.Adapters(gpu["a"], gpu["b"], gpu["times"]), q_start=gpu["q_start"], adapter=gpu["adapter"])
    fdm.project(gpu["x"], gpu["w"], out, x_scale=gpu["x_scale"], w_scale=gpu["w_scale"], workspace=workspace, stream=stream, **more)
    return out


def want_of(s, out_type):
    return C.projected(*s["wide"], out_type, s.get("a"), s.get("b"), s.get("times"), s.get("q_start"), s.get("adapter"), s["half"],
                       native=s["x_scale"] is not None and out_type is not torch.float32)


SHAPES = [  # T, in, out, adapters, rank, tokens of the requests
    (1, 16, 1, 0, 0, None), (1, 1024, 130, 1, 8, [1]), (2, 48, 33, 2, 16, [1, 1]), (5, 400, 257, 3, 24, [1, 3, 1]), (31, 128, 96, 4, 32, [7] * 4),
    (32, 2064, 128, 0, 0, None), (33, 256, 129, 9, 8, [1] * 33), (64, 528, 300, 5, 64, [16] * 4), (65, 144, 64, 2, 40, [60, 5]), (128, 512, 384, 3, 128, [1] * 100),
    (129, 80, 65, 6, 16, [0, 50, 0, 79, 0]), (200, 1040, 256, 1, 72, [180]), (300, 96, 1000, 7, 8, [3] * 100), (513, 272, 4100, 4, 32, [100, 413])]


@pytest.mark.parametrize("fmt,ty", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("fp8", "bf16"), ("fp8", "f32")])
@pytest.mark.parametrize("T,inner,out,n,rank,counts", SHAPES)
def test_project_matches_definition(fdm, fmt, ty, T, inner, out, n, rank, counts):
    s = project_case(rng(T * 31 + out), fmt, T, inner, out, n, rank, counts)
    y = torch.full((T, out), 7.0, dtype=C.DTYPES[ty], device="cuda")
    say(f"project {fmt}->{ty} T={T} in={inner} out={out} adapters={n} rank={rank}")
    run_project(fdm, s, y)
    C.check(y.cpu(), *want_of(s, y.dtype), "project")


@pytest.mark.parametrize("fmt", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("T,out,counts", [(7000, 2000, [1] * 40 + [3000, 0, 3900]), (3000, 4099, [700, 1, 2, 2200])])
def test_project_of_many_rows(fdm, fmt, T, out, counts):
    """The largest tiles, several adapters in one."""
    s = project_case(rng(T), fmt, T, 144, out, 5, 24, counts)
    y = torch.empty(T, out, dtype=s["half"], device="cuda")
    say(f"project {fmt} T={T} out={out}")
    run_project(fdm, s, y)
    C.check(y.cpu(), *want_of(s, y.dtype), "project")


@pytest.mark.parametrize("fmt,ty", [("bf16", "bf16"), ("f16", "f32"), ("fp8", "bf16"), ("fp8", "f32")])
@pytest.mark.parametrize("T", [20, 60, 128, 200])
def test_project_to_many_columns(fdm, fmt, ty, T):
    """Small tiles in whole rounds and a last one in parts, with adapters in both."""
    s = project_case(rng(T), fmt, T, 512 if fmt == "fp8" else 256, 70000, 3, 24, [T // 4, 3, T - T // 4 - 3])
    y = torch.empty(T, 70000, dtype=C.DTYPES[ty], device="cuda")
    say(f"project {fmt}->{ty} T={T} out=70000")
    run_project(fdm, s, y)
    C.check(y.cpu(), *want_of(s, y.dtype), "project")
