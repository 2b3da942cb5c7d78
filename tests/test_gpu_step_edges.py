"""Where the cache's books, the residual's norm and projections with adapters can go
wrong: what stands in other rows and adapters, strides, scales and numbers at the ends
of their ranges, workspaces, streams and graphs, and offsets that pass 32 bits."""
import math

import pytest
import torch

from tests import step_case as C
from tests._helpers import say
from tests.test_gpu_step import books, ints, normal, on_gpu, project_case, rng, run_project, same, want_of

pytestmark = pytest.mark.gpu


def bits(t):
    return t.contiguous().view(torch.uint8)


# ---- a row alone ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("ty", ["half", "f32"])
@pytest.mark.parametrize("T,out,rank", [(1, 40, 8), (7, 300, 16), (20, 2000, 72), (50, 200, 32), (100, 520, 64), (300, 600, 128), (2100, 4100, 24)])
def test_a_row_stands_alone(fdm, fmt, ty, T, out, rank):
    """Rows of requests 0, 2, 4, .. keep their bits when all others' rows and adapters become NaN and infinities."""
    g = rng(T + rank)
    counts = [T] if T == 1 else [T // 5, T // 7 + 1, 1, T - T // 5 - T // 7 - 2]
    s = project_case(g, fmt, T, 144, out, 2 * len(counts), rank, counts)
    s["adapter"] = torch.arange(len(counts), dtype=torch.int32) * 2
    first = run_project(fdm, s, torch.empty(T, out, dtype=s["half"] if ty == "half" else torch.float32, device="cuda"))
    C.check(first.cpu(), *want_of(s, first.dtype), "project")
    mine = torch.zeros(T, dtype=torch.bool)
    for r in range(0, len(counts), 2):
        mine[s["q_start"][r]:s["q_start"][r + 1]] = True
    s["x"] = s["x"].clone()
    if fmt == "fp8":
        s["x"].view(torch.uint8)[~mine] = 0x7f  # NaN
    else:
        s["x"][~mine] = torch.where(torch.arange(144) % 2 == 0, math.inf, math.nan).to(s["half"])
    for k in range(2 * len(counts)):
        if k not in range(0, 2 * len(counts), 4):
            s["a"][k], s["b"][k], s["times"][k] = math.nan, math.inf, math.nan
    again = run_project(fdm, s, torch.empty_like(first))
    assert torch.equal(bits(again[mine]), bits(first[mine]))
    assert again[~mine.cuda()].isnan().all()


@pytest.mark.parametrize("T,out", [(1, 200), (30, 1000), (70, 500), (200, 700), (2500, 4500)])
def test_rows_of_no_request_and_odd_ranges(fdm, T, out):
    """Ranges that begin before the rows or end behind them are cut; empty ones, adapters that are none, and one adapter of many requests."""
    s = project_case(rng(T), "bf16", T, 80, out, 3, 16, [T])
    s["times"] = None
    a, b = T // 3, T // 2
    for q, ad in (([-5, a, a, b, 2 ** 31 - 1], [1, 2, -1, 1]), ([-2 ** 31, -7, 1, 2 ** 31 - 1], [0, 2, 2]), ([a, b, T], [3, 2 ** 31 - 1]), ([a, b, b], [-2 ** 31, 0]),
                  ([T, T + 5, T + 9], [0, 1]), ([-9, -3, 0], [0, 1]), ([a] + [b] * 40, [2] * 40)):
        s["q_start"], s["adapter"] = torch.tensor(q).clamp(max=2 ** 31 - 1).int(), torch.tensor(ad).int()
        y = run_project(fdm, s, torch.full((T, out), 7.0, dtype=torch.bfloat16, device="cuda"))
        C.check(y.cpu(), *want_of(s, y.dtype), f"{q} {ad}")


def test_requests_out_of_order_touch_nothing_else(fdm):
    """Where ranges fall, what a row is given is open; rows in no range keep W x, and no range reads elsewhere."""
    for T in (40, 500):
        s = project_case(rng(T), "bf16", T, 80, 300, 2, 16, [T])
        plain = {k: v for k, v in s.items() if k not in ("a", "b", "times")}
        want, tol = want_of(plain, torch.float32)
        for q in ([0, 5, -2 ** 31, 9], [9, 3, 5, -1], [4, 2 ** 31 - 1, -2 ** 31, 2]):
            s["q_start"], s["adapter"] = torch.tensor(q).int(), torch.tensor([0, 1, 0]).int()
            y = run_project(fdm, s, torch.empty(T, 300, device="cuda")).cpu()
            if q[1] < T:
                C.check(y[9:], want[9:], tol[9:], f"{q}")


@pytest.mark.parametrize("T", [5, 4096, 5000])
def test_many_requests_of_many_adapters(fdm, T):
    n, B = 1024, 4096
    g = rng(T)
    cut = torch.sort(torch.randint(0, T + 1, (B - 1,), generator=g)).values
    s = project_case(g, "f16", T, 64, 96, n, 8, [T])
    s["q_start"] = torch.cat((torch.tensor([0]), cut, torch.tensor([T]))).int()
    s["adapter"] = torch.randint(-1, n, (B,), generator=g).int()
    say(f"project T={T} with {n} adapters and {B} requests")
    y = run_project(fdm, s, torch.empty(T, 96, dtype=torch.float16, device="cuda"))
    C.check(y.cpu(), *want_of(s, y.dtype), "project")


# ---- places ----------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,out", [(3, 250), (60, 520), (200, 400), (2200, 4200)])
def test_rows_inside_wider_ones(fdm, fmt, ty, T, out):
    """x, W and y inside larger tensors, y aligned and not; what lies beside y stays."""
    s = project_case(rng(out), fmt, T, 208, out, 2, 16, [T // 2, T - T // 2])
    want = run_project(fdm, s, torch.empty(T, out, dtype=ty, device="cuda"))
    C.check(want.cpu(), *want_of(s, ty), "project")
    wide = dict(s)
    for k in ("x", "w"):
        v = torch.zeros(s[k].shape[0], 208 + 48).to(s[k].dtype).cuda()
        v.view(torch.uint8).fill_(0x7f)
        v[:, 16:224] = s[k].cuda()
        wide[k] = v[:, 16:224]
    if fmt == "fp8":
        wide["x_scale"] = torch.cat((torch.full((T, 1), 255, dtype=torch.uint8), s["x_scale"], torch.full((T, 4), 255, dtype=torch.uint8)), 1).cuda()[:, 1:3]
    for off in (0, 8, 5):
        room = torch.full((T + 2, out + 16), 3.0, dtype=ty, device="cuda")
        run_project(fdm, wide, room[1:-1, off:off + out])
        assert torch.equal(room[1:-1, off:off + out], want)
        assert (room[0] == 3).all() and (room[-1] == 3).all() and (room[:, :off] == 3).all() and (room[:, off + out:] == 3).all()


def test_one_row_for_all(fdm):
    s = project_case(rng(2), "bf16", 1, 96, 500)
    for T in (4, 90, 3000):
        s["x"] = s["x"][:1].cuda().expand(T, 96)
        y = run_project(fdm, s, torch.empty(T, 500, dtype=torch.bfloat16, device="cuda"))
        assert torch.equal(y, y[:1].expand(T, 500))
    s["wide"] = s["x"][:1].double().cpu(), s["wide"][1]
    C.check(y[:1].cpu(), *want_of(s, y.dtype), "project")


def test_no_rows(fdm):
    s = project_case(rng(2), "fp8", 4, 96, 50, 2, 16, [4])
    s["x"], s["x_scale"] = s["x"][:0], s["x_scale"][:0]
    run_project(fdm, s, torch.empty(0, 50, device="cuda"))
    fdm.add_rms_norm(torch.empty(0, 64, device="cuda"), None, None, torch.empty(0, 64, device="cuda"))


@pytest.mark.parametrize("T", [30, 600])
def test_offsets_past_32_bits(fdm, T):
    """Rows of x, W and y 8 MB apart: the last ones lie behind 4 GB."""
    far, out = 1 << 22, 600
    s = project_case(rng(9), "bf16", T, 64, out, 2, 8, [T - 3, 3])
    big = {k: torch.empty(s[k].shape[0] * far, dtype=torch.bfloat16, device="cuda").as_strided((s[k].shape[0], 64), (far, 1)) for k in ("x", "w")}
    for k in big:
        big[k].copy_(s[k])
    y = torch.empty(T * far, dtype=torch.bfloat16, device="cuda").as_strided((T, out), (far, 1))
    say(f"project T={T} of rows {2 * far} bytes apart")
    run_project(fdm, {**s, **big}, y)
    C.check(y.cpu(), *want_of(s, y.dtype), "project")
    w = torch.ones(64, device="cuda")
    z = torch.empty(T * far, dtype=torch.bfloat16, device="cuda").as_strided((T, 64), (far, 1))
    fdm.add_rms_norm(big["x"], None, w, z)
    want = torch.empty(T, 64, dtype=torch.bfloat16, device="cuda")
    fdm.add_rms_norm(s["x"].cuda(), None, w, want)
    assert torch.equal(z, want)


# ---- numbers at the ends ---------------------------------------------------------------------
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [2, 100, 2100])
def test_scales_that_are_none(fdm, T, ty):
    """255 on a group of x: its row; on a tile of W: its columns.  The others do not notice."""
    s = project_case(rng(T), "fp8", T, 400, 4400)
    s["x_scale"][T // 2, 2] = 255
    s["w_scale"][1, 3] = 255
    s["wide"] = C.widened_rows(s["x"], s["x_scale"]), C.widened_matrix(s["w"], s["w_scale"])
    y = run_project(fdm, s, torch.empty(T, 4400, dtype=ty, device="cuda"))
    C.check(y.cpu(), *want_of(s, ty), "project")


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [3, 140, 2100])
def test_scales_at_their_ends(fdm, T, ty):
    """Scale bytes 10 .. 246, of x and W against each other."""
    s = project_case(rng(T), "fp8", T, 272, 4300)
    for k, e in (("x_scale", 117), ("w_scale", -117)):
        s[k] = (s[k].int() * 0 + 127 + e).to(torch.uint8)
    s["x_scale"][:, 1], s["w_scale"][:, 1] = 10, 244
    s["x"] = s["x"].float().clamp(-2, 2).to(s["x"].dtype)
    s["wide"] = C.widened_rows(s["x"], s["x_scale"]), C.widened_matrix(s["w"], s["w_scale"])
    y = run_project(fdm, s, torch.empty(T, 4300, dtype=ty, device="cuda"))
    C.check(y.cpu(), *want_of(s, ty), "project")


@pytest.mark.parametrize("T", [4, 64, 2100])
@pytest.mark.parametrize("fmt", ["f16", "bf16"])
def test_adapters_of_large_and_small_numbers(fdm, fmt, T):
    """A x past the largest F16 number and below its smallest ones, row by row."""
    s = project_case(rng(T), fmt, T, 128, 4200, 2, 40, [T // 2, T - T // 2])
    s["adapter"] = torch.tensor([0, 1], dtype=torch.int32)
    s["times"] = torch.tensor([1e6, 3e-12])
    for ty in (torch.float32, torch.bfloat16 if fmt == "bf16" else torch.float32):
        y = run_project(fdm, s, torch.empty(T, 4200, dtype=ty, device="cuda"))
        C.check(y.cpu(), *want_of(s, ty), "project")
    s["times"] = torch.tensor([math.inf, 0.0])
    y = run_project(fdm, s, torch.empty(T, 4200, device="cuda"))
    assert not y[:T // 2].isfinite().any()
    C.check(y[T // 2:].cpu(), *(v[T // 2:] for v in want_of({**s, "times": torch.zeros(2)}, y.dtype)), "project")


def test_norm_of_large_and_small_numbers(fdm):
    x = torch.tensor([[1e18, -2e18, 3e17, 1e18] * 40, [1e-18, 2e-18, -1e-18, 0.0] * 40, [1e-30] * 160])
    y = torch.empty(3, 160, device="cuda")
    fdm.add_rms_norm(x.cuda(), None, None, y, eps=0.0)
    want = C.normed(x, None, None, 0.0)[1]
    C.check(y[:2].cpu(), want[:2], want[:2].abs() * (C.NORM_TOL + 2.0 ** -24), "norm")
    fdm.add_rms_norm(x.cuda(), None, None, y, eps=1e-6)
    want = C.normed(x, None, None, 1e-6)[1]
    C.check(y.cpu(), want, want.abs() * (C.NORM_TOL + 2.0 ** -24), "norm")


# ---- workspaces, streams, graphs ---------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_workspaces(fdm, fmt):
    """One workspace for calls of fewer rows, with anything in it, and of the least size; same bits each time."""
    big = fdm.project_workspace(3000, 528, 700, 32)
    for T in (1, 33, 100, 400, 2500):
        s = project_case(rng(T), fmt, T, 528, 700, 3, 32, [T // 2, T - T // 2])
        want = run_project(fdm, s, torch.empty(T, 700, dtype=torch.bfloat16, device="cuda"))
        C.check(want.cpu(), *want_of(s, want.dtype), "project")
        for ws in (big, fdm.project_workspace(T, 528, 700, 32)):
            ws.fill_(255)  # NaN
            assert torch.equal(run_project(fdm, s, torch.empty_like(want), workspace=ws), want)
        with pytest.raises(fdm.FdmError, match="workspace of"):
            run_project(fdm, s, torch.empty_like(want), workspace=big[:64])


@pytest.mark.parametrize("fmt,T,inner,out", [("bf16", 1, 1024, 200), ("fp8", 40, 1040, 300), ("bf16", 200, 512, 700), ("f16", 2300, 144, 4200), ("fp8", 3000, 272, 4400)])
def test_project_in_graphs_and_on_streams(fdm, fmt, T, inner, out):
    """Two captured calls that share a workspace, replayed one after the other with changed rows between; a call on another stream."""
    s = project_case(rng(T), fmt, T, inner, out, 3, 24, [T // 3, T - T // 3])
    gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    adapters = fdm.Adapters(gpu["a"], gpu["b"], gpu["times"])
    more = dict(x_scale=gpu["x_scale"], w_scale=gpu["w_scale"], adapters=adapters, q_start=gpu["q_start"], adapter=gpu["adapter"])
    ws = fdm.project_workspace(T, inner, out, 24)
    outs = [torch.zeros(T, out, dtype=s["half"], device="cuda") for _ in range(2)]
    rows = [gpu["x"].clone(), gpu["x"].view(torch.uint8).flip(0).view(gpu["x"].dtype).clone() if fmt == "fp8" else gpu["x"].flip(0).contiguous()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, x, y in zip(graphs, rows, outs):
        with torch.cuda.graph(graph, stream=stream):
            fdm.project(x, gpu["w"], y, workspace=ws, **more)
    for turn in range(4):
        if turn:  # other rows, other requests
            for x in rows:
                x.copy_(x.view(torch.uint8).roll(1, 0).view(x.dtype))
            gpu["adapter"].copy_(torch.tensor([turn % 3, -1 if turn == 2 else 0]).int())
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(rows, outs):
            want = torch.empty_like(y)
            fdm.project(x, gpu["w"], want, **more)
            assert torch.equal(want, y)
            y.zero_()
            torch.cuda.synchronize()
    side = torch.empty_like(want)
    stream.wait_stream(torch.cuda.current_stream())
    fdm.project(rows[1], gpu["w"], side, stream=stream, **more)
    stream.synchronize()
    assert torch.equal(side, want)


def test_norm_in_a_graph_and_on_a_stream(fdm):
    x, w = normal(rng(1), 20, 1536).cuda(), torch.rand(1536, device="cuda")
    codes, scale, total = torch.empty(20, 1536, device="cuda").to(torch.float8_e4m3fn), torch.empty(20, 12, dtype=torch.uint8, device="cuda"), torch.empty_like(x)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        fdm.add_rms_norm(x, total, w, codes, scale=scale, sum=x)
    total.copy_(x)
    for turn in range(4):
        start = x.clone()
        want, ws, wt = torch.empty_like(codes), torch.empty_like(scale), torch.empty_like(x)
        fdm.add_rms_norm(start, total, w, want, scale=ws, sum=wt)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(want), bits(codes)) and torch.equal(ws, scale) and torch.equal(wt, x)
    fdm.add_rms_norm(start, total, w, codes, scale=scale, stream=stream)
    stream.synchronize()
    assert torch.equal(bits(want), bits(codes)) and torch.equal(ws, scale)


def test_books_of_two_caches_at_once(fdm):
    """Two caches' books on two streams, several workgroups each: nothing is shared."""
    g = rng(12)
    pair = [books(g, 40, 400, 17000, 16, 4000) for _ in range(2)]
    on = [on_gpu(fdm, b) for b in pair]
    streams = [torch.cuda.Stream() for _ in pair]
    new = [torch.randint(0, 1500, (40,), generator=g).tolist() for _ in pair]
    keep = [torch.randint(0, 4000, (40,), generator=g).tolist() for _ in pair]
    N = 40 * 1500
    out = [[torch.empty(k, dtype=torch.int32, device="cuda") for k in (41, N, N)] for _ in pair]
    dn, dk = [ints(n) for n in new], [ints(k) for k in keep]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            fdm.kv_trim(on[i], dk[i], stream=streams[i])
            fdm.kv_grow(on[i], dn[i], *out[i], stream=streams[i])
    torch.cuda.synchronize()
    for b, p, n, k, o in zip(pair, on, new, keep, out):
        for _ in range(5):
            b.trim(k)
            want = b.grow(n, N)
        assert [v.tolist() for v in o] == list(want[:3])
        same(p, b)


def test_books_made_beside_other_work(fdm):
    """A handle that is made while its stream is busy serves another stream at once."""
    b = books(rng(5), 3, 40, 200, 16, 300)
    tensors = ints(b.pages), ints(b.kv_len), ints(b.free), ints([b.n_free])
    new, q, pos, slots = ints([5, 0, 70]), *(torch.empty(k, dtype=torch.int32, device="cuda") for k in (4, 80, 80))
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    x = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        x = x @ x * 1e-2
    p = fdm.KvPages(*tensors, 16)
    fdm.kv_grow(p, new, q, pos, slots, stream=other)
    other.synchronize()
    want = b.grow([5, 0, 70], 80)
    assert [q.tolist(), pos.tolist(), slots.tolist()] == list(want[:3])
    same(p, b)


@pytest.mark.parametrize("fmt,ty", [("f16", torch.bfloat16), ("bf16", torch.float16), ("fp8", torch.float16)])
@pytest.mark.parametrize("T,out", [(3, 300), (50, 520), (300, 2100), (2100, 4200)])
def test_rows_in_one_type_results_in_another(fdm, fmt, ty, T, out):
    s = project_case(rng(T), fmt, T, 176, out, 3, 40, [T // 2, 1, T - T // 2 - 1])
    y = run_project(fdm, s, torch.empty(T, out, dtype=ty, device="cuda"))
    C.check(y.cpu(), *want_of(s, ty), "project")


@pytest.mark.parametrize("fmt", ["f16", "bf16", "fp8"])
@pytest.mark.parametrize("ty", [torch.float32, torch.float16])
@pytest.mark.parametrize("T,out,rank,counts", [(500, 2111, 64, [250, 250]), (500, 2112, 16, [3, 497]), (700, 2113, 128, [1] * 700), (700, 2120, 8, [7] * 100),
                                               (300, 7200, 40, [1] * 300), (2100, 7001, 24, [900, 1200])])
def test_joins_of_many_chunks(fdm, fmt, ty, T, out, rank, counts):
    """Parts joined on the matrix cores and value by value, long and short ranks, odd columns."""
    s = project_case(rng(T + rank), fmt, T, 1552, out, 9, rank, counts)
    y = run_project(fdm, s, torch.empty(T, out, dtype=ty, device="cuda"))
    C.check(y.cpu(), *want_of(s, ty), "project")


# ---- the largest -----------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,T,inner,out,rank", [("bf16", 1 << 20, 16, 24, 8), ("fp8", 2, 16, 1 << 18, 8), ("bf16", 3, 1 << 18, 5, 16), ("fp8", 40, 1 << 18, 130, 128),
                                                 ("f16", 1000, 1 << 16, 260, 24)])
def test_projections_of_the_largest_sizes(fdm, fmt, T, inner, out, rank):
    s = project_case(rng(T), fmt, T, inner, out, 2, rank, [T - 2, 1, 1])
    say(f"project {fmt} T={T} in={inner} out={out}")
    y = run_project(fdm, s, torch.empty(T, out, device="cuda"))
    C.check(y.cpu(), *want_of(s, y.dtype), "project")


def test_norm_of_the_most_rows(fdm):
    x = normal(rng(1), 1 << 21, 8)
    y = torch.empty(1 << 21, 8, device="cuda")
    fdm.add_rms_norm(x.cuda(), None, None, y)
    want = C.normed(x, None, None, 1e-6)[1]
    C.check(y.cpu(), want, want.abs() * (C.NORM_TOL + 2.0 ** -24), "norm")


def test_books_of_the_most_places(fdm):
    """2^25 places in one call, and slots just below 2^31."""
    n, page = 1 << 23, 1 << 15
    p = fdm.kv_pages(4, 300, 65535, page)
    p.free.copy_(torch.arange(65535, dtype=torch.int32))  # the last pages first
    q, pos, slots = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (5, 4 * n, 4 * n))
    fdm.kv_grow(p, ints([5, 0, 7, 0]), q, pos, slots)
    assert slots[:5].tolist() == [65534 * page + i for i in range(5)] and slots[5:12].tolist() == [65533 * page + i for i in range(7)]
    assert (slots[12:] == -1).all() and (pos[12:] == 0).all()
    fdm.kv_grow(p, ints([n] * 4), q, pos, slots)
    assert q.tolist() == [k * n for k in range(5)] and p.kv_len.tolist() == [n + 5, n, n + 7, n]
    for b, at in enumerate((5, 0, 7, 0)):
        want = torch.arange(at, at + n, device="cuda")
        assert torch.equal(pos[b * n:(b + 1) * n].long(), want)
        assert torch.equal(slots[b * n:(b + 1) * n].long(), p.pages[b].long()[want // page] * page + want % page)
    used = torch.cat([p.pages[b][:-(-m // page)] for b, m in enumerate(p.kv_len.tolist())])
    assert used.unique().numel() == used.numel() == 65535 - p.n_free.item()
    fdm.kv_trim(p, ints([0, 0, 0, 0]))
    assert p.n_free.item() == 65535 and p.free.unique().numel() == 65535 and p.kv_len.sum() == 0


def test_calls_of_two_threads(fdm):
    """Two threads with a stream and a workspace each."""
    import threading
    jobs, failed = [], []
    for k, (T, out) in enumerate(((70, 700), (300, 2100))):
        s = {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in project_case(rng(k), "bf16", T, 528, out, 3, 32, [T // 2, T - T // 2]).items()}
        want = run_project(fdm, s, torch.empty(T, out, dtype=torch.bfloat16, device="cuda"))
        jobs.append((s, want, fdm.project_workspace(T, 528, out, 32), torch.cuda.Stream()))
    torch.cuda.synchronize()

    def work(s, want, ws, stream):
        outs = [torch.empty_like(want) for _ in range(20)]
        stream.wait_stream(torch.cuda.current_stream())
        for y in outs:
            run_project(fdm, s, y, workspace=ws, stream=stream)
        stream.synchronize()
        failed.extend(i for i, y in enumerate(outs) if not torch.equal(y, want))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
