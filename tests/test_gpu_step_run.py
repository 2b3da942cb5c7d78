"""Steps of a paged, drafted, adapter-carrying attention as a server runs them:
kv_trim and kv_grow, add_rms_norm into 8 bits, projections with the requests'
adapters, kv_write, mla_attend and the projection back, one behind the other."""
import math

import pytest
import torch

from tests import latent_case as L
from tests import step_case as C
from tests._helpers import say
from tests.test_gpu_step import ints, normal, rng, same

pytestmark = pytest.mark.gpu
HID, H, N, B, P, PAGE, RANK = 512, 16, 80, 5, 12, 16, 16
SCALE = 1.0 / math.sqrt(192.0)
# what each step rolls back to (relative to what is cached: so many positions less) and adds
STEPS = [([0] * 5, [37, 1, 20, 0, 5]), ([0] * 5, [4, 4, 4, 30, 0]), ([2, 3, 0, 4, 1], [4, 4, 4, 4, 1]), ([1, 9, 99, 0, 0], [1, 1, 40, 1, 1]), ([3, 0, 1, 2, 5], [3, 3, 3, 3, 3])]


class Model:
    def __init__(self, fdm):
        g = rng(77)
        self.fdm = fdm
        self.norm_w, self.kv_norm = 1 + 0.1 * normal(g, HID), 1 + 0.1 * normal(g, 512)
        self.table = fdm.rope_table(64, scaling="yarn", factor=40.0, orig_ctx=4096)
        self.w, self.on = {}, {}
        for name, out, inner, fp8 in (("kv", 576, HID, True), ("q", H * 576, HID, True), ("o", HID, H * 512, False)):
            w = normal(g, out, inner, std=inner ** -0.5)
            a, b = normal(g, 3, RANK, inner, std=inner ** -0.5).bfloat16(), normal(g, 3, out, RANK, std=RANK ** -0.5).bfloat16()
            times = torch.tensor([0.5, 1.0, -0.25])
            codes, scale = C.quantised_matrix(w) if fp8 else (w.bfloat16(), None)
            self.w[name] = (C.widened_matrix(codes, scale) if fp8 else codes.double(), a, b, times)
            self.on[name] = (codes.cuda(), None if scale is None else scale.cuda(), fdm.Adapters(a.cuda(), b.cuda(), times.cuda()))
        self.adapter = [1, -1, 0, 2, 1]

    def state(self):
        """A cache, its books and a step's buffers."""
        s, z = type("State", (), {})(), lambda *k, t=torch.int32: torch.zeros(*k, dtype=t, device="cuda")
        s.cache, s.pages = self.fdm.kv_cache("bf16", B * P, PAGE), self.fdm.kv_pages(B, P, B * P, PAGE)
        s.keep, s.new, s.q_start, s.pos, s.slots, s.refused = z(B), z(B), z(B + 1), z(N), z(N), z(1)
        s.h, s.add = z(N, HID, t=torch.float32), z(N, HID, t=torch.bfloat16)
        s.codes, s.scale = z(N, HID, t=torch.uint8).view(torch.float8_e4m3fn), z(N, HID // 128, t=torch.uint8)
        s.kv, s.q, s.out = z(N, 576, t=torch.float32), z(N, H * 576, t=torch.bfloat16), z(N, H, 512, t=torch.bfloat16)
        s.adapter = ints(self.adapter)
        s.work = self.fdm.project_workspace(N, H * 512, H * 576, RANK)
        s.mla = self.fdm.mla_workspace(N, H)
        return s

    def step(self, s):
        fdm = self.fdm
        fdm.kv_trim(s.pages, s.keep)
        fdm.kv_grow(s.pages, s.new, s.q_start, s.pos, s.slots, refused=s.refused)
        fdm.add_rms_norm(s.h, s.add, self.norm_w_on, s.codes, scale=s.scale, sum=s.h)
        for name, out in (("kv", s.kv), ("q", s.q)):
            w, scale, adapters = self.on[name]
            fdm.project(s.codes, w, out, x_scale=s.scale, w_scale=scale, adapters=adapters, q_start=s.q_start, adapter=s.adapter, workspace=s.work)
        fdm.kv_write(s.cache, s.kv, s.slots, norm_w=self.kv_norm_on, table=self.table, pos=s.pos)
        q = s.q.view(N, H, 576)
        fdm.mla_attend(s.cache, q[..., :512], q[..., 512:], s.q_start, s.pages.kv_len, s.pages.pages, SCALE, s.out, workspace=s.mla)
        w, _, adapters = self.on["o"]
        fdm.project(s.out.view(N, H * 512), w, s.add, adapters=adapters, q_start=s.q_start, adapter=s.adapter, workspace=s.work)


@pytest.fixture(scope="module")
def model(fdm):
    m = Model(fdm)
    m.norm_w_on, m.kv_norm_on = m.norm_w.cuda(), m.kv_norm.cuda()
    return m


def inputs(s, books, i):
    back, new = STEPS[i]
    keep = [max(n - k, 0) for n, k in zip(books.kv_len, back)]
    s.keep.copy_(ints(keep))
    s.new.copy_(ints(new))
    h, add = normal(rng(i), N, HID), normal(rng(100 + i), N, HID).bfloat16()
    s.h.copy_(h)
    s.add.copy_(add)
    books.trim(keep)
    return (h, add) + books.grow(new, N)


def new_books():
    return C.Books([[-1] * P for _ in range(B)], [0] * B, list(range(B * P - 1, -1, -1)), B * P, PAGE)


def test_steps_against_their_definitions(fdm, model):
    """Each operator of each step against its formula on what the one before it gave."""
    s, books = model.state(), new_books()
    assert same(s.pages, books) is None
    for i in range(len(STEPS)):
        s.out.fill_(1.0)
        h, add, q_start, pos, slots, refused = inputs(s, books, i)
        say(f"step {i}")
        model.step(s)
        same(s.pages, books)
        assert (s.q_start.tolist(), s.pos.tolist(), s.slots.tolist(), s.refused.item()) == (q_start, pos, slots, refused)
        total, y = C.normed(h, add, model.norm_w, 1e-6)
        C.check(s.h.cpu(), total, total.abs() * 2.0 ** -24, "sum")
        C.check_codes(s.codes.cpu(), s.scale.cpu(), y, C.NORM_TOL)
        x = C.widened_rows(s.codes.cpu(), s.scale.cpu())
        for name, got in (("kv", s.kv), ("q", s.q)):
            want = C.projected(x, model.w[name][0], got.dtype, *model.w[name][1:], q_start, model.adapter, native=name == "q")
            C.check(got.cpu(), *want, name)
        # the cached rows: normed latents and turned keys of what was projected
        n, kv = q_start[-1], s.kv.cpu()[:q_start[-1]].double()
        rows = L.widened(s.cache.latent.cpu(), s.cache.rope.cpu())
        assert all(v >= 0 for v in slots[:n])
        mine = rows[torch.tensor(slots[:n])]
        want = L.normed(kv[:, :512], model.kv_norm.double())
        C.check(mine[:, :512], want, want.abs() * (2.0 ** -8 + C.NORM_TOL), "latent")
        freq = L.frequencies(64, scaling="yarn", factor=40.0)
        want, size = L.turned(kv[:, None, 512:], torch.tensor(pos[:n]), freq, "interleaved")
        C.check(mine[:, None, 512:], want, size * L.TURN_TOL + (want.abs() + size * L.TURN_TOL) * 2.0 ** -8, "keys")
        q = s.q.cpu().view(N, H, 576)
        out, _, tol, _ = L.attend(rows, PAGE, q[..., :512], q[..., 512:], q_start, books.kv_len, books.pages, SCALE)
        C.check(s.out.cpu()[:n], out[:n], tol[:n], "attention")
        assert (s.out[n:] == 1).all()  # rows behind the last sequence
        C.check(s.add.cpu(), *C.projected(s.out.cpu().view(N, H * 512), model.w["o"][0], torch.bfloat16, *model.w["o"][1:], q_start, model.adapter), "o")


def test_steps_in_a_graph(fdm, model):
    """The step captured once and replayed is the same steps, bit for bit; every step serves other sequences and lengths."""
    eager, held = model.state(), model.state()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        model.step(held)
    b0, b1 = new_books(), new_books()
    for i in range(len(STEPS)):
        inputs(eager, b0, i)
        inputs(held, b1, i)
        say(f"step {i}")
        model.step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(held.pages, b1)
        for k in ("q_start", "pos", "slots", "refused", "h", "codes", "scale", "kv", "q", "out", "add"):
            x, y = (getattr(v, k).contiguous().view(torch.uint8) for v in (eager, held))
            assert torch.equal(x, y), (i, k)
        assert torch.equal(eager.cache.latent, held.cache.latent) and torch.equal(eager.cache.rope, held.cache.rope)
