"""The same tokens through fdm_attn_forward, one after the other over its own fp32
cache, and through kv_write, rope and mla_attend as one step of a paged cache, with
the layer's projections around them in float64."""
import math

import pytest
import torch

from tests._helpers import say
from tests.mla_case import H, KVL, NH, NOPE, QA, QK, ROPE, VH, mla_weights

pytestmark = pytest.mark.gpu
SCALE = (0.1 * math.log(40.0) + 1.0) ** 2 / math.sqrt(192.0)

# Relative L2 error of a token's attention output.  The layer of one token is within 1e-6 of
# float64.  Here queries, cached rows, softmax weights and results round to 16 bits, each by at
# most u (2^-11, 2^-8), by u / sqrt(3) in the mean square.  Weights, rows and results: three such
# errors of the sum itself.  Queries and rows in a score: sqrt(2) u / sqrt(3) of sqrt(sum q^2 k^2)
# scale, which is the scores' deviation (about 1 here, 2 at most), moves a weight by as much:
# 1.63 u.  Together sqrt(3 / 3 + 1.63^2) u = 1.9 u; the projections behind are random matrices,
# which keep relative errors.  Twice that is asked for.
TOL = {"f16": 4 * 2.0 ** -11, "bf16": 4 * 2.0 ** -8}
N = 40


@pytest.fixture(scope="module")
def reference(fdm):
    w = mla_weights(911)
    say("attn_upload L=2")
    fdm.attn_upload(2, w, max_seq=64)
    hidden = torch.randn(N, H, generator=torch.Generator().manual_seed(17))
    out = []
    for t in range(N):
        d = hidden[t].cuda()
        fdm.attn_forward(2, d, t)
        out.append(d.double().cpu() - hidden[t].double())
    fdm.attn_release(2)
    half = {k: torch.from_numpy(v.view("float16") if v.dtype == "uint16" else v).cuda().double() for k, v in w.items()}
    return half, hidden, torch.stack(out)


def norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


@pytest.mark.parametrize("fmt,steps", [("f16", [N]), ("bf16", [N]), ("f16", [1, 30, 1, 1, 7])])
def test_agrees_with_the_layer_of_one_token(fdm, reference, fmt, steps):
    w, hidden, want = reference
    t = torch.float16 if fmt == "f16" else torch.bfloat16
    table = fdm.rope_table(ROPE, scaling="yarn", factor=40.0, orig_ctx=4096)
    cache = fdm.kv_cache(fmt, 9, 8)
    pages = torch.randperm(9, generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()
    k_b, v_b = w["k_b"].view(NH, KVL, NOPE), w["v_b"].view(NH, VH, KVL)
    got, done = [], 0
    for n in steps:
        x = norm(hidden[done:done + n].cuda().double(), w["attn_norm"])
        q = (norm(x @ w["q_a"].view(QA, H).T, w["q_a_norm"]) @ w["q_b"].view(NH * QK, QA).T).view(n, NH, QK)
        kv = (x @ w["kv_a"].view(KVL + ROPE, H).T).float()
        pos = torch.arange(done, done + n, dtype=torch.int32, device="cuda")
        slots = pages[pos.long() // 8] * 8 + pos % 8
        say(f"kv_write, rope and mla_attend of {n} tokens behind {done}, {fmt}")
        fdm.kv_write(cache, kv, slots, norm_w=w["kv_a_norm"].float(), table=table, pos=pos)
        q_rope = torch.empty(n, NH, ROPE, dtype=t, device="cuda")
        fdm.rope(table, q[..., NOPE:].float().contiguous(), pos, q_rope)
        q_lat = torch.stack([q[:, h, :NOPE] @ k_b[h].T for h in range(NH)], 1).to(t)
        o = torch.empty(n, NH, KVL, dtype=t, device="cuda")
        done += n
        i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
        fdm.mla_attend(cache, q_lat, q_rope, i32(0, n), i32(done), pages[None].contiguous(), SCALE, o)
        heads = torch.stack([o[:, h].double() @ v_b[h].T for h in range(NH)], 1)
        got.append((heads.view(n, NH * VH) @ w["o_proj"].view(H, NH * VH).T).cpu())
    got = torch.cat(got)
    err = (got - want).norm(dim=1) / want.norm(dim=1)
    print(f"relative L2 of {N} tokens: {float(err.max()):.2e} at most")
    assert err.max() <= TOL[fmt], err
