"""Numbers of a projection's adapters far apart from each other and near the ends of
their range, and what the products of e4m3 rows cut off, against float64."""
import pytest
import torch

from tests import step_case as C
from tests._helpers import say
from tests.test_gpu_step import normal, project_case, rng, run_project, want_of

pytestmark = pytest.mark.gpu


# T, out, rank: whole tiles of each size, and parts joined on the matrix cores (in = 64)
SIZES = [(12, 40000, 24), (4100, 128, 72), (454, 4126, 72), (300, 12100, 40), (284, 2917, 72), (4168, 140, 24)]


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("T,out,rank", SIZES)
def test_adapters_at_the_ends_of_fp32(fdm, fmt, T, out, rank):
    """A x near 2^122 and near 2^-112 (2^-100 in BF16, whose third number is a normal one then), whose
    products with B are numbers of fp32; W 0, so that the small ones show."""
    s = project_case(rng(T + rank), fmt, T, 64, out, 2, rank, [T // 2, T - T // 2])
    s["adapter"], s["times"] = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([2.0 ** 122, 2.0 ** (-112 if fmt == "f16" else -100)])
    s["w"] = torch.zeros_like(s["w"])
    s["wide"] = s["wide"][0], s["w"].double()
    say(f"project {fmt} T={T} out={out} rank={rank}, the ends of fp32")
    y = run_project(fdm, s, torch.empty(T, out, device="cuda"))
    C.check(y.cpu(), *want_of(s, y.dtype), "project")


@pytest.mark.parametrize("T,out,rank", SIZES)
def test_adapters_of_values_far_apart(fdm, T, out, rank):
    """A x spread over 2^-18 of its largest and B the other way round, so that every value of the
    rank counts the same.  In F16: each off by 2^-16 of itself, or 2^-36 of the largest, at most."""
    g = rng(T + rank)
    s = project_case(g, "f16", T, 64, out, 2, rank, [T // 2, T - T // 2])
    s["adapter"], s["times"] = torch.tensor([0, 1], dtype=torch.int32), None
    s["w"] = (normal(g, out, 64) * 2.0 ** -8).half()
    down = torch.exp2(-18.0 * torch.randperm(rank, generator=g) / (rank - 1)).round(decimals=9)
    s["a"] = (normal(g, 2, rank, 64) * 2.0 ** 5 * down[None, :, None]).half()
    s["b"] = (normal(g, 2, out, rank) * 2.0 ** -10 / down).half()
    x, w, a, b = (s[k].cuda().double() for k in ("x", "w", "a", "b"))
    n = 64 / 8 + 24
    want, tol = x @ w.T, (x.abs() @ w.abs().T) * n * 2.0 ** -23
    for k, t in ((0, slice(0, T // 2)), (1, slice(T // 2, T))):
        u = x[t] @ a[k].T
        du = (x[t].abs() @ a[k].abs().T) * (n + 2) * 2.0 ** -23 + torch.maximum(u.abs() * 2.0 ** -16, u.abs().amax(-1, keepdim=True) * 2.0 ** -36)
        want[t] += u @ b[k].T
        tol[t] += du @ b[k].abs().T + (u.abs() @ b[k].abs().T) * (rank / 8 + 24) * 2.0 ** -23
    say(f"project f16 T={T} out={out} rank={rank}, far apart")
    y = run_project(fdm, s, torch.empty(T, out, device="cuda"))
    C.check(y, want, tol + want.abs() * 2.0 ** -24, "project")


@pytest.mark.parametrize("ty", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T", [5, 40, 100, 140])
def test_where_e4m3_products_end(fdm, T, ty):
    """1 + 2^-j - 1, the first two among eight neighbours: kept to 2^-13, and off by less than that below; all of it in fp32."""
    out, j = 200, 6 + torch.arange(200) // 2 % 10
    sign = 1.0 - 2.0 * (torch.arange(200) % 2)
    x, w = torch.zeros(T, 64), torch.zeros(out, 64)
    x[:, 1] = 2.0 ** -6
    x[:, 0] = x[:, 16] = w[:, 0] = 1.0
    w[:, 16] = -1.0
    w[:, 1] = sign * torch.exp2(6.0 - j)
    F8 = torch.float8_e4m3fn
    s = {"x": x.to(F8), "w": w.to(F8), "x_scale": torch.full((T, 1), 127, dtype=torch.uint8), "w_scale": torch.full((2, 1), 127, dtype=torch.uint8)}
    y = run_project(fdm, s, torch.empty(T, out, dtype=ty, device="cuda")).double().cpu()
    want = (sign * torch.exp2(-j.double())).expand(T, out)
    kept = (j <= 13) | (ty is torch.float32)
    assert torch.equal(y[:, kept], want[:, kept])
    assert ((y - want).abs() < 2.0 ** -13).all()


@pytest.mark.parametrize("ty", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,out", [(20, 2112), (64, 2112), (256, 2112), (2048, 4200)])
def test_what_e4m3_products_lose(fdm, T, out, ty):
    """Of 7168 normal values, with steps of 2^-13 of the power of two of the largest of eight: 2.0e-5 of
    the results' rms where each product is cut to them, 1.5e-5 where it is rounded (a model of the eight
    in float64; cut downwards it would be 2.2e-4).  Beside the rounding of the results themselves, and
    sqrt(7168 / 32) roundings of 2^-24 of sums of that size in fp32."""
    g = rng(T)
    x, w = torch.randn(T, 7168, generator=g), torch.randn(out, 7168, generator=g) * 7168 ** -0.5
    (xc, xs), (wc, ws) = C.quantised_rows(x), C.quantised_matrix(w)
    y = run_project(fdm, {"x": xc, "w": wc, "x_scale": xs, "w_scale": ws}, torch.empty(T, out, dtype=ty, device="cuda"))
    want = C.widened_rows(xc.cuda(), xs.cuda()) @ C.widened_matrix(wc.cuda(), ws.cuda()).T
    own = (want.to(ty).double() - want).square().mean()
    lost = 2.5e-5 if ty is not torch.float32 else 15 * 2.0 ** -24
    assert (y.double() - want).square().mean() <= own + (lost * want.square().mean().sqrt()) ** 2
