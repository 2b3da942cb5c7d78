"""Numbers of a projection's adapters far apart from each other and near the ends of
their range, and what the products of e4m3 rows cut off, against float64."""
import math

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
