"""Projections through every way that they are cut, joined and given their adapters, in each
format, against float64."""
import pytest
import torch

from tests import step_case as C
from tests._helpers import say
from tests.project_paths import PATHS
from tests.test_gpu_step import project_case, rng, run_project

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,ty", [("bf16", "bf16"), ("f16", "f32"), ("fp8", "bf16"), ("fp8", "f32")])
@pytest.mark.parametrize("tile,whole,join,call", PATHS)
def test_projections_by_every_way(fdm, fmt, ty, tile, whole, join, call):
    T, row_bytes, out, n, rank, B = call
    counts = [T * (b + 1) // B - T * b // B for b in range(B)]
    s = project_case(rng(T + out), fmt, T, row_bytes // (1 if fmt == "fp8" else 2), out, n, rank, counts)
    y = torch.empty(T, out, dtype=C.DTYPES[ty], device="cuda")
    say(f"project {fmt}->{ty} {call}: tiles of {tile}, join {join}")
    run_project(fdm, s, y)
    a, b = (s[k].cuda() if n else None for k in ("a", "b"))  # (large sums of float64: on the GPU)
    C.check(y, *C.projected(*(v.cuda() for v in s["wide"]), y.dtype, a, b, s.get("times"), s.get("q_start"), s.get("adapter"), s["half"],
                            native=fmt == "fp8" and ty != "f32"), "project")
