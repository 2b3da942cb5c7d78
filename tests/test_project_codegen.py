"""What the projections' tiles rely on in the code generated for them, read from the
assembly of project_kernels.hip compiled here (no GPU needed): sums that stay in
registers, and turns whose products run where the source has them, behind the operands'
reads and before the next barrier."""
import os
import re
import subprocess

import pytest

from flash_deepseek_amd import build as B

# products of a turn of the largest tile, by format (F16, BF16, e4m3 at once, e4m3 widened)
PRODUCTS = {0: 32, 1: 32, 2: 8, 3: 64}


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """{kernel: its assembly lines}, and the private bytes of each kernel"""
    try:
        hipcc = B._hipcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    out = str(tmp_path_factory.mktemp("project") / "project.s")
    subprocess.run([hipcc, *B.CXXFLAGS, "--cuda-device-only", "-S", os.path.join(B.CSRC, "project_kernels.hip"), "-o", out], check=True, capture_output=True)
    kernels, lines, private, name = {}, None, {}, None
    with open(out) as f:
        for ln in f:
            if re.match(r"_ZN\w+:", ln):
                lines = kernels.setdefault(ln.split(":")[0], [])
            elif lines is not None:
                lines.append(ln.strip())
            m = re.match(r"\s+\.name:\s+(_ZN\w+)", ln)
            name = m[1] if m else name
            m = re.match(r"\s+\.private_segment_fixed_size:\s+(\d+)", ln)
            if m:
                private[name] = int(m[1])
    return kernels, private


def test_nothing_is_spilled(assembly):
    private = assembly[1]
    assert sum("k_project" in k for k in private) >= 16
    assert not {k: v for k, v in private.items() if v}


def test_turns_hold_their_products(assembly):
    seen = set()
    for name, lines in assembly[0].items():
        m = re.search(r"k_projectILi(\d)ELi256E", name)
        if not m:
            continue
        turns, count = [], None
        for ln in lines:
            if ln.startswith("s_setprio 1"):
                count = 0
            elif ln.startswith("s_setprio 0"):
                turns.append(count)
                count = None
            elif count is not None:
                assert not ln.startswith(("s_barrier", "ds_read", "global_load", "s_cbranch")), (name, ln)
                count += ln.startswith("v_mfma")
        assert turns and set(turns) == {PRODUCTS[int(m[1])]}, (name, turns)
        seen.add(int(m[1]))
    assert seen == set(PRODUCTS)


def test_no_packed_fp32(assembly):
    for name, lines in assembly[0].items():
        assert not [ln for ln in lines if re.match(r"v_pk_(add|mul|fma)_f32", ln)], name
