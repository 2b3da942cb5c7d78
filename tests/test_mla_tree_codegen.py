"""What the latent attention's products in assembly rely on in the code
generated around them, read from the assembly of mla_tree_kernels.hip compiled
here (no GPU needed).  The compiler knows nothing of such a product: neither
the states that its operands and results take, nor the direct loads' base."""
import os
import re
import subprocess

import pytest

from flash_deepseek_amd import build as B

READY = 11    # states between a product's issue and an ALU instruction on its result
OPERAND = 2   # between an ALU instruction's result and a product that reads it
BASE = 5      # between a scalar written from a lane and a load that it is the base of


def registers(text):
    m = re.match(r"([avs])\[(\d+):(\d+)\]", text)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.match(r"([avs])(\d+)\b", text)
    return {(m[1], int(m[2]))} if m else set()


def too_close(lines):
    """The instructions of `lines`, in their order, that come too early."""
    found, state, product, alu, lane = [], 0, {}, {}, {}
    for ln in lines:
        ln = ln.split(";")[0].strip()
        if not ln or ln.startswith(".") or ln.endswith(":"):
            continue
        op, _, rest = ln.partition(" ")
        if op == "s_nop":
            state += int(rest) + 1
            continue
        state += 1
        args = [registers(t.strip()) for t in rest.split(",")]
        writes = not op.startswith(("ds_write", "global_store", "global_load_lds", "scratch_store", "v_cmp", "s_cmp", "s_wait", "s_cbranch"))
        to = args[0] if writes else set()
        if op.startswith("v_mfma"):
            if any(state - alu.get(r, -99) <= OPERAND for a in args[1:] for r in a):
                found.append(("operand", ln))
            if any(state - product.get(r, -99) <= READY for a in args[1:3] for r in a):
                found.append(("operand is a result", ln))
            product.update(dict.fromkeys(to, state))
        else:
            if any(state - product.get(r, -99) <= READY for a in args for r in a):
                found.append(("result", ln))
            if op.startswith("global_load_lds") and any(state - lane.get(r, -99) <= BASE for a in args[1:] for r in a):
                found.append(("base", ln))
            for r in to:
                product.pop(r, None)
                if op.startswith("v_"):
                    alu[r] = state
                if op.startswith("v_read"):
                    lane[r] = state
                else:
                    lane.pop(r, None)
    return found


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """{kernel: its assembly lines}"""
    try:
        hipcc = B._hipcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    out = str(tmp_path_factory.mktemp("mla") / "mla_tree.s")
    subprocess.run([hipcc, *B.CXXFLAGS, "--cuda-device-only", "-S", os.path.join(B.CSRC, "mla_tree_kernels.hip"), "-o", out],
                   check=True, capture_output=True)
    kernels, lines = {}, None
    with open(out) as f:
        for ln in f:
            if re.match(r"_ZN\w+:", ln):
                lines = kernels.setdefault(ln.split(":")[0], [])
            elif lines is not None:
                lines.append(ln.strip())
    kernels = {k: v for k, v in kernels.items() if re.search(r"k_mla_treeILi\dE", k)}
    assert len(kernels) == 6  # three formats, pages of a step and more or of less
    return kernels


def test_the_check_sees_what_it_looks_for():
    score = "v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], v[0:15]"
    assert [k for k, _ in too_close(["v_mov_b32_e32 v21, 0", "s_nop 0", score])] == ["operand"]
    assert too_close(["v_mov_b32_e32 v21, 0", "s_nop 1", score, score]) == []
    assert [k for k, _ in too_close([score, "s_nop 9", "v_add_f32_e32 v30, v15, v31"])] == ["result"]
    assert too_close([score, "s_nop 11", "v_add_f32_e32 v30, v15, v31"]) == []
    assert [k for k, _ in too_close(["v_readlane_b32 s4, v0, 8", "s_nop 3", "global_load_lds_dwordx4 v1, s[4:5]"])] == ["base"]
    assert too_close(["v_readlane_b32 s4, v0, 8", "s_nop 4", "global_load_lds_dwordx4 v1, s[4:5]"]) == []


def test_products_and_direct_loads_have_their_states(assembly):
    for kernel, lines in assembly.items():
        assert sum(ln.startswith("v_mfma") for ln in lines) >= 36 + 68 + 32, kernel
        assert too_close(lines) == [], kernel


def test_the_steps_reload_nothing(assembly):
    """No block with products (but the last values') reloads a spilled register:
    such a load waits for all that is being brought, 10 to 30 % of a step."""
    for kernel, lines in assembly.items():
        blocks, block = [], []
        for ln in lines:
            if ln.startswith(".LBB"):
                blocks.append(block)
                block = []
            block.append(ln)
        blocks.append(block)
        for block in blocks:
            products = sum(ln.startswith("v_mfma") for ln in block)
            if 0 < products < 32:
                assert not any(ln.startswith("scratch_") for ln in block), (kernel, block[0], products)
