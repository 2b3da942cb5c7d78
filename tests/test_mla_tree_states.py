"""The states that a 32x32x16 product's result takes on gfx950, as this compiler keeps
them for its own products: 12 before an ALU instruction reads it, and so for
the latent attention's products in assembly."""
import os
import re
import subprocess

import pytest

from flash_deepseek_amd import build as B
from tests import test_mla_tree_codegen as codegen
from tests.test_mla_tree_codegen import assembly  # noqa: F401  (a fixture)

READY = 12

BUILTIN = r"""
#include <hip/hip_runtime.h>
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__global__ void k(const bf16x8* a, float* o) {
  f32x16 c = {};
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[threadIdx.x], a[threadIdx.x + 64], c, 0, 0, 0);
  o[threadIdx.x] = c[0] * 2.0f;
}
"""


@pytest.fixture(autouse=True)
def ready(monkeypatch):
    monkeypatch.setattr(codegen, "READY", READY)


def test_what_the_compiler_keeps_for_its_own(tmp_path):
    try:
        hipcc = B._hipcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    src, out = tmp_path / "k.hip", tmp_path / "k.s"
    src.write_text(BUILTIN)
    subprocess.run([hipcc, *B.CXXFLAGS, "--cuda-device-only", "-S", str(src), "-o", str(out)], check=True, capture_output=True)
    lines = [ln.split(";")[0].strip() for ln in out.read_text().splitlines()]
    at = next(i for i, ln in enumerate(lines) if ln.startswith("v_mfma_f32_32x32x16_bf16"))
    states, i = 0, at + 1
    first = re.match(r"v_mfma\S+ v\[(\d+):", lines[at])[1]
    while not re.search(rf"\bv{first}\b", lines[i]):
        if lines[i] and not lines[i].endswith(":"):
            states += int(lines[i].split()[1]) + 1 if lines[i].startswith("s_nop") else 1
        i += 1
    assert states == READY


def test_a_state_too_few_is_seen():
    score = "v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], v[0:15]"
    read = "v_add_f32_e32 v30, v15, v31"
    assert [k for k, _ in codegen.too_close([score, "s_nop 10", read])] == ["result"]
    assert codegen.too_close([score, "s_nop 11", read]) == []


def test_products_have_their_states(assembly):  # noqa: F811
    for kernel, lines in assembly.items():
        assert codegen.too_close(lines) == [], kernel
