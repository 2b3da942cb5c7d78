"""The norm of more rows than the card has CUs, whose workgroups take several chunks a thread,
and of aligned F16 rows."""
import pytest

from tests import test_gpu_step as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,d", [(257, 512), (300, 520), (300, 2048), (300, 2056), (257, 4096), (300, 4104), (300, 7168), (260, 8192), (300, 8200), (300, 16384), (300, 16392),
                                 (256, 7168), (300, 7167)])
@pytest.mark.parametrize("tx,ta,ty", [("bf16", "bf16", "fp8"), ("f32", "bf16", "fp8"), ("bf16", None, "bf16"), ("f32", "f32", "f32")])
def test_norm_of_many_rows(fdm, T, d, tx, ta, ty):
    S.test_norm_matches_definition(fdm, T, d, tx, ta, ty, True)


@pytest.mark.parametrize("T,d", [(5, 512), (16, 1536), (3, 7168), (300, 1536), (300, 7168), (300, 8192), (2, 32768)])
@pytest.mark.parametrize("ta,ty", [("f16", "fp8"), ("f16", "f16"), (None, "fp8"), (None, "f32"), ("bf16", "f16")])
def test_norm_of_f16_rows(fdm, T, d, ta, ty):
    S.test_norm_matches_definition(fdm, T, d, "f16", ta, ty, d != 512)
