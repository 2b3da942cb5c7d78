"""The sizes of tests/project_paths.py still take the ways that they stand for: how calls are cut
and joined (project_work.h), compiled here for the CPU."""
import subprocess

from flash_deepseek_amd import build as B
from tests.project_paths import PATHS

MAIN = r"""
#include <cstdio>
#include "project_work.h"
using namespace fdm;
int main() {
  int T, bytes, out, n, rank, B;
  while (scanf("%d %d %d %d %d %d", &T, &bytes, &out, &n, &rank, &B) == 6) {
    const ProjectPlan p = project_plan(T, bytes, out, B, n, rank, 256);
    printf("%d %d %d\n", kTiles[p.tile].rows, p.full > 0, (int)project_join(p, T, out, B, rank, 256));
  }
}
"""


def test_every_path_is_taken(tmp_path):
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = str(tmp_path / "paths")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", B.CSRC, str(tmp_path / "main.cpp"), "-o", exe], check=True)
    text = "\n".join(" ".join(map(str, call)) for *_, call in PATHS)
    out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
    joins = ("none", "one", "four", "rows")
    assert [(int(a), b == "1", joins[int(c)], call) for (a, b, c), (*_, call) in zip(map(str.split, out), PATHS)] == PATHS
    # every tile, whole and in parts, with each join that its number of values allows, with and without a second half of the rank
    ways = {(tile, whole, join, call[4] > 64) for tile, whole, join, call in PATHS if call[4]}
    for tile in (32, 64, 128, 256):
        for whole in (False, True):
            for far in (False, True):
                assert (tile, whole, "one", far) in ways and (not whole or (tile, whole, "none", far) in ways)
                assert tile < 128 or (tile, whole, "rows", far) in ways
