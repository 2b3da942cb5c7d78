"""How a projection's work is cut (project_work.h), compiled here for the CPU: every tile is
done once, parts have work, and a workspace suffices for every call that it is asked for."""
import os
import random
import subprocess

import pytest

from flash_deepseek_amd import build as B

MAIN = r"""
#include <cstdio>
#include "project_work.h"
using namespace fdm;
int main() {
  int T, in, out, rank, B, n, size, cus;
  while (scanf("%d %d %d %d %d %d %d %d", &T, &in, &out, &rank, &B, &n, &size, &cus) == 8) {
    const ProjectPlan p = project_plan(T, (int64_t)in * size, out, B, n, rank, cus);
    printf("%d %d %d %d %lld %d %zu %zu %zu\n", p.tile, p.full, p.splits, p.u_splits, (long long)tiles_of(p.tile, T, out), steps_of((int64_t)in * size),
           project_bytes(p, T, out, rank), project_most_bytes(T, in, out, rank, cus), project_most_bytes(2 * T + 100, in, out, rank, cus));
  }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("work")
    (d / "main.cpp").write_text(MAIN)
    exe = str(d / "work")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", B.CSRC, str(d / "main.cpp"), "-o", exe], check=True)

    def run(calls):
        text = "\n".join(" ".join(map(str, c)) for c in calls)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout
        return [list(map(int, line.split())) for line in out.splitlines()]
    return run


def calls(count):
    r = random.Random(7)
    log = lambda lo, hi: int(lo * (hi / lo) ** r.random())
    got = [(T, 8, 1, 0, 0, 0, 2, 256) for T in (1, 32, 33, 64, 65, 128, 129, 1 << 20)] + [(1 << 20, 262144, 262144, 128, 4096, 1024, 2, 256)]
    for _ in range(count):
        rank = r.choice([0, 8, 64, 72, 128])
        got.append((log(1, 1 << 20), 8 * log(1, 32768), log(1, 262144), rank, log(1, 4096), log(1, 1024), r.choice([1, 2]), r.choice([256, 256, 304, 64])))
    return got


def test_every_tile_is_done_once_and_fits(plans):
    asked = calls(4000)
    rows, cols = (32, 64, 128, 256), (128, 128, 128, 256)
    for (T, inner, out, rank, B, n, size, cus), (tile, full, splits, u, tiles, steps, need, most, more) in zip(asked, plans(asked)):
        case = (T, inner, out, rank, B, n, size, cus)
        assert tiles == -(-T // rows[tile]) * -(-out // cols[tile]) and 0 <= full <= tiles, case
        assert full == tiles or full == tiles - tiles % cus, case  # whole rounds, or all
        assert 1 <= splits <= steps == -(-inner * size // 128), case
        assert splits == 1 or (tiles - full) * splits <= 2 * cus, case
        assert full == tiles or splits > 1 or rank, case
        assert (1 <= u <= min(8, steps)) if rank else u == 0, case
        assert not (rank and full) or u == 1, case  # whole tiles read one sum
        assert need <= most <= more, case
        assert 256 <= most <= max(T, min(8 * T, 64 * cus)) * rank * 4 + 512 + 2 * cus * 128 * 128 * 4 + cus * 256 * 256 * 4, case


def test_the_measured_sizes_are_cut_as_measured(plans):
    """Where one tile was clearly faster."""
    got = plans([(500, 2048, 7168, 0, 0, 0, 2, 256), (1000, 16384, 7168, 0, 0, 0, 2, 256), (256, 16384, 7168, 0, 0, 0, 2, 256), (8192, 8192, 8192, 0, 0, 0, 2, 256),
                 (128, 1536, 24576, 0, 0, 0, 2, 256), (5050, 16384, 7168, 0, 0, 0, 2, 256)])
    assert [(g[0], g[2]) for g in got[:5]] == [(2, 1), (3, 2), (2, 2), (3, 1), (2, 1)]
    assert got[5][0] == 3 and got[5][1] == 512 and got[5][2] > 1  # the last round's 48 tiles are cut
