"""How the latent attention counts and cuts its work (mla_work.h, compiled on its
own with g++): the closed forms against sums over tiles, calls of more than 2^32
units, and the calls that the host refuses."""
import ctypes
import os
import subprocess

import pytest

from flash_deepseek_amd import _lib
from tests.test_latent_args import INVAL, STATE, attend, cache

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash_deepseek_amd", "csrc")

HEAD = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include "mla_work.h"
using namespace fdm;
constexpr int R = kTileRows, S = kTilePos;
// steps of a tile from its rows alone: the last one's token, and what that sees
static int64_t steps(const SeqWork& s, int tile, int H, bool in_order) {
  const int64_t row = std::min<int64_t>((int64_t)R * (tile + 1), (int64_t)s.n * H) - 1;
  const int64_t sees = in_order ? s.len - s.n + row / H + 1 : s.len;
  int64_t n = 0;
  while (n * S < sees) ++n;
  return std::max<int64_t>(n, 1);
}
static int fail(const char* what, const SeqWork& s, int H, int tile) {
  std::printf("%s: n %d len %d H %d tile %d\n", what, s.n, s.len, H, tile);
  return 1;
}
"""

DRIVERS = {
    "sums": r"""
int main() {
  std::srand(3);
  const int heads[] = {1, 2, 3, 7, 16, 24, 40, 64, 96, 127, 128};
  for (int H : heads)
    for (int k = 0; k < 60; ++k) {
      SeqWork s;
      s.n = 1 + std::rand() % (k < 30 ? 12 : 700);
      s.len = std::rand() % (k % 3 ? 3000 : 60);
      s.t0 = 0;
      for (bool in_order : {true, false}) {
        const int tiles = tiles_of<R>(s, H);
        if ((int64_t)tiles * R < (int64_t)s.n * H || (int64_t)(tiles - 1) * R >= (int64_t)s.n * H) return fail("tiles", s, H, tiles);
        int64_t sum = 0;
        for (int t = 0; t <= tiles; ++t) {
          if (units_before<R, S>(s, t, H, in_order) != sum) return fail("sum", s, H, t);
          if (t == tiles) break;
          if (tile_steps<R, S>(s, t, H, in_order) != steps(s, t, H, in_order)) return fail("steps", s, H, t);
          sum += steps(s, t, H, in_order) + kTileCost;
        }
        if ((uint64_t)sum > most_units(s.n, H, 1, s.len)) return fail("bound", s, H, tiles);
      }
    }
  return 0;
}
""",
    "large": r"""
// calls whose units pass 2^31 and 2^32: every unit belongs to one range, every tile's parts are counted
int main() {
  struct { int B, n, len, H; bool in_order; } calls[] = {
      {2, 262144, 262144, 128, true}, {1, 524288, 524288, 128, true}, {1, 65536, 1048576, 128, false},
      {4, 262144, 1048576, 128, true}, {512, 2048, 1048576, 40, false}, {1, 1048576, 1048576, 128, true}};
  for (auto& c : calls) {
    const SeqWork s{c.n, c.len, 0};
    static UnitMarks before;
    uint64_t total = 0;
    for (int b = 0; b < c.B; ++b) {
      before.put(b, total);
      if (before.at(b) != total) return fail("mark", s, c.H, b);
      total += units_before<R, S>(s, tiles_of<R>(s, c.H), c.H, c.in_order);
    }
    before.put(c.B, total);
    int64_t slow = 0;
    for (int t = 0; t < tiles_of<R>(s, c.H); ++t) slow += tile_units<R, S>(s, t, c.H, c.in_order);
    if ((uint64_t)slow * c.B != total || before.at(c.B) != total) return fail("total", s, c.H, 0);
    if (total <= 0x7FFFFFFFull) return fail("not a large one", s, c.H, 0);
    if (total > most_units(c.B * c.n, c.H, c.B, c.len) || total > kMaxUnits) return fail("bound", s, c.H, 0);
    for (uint64_t T : {total, kMaxUnits, (uint64_t)2 * 256 + 5, (uint64_t)65535, (uint64_t)65536 * 256 + 255})
      for (uint64_t G : {1, 3, 32, 255, 256}) {
        const Ranges ranges(T, G);
        for (uint64_t g = 0; g < G; ++g) {
          const uint64_t from = ranges.start(g), to = ranges.start(g + 1);
          if (from != g * T / G || to != (g + 1) * T / G || from >= to) return fail("range", s, c.H, (int)g);
          if (ranges.at(from) != (int)g || ranges.at(to - 1) != (int)g || ranges.at(from + (to - from) / 2) != (int)g) return fail("at", s, c.H, (int)g);
        }
        if (ranges.start(0) != 0 || ranges.start(G) != T) return fail("ends", s, c.H, 0);
      }
  }
  return 0;
}
""",
}
DRIVERS["quick"] = r"""
#include <ctime>
// sequences of more tokens than positions: counted without a walk over their tiles
int main() {
  const clock_t start = std::clock();
  int64_t all = 0;
  for (int len : {0, 1, 100, 5000, 1048575}) {
    const SeqWork s{1 << 20, len, 0};
    for (int H : {128, 127, 16, 1})
      for (int t = 0; t < 2000; ++t) all += units_before<R, S>(s, tiles_of<R>(s, H) - t, H, true);
  }
  const double seconds = (double)(std::clock() - start) / CLOCKS_PER_SEC;
  std::printf("%.3f s for 40000 sums (%lld)", seconds, (long long)all);
  return seconds > 2.0;  // 40000 sums of a few divisions; a walk over up to 2^20 tiles each takes minutes
}
"""


def run(tmp_path, name):
    src, exe = tmp_path / f"{name}.cpp", tmp_path / name
    src.write_text(HEAD + DRIVERS[name])
    subprocess.run(["g++", "-std=c++17", "-O2", "-w", "-D__HIP_PLATFORM_AMD__", "-I", CSRC, "-I", "/opt/rocm/include", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stdout


def test_sums_over_tiles(tmp_path):
    run(tmp_path, "sums")


def test_more_tokens_than_positions(tmp_path):
    run(tmp_path, "quick")


def test_more_than_32_bits_of_units(tmp_path):
    run(tmp_path, "large")


@pytest.mark.parametrize("kw", [dict(N=1 << 20, H=128, pages_stride=1 << 21, o0=65536, ql0=65536), dict(N=1 << 20, H=64, pages_stride=(1 << 31) - 1, o0=65536),
                                dict(N=1 << 18, H=128, pages_stride=(1 << 27) - 1, o0=65536)])
def test_more_work_than_a_call_takes_is_refused(kw):
    assert attend(**kw) == INVAL and "more work" in _lib.lib.fdm_last_error().decode()


def test_the_largest_work_gets_as_far_as_the_device():
    if _lib.lib.fdm_available():
        pytest.skip("library already initialised in this process")
    # 2^20 + 2 tiles of (2^25 - 2048) / 32 + 7 units: below 2^40
    page = ctypes.byref(_lib.KvCacheDesc(1 << 20, 1 << 20, None, 1, 4, 2048))
    assert attend(c=page, N=1 << 20, H=128, pages_stride=(1 << 14) - 1, o0=65536) == STATE
    assert attend(c=cache(), N=1, H=1, pages_stride=(1 << 31) - 1) == STATE
