"""Launches whose workgroups wait for one another, several at once: a model of
how a device dispatches them, and the turns that the library has them take
(launch_turns.h, compiled on its own with g++)."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

XCDS, PLACES = 8, 128  # 32 CUs of four workgroups each


def layer_list(K, q6, norm):
    """The batch-1 layer's work list: (what an item ends, what it waits for), in order."""
    gu, down, fin = 128, 112 if q6 else 64, 448 if q6 else 224
    items = [("inv", ())] if norm else []
    inv = ("inv",) if norm else ()
    items += [("digits", inv)] * 28 + [("row", inv)] * 256 + [("set", ("row",)), ("exact", ("row", "set"))]
    for p in range(2):
        items += [(f"shared{p}", ("digits",))] * gu
    items += [(f"record{p}", (f"shared{p}",)) for p in range(2)]
    for step in range(3):
        if step < 2:
            items += [(f"act{k}.{step}", ("digits", "set")) for k in range(K) for _ in range(gu)]
        if step > 0:
            items += [("down", ("set", f"act{k}.{step - 1}")) for k in range(K) for _ in range(down)]
    return items + [("final", ("record0", "record1", "down", "exact"))] * fin


def drains(launches, prefers):
    """Whether all items of the launches end.  Workgroup i of a launch runs on XCD
    i mod 8; an XCD dispatches a launch's workgroups in order, and fills its places
    from the launches in the order prefers(xcd)."""
    left = [{} for _ in launches]
    for n, items in zip(left, launches):
        for end, _ in items:
            n[end] = n.get(end, 0) + 1
    queue = [[list(range(x, len(items), XCDS))[::-1] for x in range(XCDS)] for items in launches]
    resident = [[] for _ in range(XCDS)]
    moved = True
    while moved:
        moved = False
        for x in range(XCDS):
            for a in prefers(x):
                while queue[a][x] and len(resident[x]) < PLACES:
                    resident[x].append((a, queue[a][x].pop()))
                    moved = True
            ready = [(a, i) for a, i in resident[x] if all(left[a].get(w, 0) == 0 for w in launches[a][i][1])]
            for a, i in ready:
                left[a][launches[a][i][0]] -= 1
            if ready:
                moved = True
                done = set(ready)
                resident[x] = [r for r in resident[x] if r not in done]
    return all(not any(n.values()) for n in left)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("q6", [False, True])
@pytest.mark.parametrize("K", [1, 8, 16])
def test_one_launch_drains(K, q6, norm):
    assert drains([layer_list(K, q6, norm)], lambda x: [0])


def test_two_launches_at_once_need_not():
    """Why the library orders them: one XCD begins with one launch, the others with the
    other; all their places fill with items that wait."""
    two = [layer_list(8, False, False)] * 2
    assert not drains(two, lambda x: [0, 1] if x == 0 else [1, 0])
    # the same launches, taken in one order everywhere
    assert drains(two, lambda x: [0, 1])


def test_a_launch_beside_work_that_does_not_wait_drains():
    """Any other kernel's workgroups only take places until they end."""
    r = random.Random(7)
    plain = [("w", ())] * 3000
    for _ in range(4):
        order = [r.sample([0, 1], 2) for _ in range(XCDS)]
        assert drains([layer_list(8, False, True), plain], lambda x: order[x])


DRIVER = r"""
#include <cstdio>
#include "launch_turns.h"
using fdm::LaunchTurns;
int main() {
  int a, b, c, bad = 0;  // their addresses are streams
  LaunchTurns t;
  if (t.before(&a) != LaunchTurns::kGo) bad |= 1;
  if (t.after(&a)) bad |= 2;                               // one stream: nothing is recorded
  if (t.before(&a) != LaunchTurns::kGo || t.after(&a)) bad |= 4;
  if (t.before(nullptr) != LaunchTurns::kMarkAndWait || t.last != &a) bad |= 8;  // the null stream is one as well
  if (!t.after(nullptr)) bad |= 16;
  if (t.before(nullptr) != LaunchTurns::kGo || !t.after(nullptr)) bad |= 32;
  if (t.before(&a) != LaunchTurns::kWait || !t.after(&a)) bad |= 64;
  if (t.before(&b) != LaunchTurns::kWait || !t.after(&b)) bad |= 128;
  t.marked = false;                                        // its event could not be recorded
  if (t.before(&c) != LaunchTurns::kMarkAndWait || t.last != &b) bad |= 256;
  t.forget(&a);                                            // not the last one
  if (t.before(&c) != LaunchTurns::kMarkAndWait) bad |= 512;
  t.forget(&b);
  if (t.before(&c) != LaunchTurns::kGo || !t.after(&c)) bad |= 1024;  // the null stream is left
  t.forget(nullptr);
  if (t.before(&c) != LaunchTurns::kGo || t.after(&c)) bad |= 2048;   // alone again
  t.forget(&c);
  if (t.any || !t.streams.empty() || t.before(&a) != LaunchTurns::kGo) bad |= 4096;
  std::printf("%d\n", bad);
  return bad != 0;
}
"""


def test_turns(tmp_path):
    src, exe = tmp_path / "turns.cpp", tmp_path / "turns"
    src.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "flash_deepseek_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "0", out.stdout


def test_turns_are_waited_for_wherever_a_grid_has_waits():
    """Every launch whose grid waits inside stands between a turn's begin and end."""
    csrc = os.path.join(ROOT, "flash_deepseek_amd", "csrc")
    waits = [f for f in sorted(os.listdir(csrc)) if f.endswith(".hip") and "spin_limit" in open(os.path.join(csrc, f)).read()]
    assert waits == ["capi.hip", "expert_kernels.hip", "layer_kernel.hip", "matvec_kernels.hip"]
    text = open(os.path.join(csrc, "capi.hip")).read()
    for launch in ("launch_layer(a, s)", "launch_expert_f32(a, s)", "launch_matvec1(a, q6, s)", "launch_matvec2_q4k(a, (int)in_dim, s)"):
        assert text.count(launch.split("(")[0] + "(") == 1, launch
        at = text.index(launch)
        assert "OneLaunch turn(s);\n" in text[at - 400:at] and "return turn.end();" in text[at:at + 100], launch
