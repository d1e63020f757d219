"""What a warp of the paged attention that gives up waits for: the slots of its
ring that are filled and not taken, all of them and no others (an unfilled one
would cost it the whole time limit). The kernel's order of fills and waits,
replayed on the host over the arithmetic of inferc_b200/csrc/paged_plan.h."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "paged_plan.h"
#include <set>
using namespace inferc_dev::paged;

// A share of `count` tiles through a ring of `slots`, given up at the wait number `at`
// (keys of tile t: 2 t, values: 2 t + 1). 0 when what is waited for then is what is in flight.
extern "C" int check_give_up(int slots, int count, int at) {
  int slot_in = 0, tiles_in = 0;
  bool fetched = false;
  std::set<int> flying;
  auto filled = [&] { slot_in = slot_in + 1 == slots ? 0 : slot_in + 1; };
  auto fill_k = [&] {
    if (tiles_in < count) { fetched = true; flying.insert(slot_in); }
    filled();
  };
  auto fill_v = [&] {
    if (fetched) { fetched = false; ++tiles_in; flying.insert(slot_in); }
    filled();
  };
  for (int i = 0; i < slots; ++i) { if (i & 1) fill_v(); else fill_k(); }
  int slot_out = 0, t = 0, keys_taken = 0, waits = 0;
  auto released = [&] { if (++slot_out == slots) slot_out = 0; };
  for (; t < count; ++t) {
    if (waits++ == at) break;
    if (!flying.erase(slot_out)) return __LINE__;
    if (slots % 2 == 0) fill_k(); else fill_v();
    released();
    if (waits++ == at) { keys_taken = 1; break; }
    if (!flying.erase(slot_out)) return __LINE__;
    if (slots % 2 == 0) fill_v(); else fill_k();
    released();
  }
  for (int i = fills_in_flight(tiles_in, fetched, 2 * t + keys_taken); i > 0; --i) {
    if (!flying.erase(slot_out)) return __LINE__;
    released();
  }
  return flying.empty() ? 0 : __LINE__;
}
"""


@pytest.fixture(scope="module")
def ring(tmp_path_factory):
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "inferc_b200", "csrc"), str(d / "ring.cc"), "-o",
                    str(d / "ring.so")], check=True)
    lib = ctypes.CDLL(str(d / "ring.so"))
    lib.check_give_up.argtypes = [ctypes.c_int] * 3
    return lib


@pytest.mark.parametrize("slots", [3, 4, 5, 6])
def test_giving_up_waits_for_what_is_in_flight(ring, slots):
    for count in range(1, 15):
        for at in range(2 * count + 1):  # the last: never
            assert ring.check_give_up(slots, count, at) == 0, (count, at)
