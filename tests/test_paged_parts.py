"""Where the parts of a cut sequence are looked up (inferc_b200/csrc/paged_plan.h),
compiled on its own with the host compiler: the slots that the warps wrote, and
no others when a kernel finds other lengths than the one before it."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "paged_plan.h"
#include <set>
using namespace inferc_dev::paged;

// Tiles t0 .. t0 + tiles - 1 of `total` by `used` warps: the slots of their parts are those
// that the warps with a tile of them write (the first one its second slot).
extern "C" int check_parts(int64_t t0, int64_t tiles, int64_t total, int64_t used) {
  std::set<int64_t> want;
  for (int64_t w = 0; w < used; ++w) {
    const int64_t a = first_tile(w, total, used), b = first_tile(w + 1, total, used);
    if (a < t0 + tiles && b > t0) want.insert(2 * w + (a <= t0 ? 1 : 0));
  }
  if (want.size() < 2) return 0;  // not cut
  const Parts p = parts_of(t0, tiles, total, used);
  std::set<int64_t> got;
  for (int i = 0; i < p.count; ++i) got.insert(p.slot(i));
  // (a share that begins with the first tile begins it, too)
  return got == want ? 0 : __LINE__;
}

// Whatever the numbers, no slot but the `used` warps'.
extern "C" int check_bounds(int64_t t0, int64_t tiles, int64_t total, int64_t used) {
  for (Parts p : {parts_of(t0, tiles, total, used), parts_within(t0, tiles, used)})
    for (int i : {0, 1, p.count - 1})
      if (i < p.count && (p.count < 1 || p.slot(i) < 0 || p.slot(i) >= 2 * (used < 1 ? 1 : used)))
        return __LINE__;
  return 0;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("parts")
    (d / "parts.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "inferc_b200", "csrc"), str(d / "parts.cc"), "-o",
                    str(d / "parts.so")], check=True)
    lib = ctypes.CDLL(str(d / "parts.so"))
    for f in (lib.check_parts, lib.check_bounds):
        f.argtypes = [ctypes.c_int64] * 4
    return lib


def test_parts_of_a_cut_sequence(plan):
    r = random.Random(1)
    for _ in range(3000):
        total = r.randint(1, 400)
        used = r.randint(1, min(total, 40))
        t0 = r.randrange(total)
        assert plan.check_parts(t0, r.randint(1, total - t0), total, used) == 0, (t0, total, used)


def test_lengths_that_changed_name_no_other_slots(plan):
    r = random.Random(2)
    for _ in range(3000):
        total = r.choice([0, 1, r.randint(1, 400), r.randint(1, 1 << 40)])
        used = min(total, r.choice([1, 7, 592, 1184]))
        t0, tiles = r.randint(0, 2 * total + 50), r.randint(1, 2 * total + 50)
        assert plan.check_bounds(t0, tiles, total, used) == 0, (t0, tiles, total, used)
