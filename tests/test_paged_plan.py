"""CPU checks of inferc_b200/csrc/paged_plan.h, the arithmetic that cuts the
paged attention's work among warps and finds pages: compiled on its own with
the host compiler."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "paged_plan.h"
using namespace inferc_dev::paged;

// 0 when every check holds, else the line of the first that does not.
#define CHECK(x) do { if (!(x)) return __LINE__; } while (0)

extern "C" int check_div(uint32_t d) {
  const FastDiv f(d);
  uint32_t probes[] = {0, 1, 2, d - 1, d, d + 1, 2 * d - 1, 2 * d, 0x7ffffffeu, 0x7fffffffu,
                       0x80000000u, 0xfffffffeu, 0xffffffffu};
  for (uint32_t n : probes) { CHECK(f.div(n) == n / d); CHECK(f.mod(n) == n % d); }
  uint32_t x = d * 2654435761u + 1;
  for (int i = 0; i < 2000; ++i) {
    x = x * 1664525u + 1013904223u;
    CHECK(f.div(x) == x / d);
    const uint32_t k = x / d * d;  // around a multiple
    CHECK(f.div(k) == k / d);
    if (k) CHECK(f.div(k - 1) == (k - 1) / d);
  }
  return 0;
}

extern "C" int check_shares(int64_t total, int64_t warps) {
  const int64_t n = warps_used(total, warps);
  CHECK(n >= 1 && n <= warps && n <= total);
  CHECK(first_tile(0, total, n) == 0 && first_tile(n, total, n) == total);
  for (int64_t w = 0; w < n; ++w) {
    const int64_t a = first_tile(w, total, n), b = first_tile(w + 1, total, n);
    CHECK(b > a);                                // every warp has work
    CHECK(b - a <= total / n + 1);               // and no more than its share
    CHECK(owner_of(a, total, n) == w && owner_of(b - 1, total, n) == w);
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "inferc_b200", "csrc"), str(d / "plan.cc"), "-o",
                    str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.check_div.argtypes = [ctypes.c_uint32]
    lib.check_shares.argtypes = [ctypes.c_int64] * 2
    return lib


def test_division_by_a_page_size_is_exact(plan):
    for d in list(range(1, 2000)) + [2 ** k + e for k in range(11, 31) for e in (-1, 0, 1)] + \
            [2 ** 31 - 1]:
        assert plan.check_div(d) == 0, d


def test_shares_cover_every_tile_once(plan):
    for total in list(range(1, 60)) + [1183, 1184, 1185, 4735, 4736, 4737, 99991, 10 ** 9 + 7,
                                       2 ** 45 + 3]:
        for warps in (1, 2, 7, 60, 592, 1184, 9472):
            assert plan.check_shares(total, warps) == 0, (total, warps)
