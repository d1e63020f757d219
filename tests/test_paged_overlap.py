"""Eviction whose weights_out shares elements with weights, other than being the
same rows, is refused: what a row got depended on which thread came first. CPU:
refusals happen on the host, before anything touches a device."""
import ctypes
import os
import random
import subprocess

import pytest

from inferc_b200 import lib
from tests.test_paged import A, INVALID, kv, message

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "paged_plan.h"
using namespace inferc_dev::paged;

extern "C" int meet(const int64_t* a, const int64_t* b) {
  auto rows = [](const int64_t* x) {
    return Rows2{x[0], x[1], {{x[2], x[3]}, {x[4], x[5]}}};
  };
  return rows_meet(rows(a), rows(b));
}
"""


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    d = tmp_path_factory.mktemp("meet")
    (d / "meet.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC",
                    "-I" + os.path.join(ROOT, "inferc_b200", "csrc"), str(d / "meet.cc"), "-o",
                    str(d / "meet.so")], check=True)
    f = ctypes.CDLL(str(d / "meet.so")).meet
    return lambda a, b: bool(f((ctypes.c_int64 * 6)(*a), (ctypes.c_int64 * 6)(*b)))


def elements(r):
    base, length, n, s, m, t = r
    return [base + i * s + j * t + e for i in range(n) for j in range(m) for e in range(length)]


def test_rows_that_meet(meet):
    r = random.Random(3)
    seen = {True: 0, False: 0}
    while min(seen.values()) < 1500:
        a, b = ([r.randint(-20, 60), r.randint(0, 6), r.randint(1, 4), r.randint(-30, 30),
                 r.randint(1, 4), r.randint(-30, 30)] for _ in range(2))
        if len(set(elements(b))) < len(elements(b)):
            continue  # the rows written are apart
        want = not set(elements(a)).isdisjoint(elements(b))
        assert meet(a, b) == want, (a, b)
        seen[want] += 1


def evict(w, out, wb=256, wh=128, ob=256, oh=128, dst=3 * A):
    """Rows of 128 weights of 4 sequences and 2 key heads."""
    return lib.load().inferc_dev_paged_kv_evict(
        ctypes.byref(kv()), dst, 8, 8, w, wb, wh, out, ob, oh, 32, 8, 2 * A, A, None)


@pytest.mark.parametrize("over", [
    dict(out=A + 4), dict(out=A - 4), dict(out=A + 4 * 128), dict(out=A + 4 * 255),
    dict(out=A + 4 * 1023), dict(out=A - 4 * 1023), dict(out=A + 64, dst=None),
    dict(out=A + 4 * 100, wb=512, wh=256, ob=512, oh=256), dict(out=A + 4 * 1000, ob=128, oh=512)],
    ids=str)
def test_weights_that_lie_in_weights_out_are_refused(over):
    assert evict(A, **over) == INVALID and "share nothing" in message()


def test_weights_beside_weights_out_are_taken(meet):
    """Rows of one buffer [batch, 2, kv_heads, positions], and rows behind the last."""
    rows = lambda base, b, h: [base, 128, 4, b, 2, h]
    assert not meet(rows(0, 512, 128), rows(256, 512, 128))
    assert not meet(rows(0, 512, 256), rows(128, 512, 256))
    assert not meet(rows(0, 256, 128), rows(1024, 256, 128))
    assert meet(rows(0, 256, 128), rows(1023, 256, 128))
