"""Boundaries of an append that name more rows than there are: the rows there
are go to their places, and the next synchronisation reports it."""
import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import DEV, F32, Cache, gen, int32, randn, sync_code, sync_ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cu,lens,places", [
    # rows 4 and 5 of sequence 0 are not there
    ([0, 6], [10], {0: (0, 4), 1: (0, 5), 2: (0, 6), 3: (0, 7)}),
    # all rows of sequence 1 are not there
    ([0, 4, 7], [9, 3], {0: (0, 5), 1: (0, 6), 2: (0, 7), 3: (0, 8)}),
    # the first two rows of sequence 0 are not there
    ([-2, 2, 4], [9, 3], {0: (0, 7), 1: (0, 8), 2: (1, 1), 3: (1, 2)})])
def test_boundaries_outside_the_rows_are_reported(cu, lens, places):
    c = Cache(gen(1), F32, lens, 2, 64, 4, poison=False)
    rows = randn(gen(2), 4, 2, 64)
    want = c.k.clone()
    for row, (b, p) in places.items():
        want[int(c.table[b, p // 4]), :, p % 4] = rows[row]
    sync_ok()
    ops.PagedKVAppend(c.kv, rows, rows, int32(cu))
    assert sync_code() == 5
    assert torch.equal(c.k, want)
    sync_ok()


def test_boundaries_within_the_rows_are_not():
    c = Cache(gen(1), F32, [9, 3], 2, 64, 4, poison=False)
    rows = randn(gen(2), 8, 2, 64)
    for cu in ([0, 4, 7], [0, 0, 3], [0, 5, 8], [0, 0, 0]):
        ops.PagedKVAppend(c.kv, rows, rows, int32(cu))
        sync_ok()
