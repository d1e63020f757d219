"""Attention whose results take the queries' place: as into memory of their own,
infinities among the operands (whose shares are walked twice) included."""
import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import BF16, DEV, F16, F32, Cache, gen, randn, sync_ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hk,group,d,page,wide", [
    (2, 4, 64, 16, None), (3, 1, 64, 16, None), (2, 8, 128, 16, 300), (1, 17, 96, 24, 200),
    (2, 1, 128, 16, 300), (1, 12, 256, 16, 300)])
@pytest.mark.parametrize("finite", [True, False])
def test_out_may_be_the_queries(dtype, hk, group, d, page, wide, finite):
    g = gen(hk + group + d)
    c = Cache(g, dtype, [300, 0, 45, 1, 97], hk, d, page, wide=wide)
    q = randn(g, 5, hk * group, d, dtype=dtype)
    if not finite:
        for b, j in ((0, 130), (2, 7), (4, 96)):
            c.v[int(c.table[b, j // page]), hk - 1, j % page, 3] = float("inf")
    w = [torch.zeros(5, hk, c.kv.capacity, device=DEV) for _ in range(2)]
    want = ops.PagedDecodeAttention(q, c.kv, weights=w[0])
    sync_ok()
    assert want.isinf().any() != finite
    got = ops.PagedDecodeAttention(q, c.kv, weights=w[1], out=q)
    sync_ok()
    assert got is q and torch.equal(q, want) and torch.equal(*w)
