"""Sums over very many positions in one warp: batches whose sequences share
pages, so that each (sequence, key head) is one warp's share of 262144
positions in half a gigabyte of cache."""
import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import BF16, DEV, F16, U, gen, half_step, sync_ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group,d", [(1, 64), (4, 64), (12, 64), (1, 128)])
def test_values_of_one_sign(dtype, group, d):
    """Equal weights of values in [1, 2), so that an accumulator that is cut at every step falls
    behind. The weights are equal powers of two and exact; a tile's values are summed in a few
    steps (2^-20 of them at most) and the n / 32 or n / 16 tiles by rounded additions, u of the
    result each; then one rounding to the type."""
    n, hk, page, batch = 262144, 8, 64, 148
    g = gen(group + d)
    k = torch.zeros(n // page, hk, page, d, device=DEV, dtype=dtype)
    v = (1 + torch.rand(n // page, hk, page, d, device=DEV, generator=g)).to(dtype)
    table = torch.arange(n // page, device=DEV, dtype=torch.int32).repeat(batch, 1)
    kv = ops.PagedKV(k, v, table, torch.full((batch,), n, device=DEV, dtype=torch.int32))
    q = torch.randn(batch, hk * group, d, device=DEV, generator=g).to(dtype)
    out = ops.PagedDecodeAttention(q, kv)
    sync_ok()
    want = v.double().mean((0, 2)).repeat_interleave(group, 0)
    tiles = n / (32 if d * 2 <= 256 else 16)
    tol = (half_step(dtype) * (1 + 2.0 ** -7) + tiles * U + 2.0 ** -20) * want
    assert ((out.double() - want).abs() <= tol).all()
    assert torch.equal(out, out[:1].expand_as(out))
