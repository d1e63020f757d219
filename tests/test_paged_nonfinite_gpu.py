"""Infinities and NaN among the queries, keys and values that the paged
attention reads, against the definition in 64 bits: a key of -inf takes its
position's weight, a value of inf is its column's result, what the definition
leaves undefined is NaN, and heads and columns that meet none of it are as they
would be without. Tolerances are those of test_paged_gpu.py."""
import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import (BF16, DEV, F16, F32, U, Cache, gen, half_step, randn, sync_ok)

pytestmark = pytest.mark.gpu

# short sequences of few heads (a block each), cut ones, pages that are no multiple of 16, two
# blocks of heads, every width of the kernels
SHAPES = [(1, 4, 64, 16, None), (2, 1, 64, 16, None), (1, 12, 64, 16, 200), (2, 8, 128, 16, 300),
          (1, 17, 96, 24, 200), (1, 3, 256, 16, 300), (1, 10, 192, 16, 200), (2, 2, 40, 8, 300),
          (2, 1, 128, 16, 300)]
LENS = [300, 45, 1, 97]


def definition(c, q, b):
    """(out, tolerance, weights, their tolerance) of sequence b, infinities and NaN as sums of
    products in 64 bits give them; tolerances relative to what is finite."""
    n, hk, d, dtype = c.lens_list[b], c.hk, c.d, c.dtype
    group = q.shape[1] // hk
    k, v = c.rows(c.k, b), c.rows(c.v, b)
    qq = q[b].double().view(hk, group, d)
    scale = d ** -0.5
    x = (qq[:, :, None] * k[:, None]).sum(-1) * scale
    # no score above -inf: zeros
    p = torch.where((x == -torch.inf).all(-1, keepdim=True), 0.0, torch.softmax(x, -1))
    out = (p[..., None] * v[:, None]).sum(2).reshape(-1, d)
    finite = lambda t: t.abs().nan_to_num(nan=0.0, posinf=0.0)
    size = scale * (finite(qq) @ finite(k).transpose(1, 2)).amax(-1, keepdim=True)
    e = 2 * size * ((d + 8) * 2 * U + 2.0 ** -20) + 2.0 ** -20
    pieces = 2.0 ** -21 if dtype == F32 else half_step(dtype) ** 2
    rel = e + (n + 64) * 2 * U + pieces
    mag = p.nan_to_num(nan=0.0) @ finite(v)
    tol = (rel * mag).reshape(-1, d) + half_step(dtype) * finite(out) * (1 + 2.0 ** -7) + \
        2.0 ** -25 + n * 2.0 ** -35 * float(finite(v).max())
    w = p.sum(1)
    return out, tol, w, (e * p.nan_to_num(nan=0.0)).sum(1) + (group + 8) * 2 * U * (1 + finite(w))


def same(got, want, tol):
    got = got.double()
    odd = ~want.isfinite()
    assert torch.equal(got[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0),
                       want[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
    err = (got - want).abs()[~odd]
    assert (err <= tol[~odd]).all(), f"worst {float((err / tol[~odd]).nan_to_num(nan=9e9).max())}"


def check(c, q):
    w = torch.zeros(len(c.lens_list), c.hk, c.kv.capacity, device=DEV)
    got = ops.PagedDecodeAttention(q, c.kv, weights=w)
    alone = ops.PagedDecodeAttention(q, c.kv)
    sync_ok()
    for b, n in enumerate(c.lens_list):
        want, tol, p, ptol = definition(c, q, b)
        same(got[b], want, tol)
        same(alone[b], want, tol)
        same(w[b, :, :n], p, ptol)
        assert (w[b, :, n:] == 0).all()


def put(c, x, b, j, h, col, value):
    """Value of position j of sequence b, key head h, column col."""
    x[int(c.table[b, j // c.page]), h, j % c.page, col] = value


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hk,group,d,page,wide", SHAPES)
def test_infinite_keys_and_values(dtype, hk, group, d, page, wide):
    g = gen(hk + group + d)
    c = Cache(g, dtype, LENS, hk, d, page, wide=wide)
    q = randn(g, len(LENS), hk * group, d, dtype=dtype)
    inf, nan = float("inf"), float("nan")
    # keys of -inf for heads whose query is positive there, weight 0; others get +inf: NaN
    q[0, :, 5] = q[0, :, 5].abs() + 0.1
    q[0, 0, 5] *= -1 if hk * group > 1 else 1
    for j in (0, 31, 130, 299):
        put(c, c.k, 0, j, 0, 5, -inf)
    # values: one infinity, both signs, NaN, and one whose key takes all weight from it
    for j, col, x in ((3, 0, inf), (44, 1, -inf), (7, 2, inf), (8, 2, -inf), (20, d - 1, nan)):
        put(c, c.v, 1, j, hk - 1, col, x)
    put(c, c.v, 2, 0, 0, 3, inf)
    q[3, :, 1] = q[3, :, 1].abs() + 0.1
    put(c, c.k, 3, 60, hk - 1, 1, -inf)
    put(c, c.v, 3, 60, hk - 1, 4, inf)
    check(c, q)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hk,group,d,page,wide", SHAPES)
def test_queries_that_are_no_numbers(dtype, hk, group, d, page, wide):
    """One head of each sequence: a NaN as the device's arithmetic makes it (every bit of it
    set but the sign), one of few bits, an infinity; the other heads are not touched by it."""
    g = gen(hk * group + d)
    c = Cache(g, dtype, LENS, hk, d, page, wide=wide)
    q = randn(g, len(LENS), hk * group, d, dtype=dtype)
    bits = q.view(torch.int32 if dtype == F32 else torch.int16)
    most = {F32: 0x7fffffff, F16: 0x7fff, BF16: 0x7fff}[dtype]
    least = {F32: 0x7f800001, F16: 0x7c01, BF16: 0x7f81}[dtype]
    bits[0, 0, 3] = most
    bits[1, -1, d - 1] = least
    q[3, 0, 0] = float("inf")
    check(c, q)


def test_no_score_above_minus_infinity_gives_zeros():
    for dtype in (F32, F16, BF16):
        for group in (1, 4):
            c = Cache(gen(1), dtype, [70, 20], 2, 64, 16)
            q = randn(gen(2), 2, 2 * group, 64, dtype=dtype).abs() + 0.1
            for j in range(70):
                put(c, c.k, 0, j, 1, 9, -float("inf"))
            check(c, q)


def test_largest_numbers():
    """Operands close to the type's largest finite number, whose halves round to infinity."""
    for group in (1, 4, 12):
        g = gen(group)
        c = Cache(g, F32, [40], 1, 64, 16)
        q = torch.zeros(1, group, 64, device=DEV)
        q[:, :, 0] = 3.4028e38
        c.k[..., 0] = c.k[..., 0].nan_to_num(nan=0.0) * 1e-37
        c.k[..., 1:] = 0.0
        c.v[..., 2] = 1e36
        check(c, q)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_short_sequences_in_one_share(dtype):
    """Some seventy (sequence, key head)s in every warp's share, infinities in a few of them."""
    g = gen(8)
    batch, hk, group, d, page = 20000, 4, 2, 16, 16
    k, v = (randn(g, batch, hk, page, d, dtype=dtype) for _ in range(2))
    q = randn(g, batch, hk * group, d, dtype=dtype)
    lens = torch.randint(0, page + 1, (batch,), generator=g, device=DEV, dtype=torch.int32)
    for x, count in ((k, 300), (v, 300)):
        at = torch.randint(0, x.numel(), (count,), generator=g, device=DEV)
        x.view(-1)[at] = torch.where(torch.rand(count, generator=g, device=DEV) < 0.5, 1.0,
                                     -1.0).to(dtype) * float("inf")
    table = torch.arange(batch, device=DEV, dtype=torch.int32)[:, None].contiguous()
    w = torch.zeros(batch, hk, page, device=DEV)
    out = ops.PagedDecodeAttention(q, ops.PagedKV(k, v, table, lens), weights=w)
    sync_ok()
    held = torch.arange(page, device=DEV) < lens[:, None]
    kk, vv = k.double(), v.double()
    x = (q.double().view(batch, hk, group, 1, d) * kk[:, :, None]).sum(-1) * d ** -0.5
    x = torch.where(held[:, None, None], x, -torch.inf)
    p = torch.where((x == -torch.inf).all(-1, keepdim=True), 0.0, torch.softmax(x, -1))
    vv = torch.where(held[:, None, :, None], vv, 0.0)
    want = (p[..., None] * vv[:, :, None]).sum(3).view(batch, hk * group, d)
    got = out.double()
    odd = ~want.isfinite()
    assert 200 < int(odd.any(-1).sum()) < 5000
    assert torch.equal(got[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0),
                       want[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
    # scores below 40, 16 positions: fp32 steps of 80 (d + 8) u, one rounding to the type
    tol = half_step(dtype) * want[~odd].abs() * (1 + 2.0 ** -7) + 2.0 ** -11 * 2.0 ** -4
    assert ((got - want)[~odd].abs() <= tol).all()
    sums = torch.where(held[:, None], p.sum(2), 0.0)  # only positions that are held get any
    assert torch.equal(w.isnan(), sums.isnan())
    assert ((w - sums)[~sums.isnan()].abs() <= 2.0 ** -15 * group).all()
