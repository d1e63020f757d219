"""Inputs under which a lost, doubled or misplaced part of a cut sequence shows,
and those under which fp32 results need every piece of their operands.

Each position has a weight of 1/2, 1 or 2 and a value that is 1 in one column
and 0 in the others, so that an output is a column's share of the weights, and
16 positions more or fewer change one by a percent. Tolerance: the scale ln 2 and its
product with log2 e are rounded, 3 u of scores up to 1, and 2^x to 2^-21; a
warp adds up a few hundred positions at most and the parts of a sequence are
joined in fewer than a hundred steps (512 u); then one rounding to the type."""
import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import BF16, DEV, F16, F32, U, Cache, close, gen, half_step, randn, sync_ok

TYPES = [F32, F16, BF16]
LENS = [([5001], 2, 4, 128, 16), ([70001], 1, 8, 128, 64), ([70001], 1, 8, 128, 24),
        ([1000, 3, 0, 4097, 77, 2500], 4, 4, 128, 32), ([33000], 1, 2, 256, 128),
        ([37] * 300, 2, 2, 64, 16), ([20000, 1, 1, 1, 1, 1, 1], 3, 1, 64, 16),
        ([9000] * 3, 2, 17, 96, 16), ([160], 12, 1, 64, 16), ([500], 2, 4, 64, 16)]
REL = 512 * U + 2.0 ** -20


def weights_of(n, device="cpu"):
    """(log2 of the weights, column of the value) of positions 0 .. n - 1, and d columns' sums."""
    j = torch.arange(n, device=device)
    return (j // 48 * 7 + j // 16) % 3 - 1, j // 16


def shares(n, d, device="cpu"):
    level, col = weights_of(n, device)
    w = 2.0 ** level.double()
    sums = torch.zeros(d, dtype=torch.float64, device=device).index_add_(0, col % d, w)
    return w, sums


def tolerance(out, dtype):
    return (half_step(dtype) * (1 + 2.0 ** -7) + REL) * out


@pytest.mark.parametrize("lens,hk,group,d,page", LENS, ids=str)
def test_the_tolerance_finds_a_lost_tile(lens, hk, group, d, page):
    """On the CPU: any 16 consecutive positions, lost or counted twice, are found in each type."""
    for n in set(lens):
        if n < 32:
            continue
        w, sums = shares(n, d)
        out = sums / sums.sum()
        _, col = weights_of(n)
        pad = -n % 16
        part = torch.cat([w, torch.zeros(pad, dtype=torch.float64)]).view(-1, 16).sum(1)
        at = col[::16] % d
        for sign in (-1, 1):
            changed = (sums[at] + sign * part) / (sums.sum() + sign * part)
            off = (changed - out[at]).abs() - tolerance(out[at], BF16)
            if pad:  # the last, incomplete tile may be a single position
                off = off[:-1]
            assert (off > 0).all(), (n, sign)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,hk,group,d,page", LENS, ids=str)
def test_every_part_counts(dtype, lens, hk, group, d, page):
    g = gen(len(lens) + d)
    c = Cache(g, dtype, lens, hk, d, page)
    p = torch.arange(max(lens), device=DEV)
    level, col = weights_of(max(lens), DEV)
    key = torch.zeros(max(lens), d, device=DEV)
    key[:, 1] = level.float()
    value = torch.zeros(max(lens), d, device=DEV)
    value[p, col % d] = 1
    for b, n in enumerate(lens):
        at = c.table[b].long()[p[:n] // page]
        for h in range(hk):
            c.k[at, h, p[:n] % page] = key[:n].to(dtype)
            c.v[at, h, p[:n] % page] = value[:n].to(dtype)
    q = torch.zeros(len(lens), hk * group, d, device=DEV, dtype=dtype)
    q[..., 1] = 1
    sums = torch.zeros(len(lens), hk, c.kv.capacity, device=DEV)
    scale = 0.6931471805599453
    out = ops.PagedDecodeAttention(q, c.kv, scale, sums)
    assert torch.equal(ops.PagedDecodeAttention(q, c.kv, scale), out)
    sync_ok()
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        w, cols = shares(n, d, DEV)
        want = (cols / cols.sum()).expand(hk * group, d)
        close(out[b], want, tolerance(want, dtype))
        each = (group * w / cols.sum()).expand(hk, n)
        close(sums[b, :, :n], each, (2 * REL + 2 * group * U) * each)
        assert (sums[b, :, n:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 2, 8, 12])
@pytest.mark.parametrize("d,page", [(64, 16), (96, 16), (128, 24), (192, 16), (256, 16)])
def test_fp32_keeps_all_pieces(group, d, page):
    """A score is a single product, a result the values' mean under 90 weights: the pieces of
    operands lose 2^-20 of each product and 2^-21 of a weight at most; without the smaller
    ones it would be 2^-11."""
    g = gen(group + d)
    c = Cache(g, F32, [90], 1, d, page, wide=200)
    q = torch.zeros(1, group, d, device=DEV)
    q[..., d - 3] = randn(g, 1, group)
    c.k[..., : d - 3] = 0
    c.k[..., d - 2:] = 0
    out = ops.PagedDecodeAttention(q, c.kv, 1.0)
    sync_ok()
    k, v = c.rows(c.k, 0)[0], c.rows(c.v, 0)[0]
    s = q[0].double() @ k.T
    p = torch.softmax(s, -1)
    e = 2 * s.abs().amax(-1, keepdim=True) * (2.0 ** -20 + 4 * U) + 2.0 ** -20
    close(out[0], p @ v, (e + (90 + 64) * 2 * U + 2.0 ** -20) * (p @ v.abs()))
