"""GPU tests of the paged-cache operators against plain 64-bit
implementations of their definitions (include/inferc_dev.h).

Tolerances, with u = 2^-24 (half a step of fp32) and h = half a step of the
result's type (finfo.eps / 2):

- every result is rounded to its type once: h * |exact|, and half the spacing
  of fp16's subnormals, 2^-25, near zero;
- norm and rotation: a sum of d squares, a square root, a division and five
  products and sums in fp32: (d + 16) u relative to |a c| + |b s|;
- attention: a score is a dot product of d terms accumulated in fp32 (one
  step, 2 u, per term where a matrix instruction truncates), with fp32
  operands in two 11-bit pieces whose dropped part is at most 2^-20 of each
  product; then a scaling by two roundings and 2^x to 2^-21. So with
  S = scale * max_j sum_i |q_i k_ij| the weights are relatively off by at most
  e = 2 S ((d + 8) 2 u + 2^-20) + 2^-20, twice over because of the normaliser,
  and an output by e + (n + 64) 2 u + (the weights' pieces: h^2 for 16-bit
  types, 2^-21 for fp32) relative to sum_j p_j |v_j|. fp16 pieces of a weight
  below 2^-38 vanish: n 2^-36 max|v| more.
- a summed weight: e * p, and 2 u of the running sum per addition.
"""
import os
import random
import subprocess
import sys

import pytest
import torch

from inferc_b200 import lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=F32).to(dtype)


def sync_ok():
    lib.check(lib.load().inferc_dev_stream_synchronize(torch.cuda.current_stream().cuda_stream))


def sync_code():
    return lib.load().inferc_dev_stream_synchronize(torch.cuda.current_stream().cuda_stream)


def close(got, want, tol):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    bad = ~(err <= tol)  # NaN counts as bad
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((err / tol.clamp_min(1e-300))[bad].max())} x the tolerance")


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Cache:
    """A pool whose unused slots and table entries hold what must not be read."""

    def __init__(self, g, dtype, lens, hk, d, page, wide=None, token_major=False, poison=True,
                 spare=0):
        need = [-(-n // page) for n in lens]
        wide = max(need + [1]) if wide is None else wide
        b, pool = len(lens), sum(need) + 2 + spare
        shape = (pool, page, hk, d) if token_major else (pool, hk, page, d)
        self.k, self.v = randn(g, *shape, dtype=dtype), randn(g, *shape, dtype=dtype)
        if token_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        ids = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
        self.table = torch.full((b, wide), -7 if poison else 0, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at: at + n]
            at += n
        self.spare = ids[at:]
        self.lens_list, self.page, self.hk, self.d, self.dtype = list(lens), page, hk, d, dtype
        self.lens = int32(lens)
        if poison:
            used = torch.zeros(pool, page, dtype=torch.bool, device=DEV)
            for i, n in enumerate(lens):
                p = torch.arange(n, device=DEV)
                used[self.table[i].long()[p // page], p % page] = True
            gone = ~used[:, None, :, None]
            self.k.masked_fill_(gone, float("nan"))
            self.v.masked_fill_(gone, float("inf"))
        self.kv = ops.PagedKV(self.k, self.v, self.table, self.lens)

    def rows(self, x, b, n=None, table=None):
        """[hk, n, d] rows of sequence b in 64 bits."""
        n = self.lens_list[b] if n is None else n
        p = torch.arange(n, device=DEV)
        t = (self.table if table is None else table)[b].long()
        return x[t[p // self.page], :, p % self.page].transpose(0, 1).double()


# ------------------------------------------------------- norm and rotation


def turn64(x, gamma, eps, cos, sin, pos, interleaved):
    """(value, magnitude its rounding errors are relative to) of [T, heads, d]."""
    y = x.double()
    if gamma is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
    if cos is None:
        return y, y.abs()
    half = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    a, b = y[..., ia], y[..., ib]
    out, mag = y.clone(), y.abs()
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = (a * c).abs() + (b * s).abs()
    mag[..., ib] = (b * c).abs() + (a * s).abs()
    return out, mag


def norm_tol(out, mag, d, dtype):
    return half_step(dtype) * out.abs() * (1 + 2.0 ** -7) + (d + 16) * U * mag + 2.0 ** -25


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,heads,hk,d,rot,interleaved", [
    (1, 12, 12, 64, 64, False), (3, 4, 1, 128, 128, True), (70, 5, 3, 128, 64, False),
    (9, 8, 2, 80, 20, False), (9, 8, 2, 80, 20, True), (5, 3, 3, 8, 8, False), (2, 1, 1, 256, 256,
    False), (6, 7, 7, 32, 8, False), (130, 2, 1, 96, 96, False), (4, 2, 2, 192, 48, True),
    (4, 1, 1, 256, 2, False), (1000, 33, 1, 40, 24, False)])
def test_norm_rotary(dtype, tokens, heads, hk, d, rot, interleaved):
    g = gen(tokens + heads * d + rot)
    packed = randn(g, tokens, (heads + 2 * hk) * d, dtype=dtype) * 3
    q = packed[:, : heads * d].view(tokens, heads, d)
    k = packed[:, heads * d: (heads + hk) * d].view(tokens, hk, d)
    cos, sin = ops.RotaryTable(5000, rot)
    pos = torch.randint(0, 5000, (tokens,), generator=g, device=DEV, dtype=torch.int32)
    gq, gk = 1 + 0.3 * randn(g, d), 1 + 0.3 * randn(g, d)
    for a, b, p in ((gq, gk, pos), (None, gk, pos), (gq, None, None), (None, None, pos)):
        at = torch.arange(tokens, device=DEV) if p is None else p.long()
        qo, ko = ops.QKNormRotary(q, k, a, b, 1e-5, cos, sin, p, interleaved)
        for got, x, gamma in ((qo, q, a), (ko, k, b)):
            want, mag = turn64(x, gamma, 1e-5, cos, sin, at, interleaved)
            close(got, want, norm_tol(want, mag, d, dtype))
    # norm alone, and in place into the packed rows
    want_q, mag_q = turn64(q, gq, 1e-5, None, None, None, False)
    want_k, mag_k = turn64(k, gk, 1e-5, cos, sin, pos.long(), interleaved)
    qo, ko = ops.QKNormRotary(q, k, gq, gk, 1e-5)
    close(qo, want_q, norm_tol(want_q, mag_q, d, dtype))
    rest = packed[:, (heads + hk) * d:].clone()
    got = ops.QKNormRotary(q, k, gq, gk, 1e-5, cos, sin, pos, interleaved, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(packed[:, (heads + hk) * d:], rest)
    close(k, want_k, norm_tol(want_k, mag_k, d, dtype))
    sync_ok()


def test_norm_rotary_positions_outside_the_table_are_reported():
    g = gen(0)
    q, k = randn(g, 4, 2, 64), randn(g, 4, 1, 64)
    cos, sin = ops.RotaryTable(10, 64)
    out = torch.full_like(q, 7.0)
    ops.QKNormRotary(q, k, None, None, 1e-6, cos, sin, int32([3, 10, -1, 9]), q_out=out)
    assert sync_code() == 5
    assert (out[1:3] == 7).all() and (out[[0, 3]] != 7).any()
    sync_ok()  # reported once


def test_norm_of_a_zero_row_is_zero_and_empty_calls_work():
    q = torch.zeros(2, 3, 64, device=DEV)
    qo, ko = ops.QKNormRotary(q, q, torch.ones(64, device=DEV), torch.ones(64, device=DEV), 1e-6)
    assert (qo == 0).all() and (ko == 0).all()
    e = torch.zeros(0, 3, 64, device=DEV)
    qo, ko = ops.QKNormRotary(e, e[:, :1])
    assert qo.shape == (0, 3, 64) and ko.shape == (0, 1, 64)
    qo, ko = ops.QKNormRotary(q, torch.zeros(2, 0, 64, device=DEV), torch.ones(64, device=DEV))
    assert (qo == 0).all() and ko.shape == (2, 0, 64)


# ------------------------------------------------------------------ append


@pytest.mark.parametrize("dtype,hk,d,page,token_major", [
    (F32, 3, 64, 16, False), (F16, 2, 128, 24, True), (BF16, 8, 128, 1, False),
    (BF16, 1, 80, 64, True), (F32, 5, 256, 7, False)])
def test_append_ragged(dtype, hk, d, page, token_major):
    g = gen(hk * d + page)
    news, lens = [0, 5, 1, 0, 33, 70], [9, 5, 100, 0, 40, 71]
    c = Cache(g, dtype, lens, hk, d, page, token_major=token_major, poison=False, spare=3)
    k0, v0 = c.k.clone(), c.v.clone()
    tokens = sum(news) + 4  # four padding rows behind the last sequence
    heads = 2 * hk
    packed = randn(g, tokens, (heads + 2 * hk) * d, dtype=dtype)
    q = packed[:, : heads * d].view(tokens, heads, d)
    k = packed[:, heads * d: (heads + hk) * d].view(tokens, hk, d)
    v = packed[:, (heads + hk) * d:].view(tokens, hk, d)
    cu = int32([0] + list(torch.tensor(news).cumsum(0)))
    cos, sin = ops.RotaryTable(200, d if d % 16 == 0 else d // 2)
    gq, gk = 1 + 0.3 * randn(g, d), 1 + 0.3 * randn(g, d)
    q_out = torch.full((tokens, heads, d), 5.0, device=DEV, dtype=dtype)
    ops.QKNormRotaryAppend(c.kv, q, k, v, gq, gk, 1e-6, cos, sin, None, False, cu, q_out)
    sync_ok()
    touched = torch.zeros(k0.shape[0], page, dtype=torch.bool, device=DEV)
    for b, (n, new) in enumerate(zip(lens, news)):
        rows = slice(int(cu[b]), int(cu[b + 1]))
        pos = torch.arange(n - new, n, device=DEV)
        touched[c.table[b].long()[pos // page], pos % page] = True
        want, mag = turn64(k[rows], gk, 1e-6, cos, sin, pos, False)
        close(c.rows(c.k, b)[:, n - new:].transpose(0, 1), want, norm_tol(want, mag, d, dtype))
        assert torch.equal(c.rows(c.v, b)[:, n - new:].transpose(0, 1), v[rows].double())
        want, mag = turn64(q[rows], gq, 1e-6, cos, sin, pos, False)
        close(q_out[rows], want, norm_tol(want, mag, d, dtype))
    assert (q_out[sum(news):] == 5).all()
    rest = ~touched[:, None, :, None]
    assert torch.equal(c.k.masked_fill(~rest, 0), k0.masked_fill(~rest, 0))
    assert torch.equal(c.v.masked_fill(~rest, 0), v0.masked_fill(~rest, 0))
    # the plain append of the same rows
    c.k.copy_(k0)
    ops.PagedKVAppend(c.kv, k, v, cu)
    for b, (n, new) in enumerate(zip(lens, news)):
        rows = slice(int(cu[b]), int(cu[b + 1]))
        assert torch.equal(c.rows(c.k, b)[:, n - new:].transpose(0, 1), k[rows].double())
    sync_ok()


@pytest.mark.parametrize("batch", [1, 33, 1100])
def test_append_one_each(batch):
    g = gen(batch)
    lens = [1 + (7 * i) % 50 for i in range(batch)]
    c = Cache(g, BF16, lens, 2, 64, 16, poison=False)
    k, v = randn(g, batch, 2, 64, dtype=BF16), randn(g, batch, 2, 64, dtype=BF16)
    last = (c.lens - 1).long()
    at = c.table.long()[torch.arange(batch, device=DEV), last // 16]
    for cu in (None, torch.arange(batch + 1, device=DEV, dtype=torch.int32)):
        c.k.zero_(), c.v.zero_()
        ops.PagedKVAppend(c.kv, k, v, cu)
        assert torch.equal(c.k[at, :, last % 16], k) and torch.equal(c.v[at, :, last % 16], v)
        assert float(c.k.double().abs().sum()) == pytest.approx(float(k.double().abs().sum()))
    sync_ok()


def test_append_skips_and_reports_what_points_outside():
    g = gen(1)
    c = Cache(g, F32, [5, 5, 5, 5], 1, 64, 4, poison=False)
    k0 = c.k.clone()
    rows = randn(g, 4, 1, 64)
    c.table[0, 1] = c.k.shape[0]  # a page past the pool
    c.table[1, 1] = -1
    c.lens[2] = 9                 # past the table's two pages
    c.lens[3] = -4
    ops.PagedKVAppend(c.kv, rows, rows)
    assert sync_code() == 5 and torch.equal(c.k[..., 1:, :], k0[..., 1:, :])
    c = Cache(g, F32, [5, 5], 1, 64, 4, poison=False)
    k0 = c.k.clone()
    ops.PagedKVAppend(c.kv, rows, rows, int32([0, 6, 4]))  # more new tokens than positions
    assert sync_code() == 5
    sync_ok()


# --------------------------------------------------------------- attention


def attend64(c, q, scale, b):
    """(out, tolerance, weights [hk, n], their tolerance) of sequence b."""
    n, hk, d, dtype = c.lens_list[b], c.hk, c.d, c.dtype
    group = q.shape[1] // hk
    k, v = c.rows(c.k, b), c.rows(c.v, b)
    qq = q[b].double().view(hk, group, d)
    if n == 0:
        z = torch.zeros(q.shape[1], d, dtype=torch.float64, device=DEV)
        return z, z, torch.zeros(hk, 0, device=DEV), torch.zeros(hk, 0, device=DEV)
    p = torch.softmax(scale * qq @ k.transpose(1, 2), -1)
    out = (p @ v).reshape(-1, d)
    size = abs(scale) * (qq.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True)
    e = 2 * size * ((d + 8) * 2 * U + 2.0 ** -20) + 2.0 ** -20
    pieces = 2.0 ** -21 if dtype == F32 else half_step(dtype) ** 2
    rel = e + (n + 64) * 2 * U + pieces
    mag = (p @ v.abs())
    tol = (rel * mag).reshape(-1, d) + half_step(dtype) * out.abs() * (1 + 2.0 ** -7) + \
        2.0 ** -25 + n * 2.0 ** -36 * float(v.abs().max())
    return out, tol, p.sum(1), (e * p).sum(1) + (group + 4) * 2 * U * p.sum(1)


def check_attention(c, q, weights=False, scale=None, out=None, repeat=False):
    s = c.d ** -0.5 if scale is None else scale
    w = torch.rand(len(c.lens_list), c.hk, c.kv.capacity + 3, generator=gen(3), device=DEV) \
        if weights else None
    w0 = None if w is None else w.clone()
    got = ops.PagedDecodeAttention(q, c.kv, scale, w, out)
    sync_ok()
    for b, n in enumerate(c.lens_list):
        want, tol, p, ptol = attend64(c, q, s, b)
        close(got[b], want, tol)
        if weights:
            sums = w0[b, :, :n].double() + p
            close(w[b, :, :n], sums, ptol + 2 * U * sums.abs())
            assert torch.equal(w[b, :, n:], w0[b, :, n:])
    if repeat:
        again = ops.PagedDecodeAttention(q, c.kv, scale, None if w is None else w0)
        assert torch.equal(again, got) and (w is None or torch.equal(w0, w))
    return got


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 129, 300]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hk,group,d,page,token_major", [
    (1, 1, 64, 16, False), (3, 1, 64, 16, True), (2, 4, 128, 16, False), (2, 8, 128, 64, True),
    (1, 16, 128, 32, False), (1, 17, 64, 16, False), (2, 3, 80, 24, True), (1, 5, 256, 8, False),
    (1, 40, 96, 16, False), (2, 2, 8, 1, False), (1, 7, 192, 5, True), (2, 1, 40, 128, False),
    (1, 9, 32, 3, False)])
def test_attention(dtype, hk, group, d, page, token_major):
    g = gen(hk * 1000 + group * 100 + d + page)
    c = Cache(g, dtype, LENS, hk, d, page, wide=max(2, 400 // page), token_major=token_major)
    h = hk * group
    packed = randn(g, len(LENS), (h + 2 * hk) * d, dtype=dtype)
    q = packed[:, : h * d].view(len(LENS), h, d)
    out = torch.full((len(LENS), h + 1, d), 9.0, device=DEV, dtype=dtype)
    got = check_attention(c, q, out=out[:, :h], repeat=True)
    assert got.data_ptr() == out.data_ptr() and (out[:, h] == 9).all()
    check_attention(c, q, weights=True, repeat=True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hk,group,d,page,token_major", [
    (1, 1, 64, 16, False), (3, 1, 96, 16, True), (2, 1, 128, 24, False), (2, 4, 128, 16, False),
    (2, 8, 64, 48, True), (1, 16, 128, 32, False), (1, 17, 64, 16, False), (2, 3, 80, 24, True),
    (1, 5, 256, 8, False), (1, 40, 96, 16, False), (2, 2, 8, 16, False), (1, 7, 192, 16, True),
    (1, 12, 256, 16, False), (2, 1, 24, 16, False), (1, 9, 32, 3, False), (1, 1, 200, 16, False)])
def test_attention_cut_among_warps(dtype, hk, group, d, page, token_major):
    """The same lengths in a table wide enough that sequences are cut wherever
    the warps' shares meet and joined by a second kernel."""
    g = gen(hk * 1000 + group * 100 + d + page)
    c = Cache(g, dtype, LENS + [1100], hk, d, page, wide=4000 // page, token_major=token_major)
    q = randn(g, len(LENS) + 1, hk * group, d, dtype=dtype)
    check_attention(c, q, repeat=True)
    check_attention(c, q, weights=True, repeat=True)


@pytest.mark.parametrize("seed", range(40))
def test_any_sizes(seed):
    """Attention, append and eviction at sizes drawn from the whole range."""
    r = random.Random(seed)
    dtype = r.choice([F32, F16, BF16])
    d, hk, group = 8 * r.randint(1, 32), r.randint(1, 6), r.choice([1, 1, 2, 3, 5, 8, 13, 20])
    page = r.choice([1, 3, 8, 16, 16, 24, 32, 48, 64, 160])
    lens = [r.choice([0, 1, r.randint(1, 40), r.randint(1, 900)]) for _ in range(r.randint(1, 9))]
    wide = max(-(-max(lens) // page), 1) + r.choice([0, 0, 1, 2000 // page])
    g = gen(seed)
    c = Cache(g, dtype, lens, hk, d, page, wide=wide, token_major=r.random() < 0.5, poison=True,
              spare=2)
    q = randn(g, len(lens), hk * group, d, dtype=dtype)
    check_attention(c, q, weights=r.random() < 0.5, repeat=True)
    keep = r.randint(1, max(max(lens), 1) + 3)
    w = torch.randint(0, 9, (len(lens), hk, c.kv.capacity), generator=g, device=DEV).float()
    dst = None
    if r.random() < 0.5:  # other pages
        n = -(-min(keep, c.kv.capacity) // page)
        extra = torch.zeros(len(lens) * n, *c.k.shape[1:], device=DEV, dtype=dtype)
        c.k, c.v = torch.cat([c.k, extra]), torch.cat([c.v, extra])
        dst = (torch.arange(len(lens) * n, device=DEV, dtype=torch.int32) + c.k.shape[0]
               - len(lens) * n).view(len(lens), n)
        c.kv = ops.PagedKV(c.k, c.v, c.table, c.lens)
    check_evict(c, w, keep, r.randint(0, keep), dst, in_place_weights=r.random() < 0.5)


def test_attention_without_pages_or_positions():
    for batch in (2, 400):
        k = torch.zeros(0, 1, 16, 64, device=DEV)
        for width in (0, 3):
            table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
            kv = ops.PagedKV(k, k, table, torch.zeros(batch, dtype=torch.int32, device=DEV))
            out = torch.full((batch, 2, 64), 7.0, device=DEV)
            ops.PagedDecodeAttention(torch.ones(batch, 2, 64, device=DEV), kv, out=out)
            sync_ok()
            assert (out == 0).all()


def test_overlapping_calls_on_two_streams():
    """Two batches of one pool, attended on two streams at once, many times."""
    g = gen(21)
    a = Cache(g, BF16, [900, 1500, 40], 4, 128, 16)
    b = Cache(g, F32, [700, 333], 2, 64, 16)
    qa, qb = randn(g, 3, 16, 128, dtype=BF16), randn(g, 2, 4, 64)
    want_a, want_b = ops.PagedDecodeAttention(qa, a.kv), ops.PagedDecodeAttention(qb, b.kv)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(30):
        for i, (q, c) in enumerate(((qa, a), (qb, b))):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.PagedDecodeAttention(q, c.kv))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want_a) for x in got[0])
    assert all(torch.equal(x, want_b) for x in got[1])


@pytest.mark.parametrize("dtype,hk,group,d,page", [(BF16, 4, 4, 128, 16), (F32, 12, 1, 64, 16),
                                                   (F16, 2, 20, 96, 24)])
def test_steps_without_waiting_equal_steps_with_waiting(dtype, hk, group, d, page):
    """Each kernel starts while the one before it drains; what it reads must
    still be that one's results: a run of steps queued at once, the lengths and
    tables changing in between, gives the bits of the same run with a wait behind
    every call."""
    def steps(wait):
        g = gen(33)
        lens = [1, 700, 260, 999]
        c = Cache(g, dtype, lens, hk, d, page, wide=-(-1100 // page), poison=False,
                  spare=4 * -(-1100 // page))
        need = torch.tensor([-(-n // page) for n in lens], device=DEV)
        free = c.spare[: c.table.numel()].view_as(c.table)
        c.table.copy_(torch.where(torch.arange(c.table.shape[1], device=DEV) < need[:, None],
                                  c.table, free))
        w = torch.zeros(4, hk, c.kv.capacity, device=DEV)
        cos, sin = ops.RotaryTable(4096, d)
        positions = c.lens.clone()
        gamma = 1 + 0.1 * randn(g, d)
        rows = [randn(g, 4, (group + 2) * hk, d, dtype=dtype) for _ in range(25)]
        outs = []
        torch.cuda.synchronize()
        for i, r in enumerate(rows):
            c.lens.add_(1)
            q = ops.QKNormRotaryAppend(c.kv, r[:, : group * hk], r[:, group * hk: (group + 1) * hk],
                                       r[:, (group + 1) * hk:], gamma, gamma, 1e-6, cos, sin,
                                       positions)
            wait()
            outs.append(ops.PagedDecodeAttention(q, c.kv, weights=w))
            wait()
            positions.add_(1)
            if i % 6 == 5:
                new, kept, _ = ops.PagedKVEvict(c.kv, w, 250 + i, 9)
                wait()
                c.lens.copy_(new)
                outs += [new, kept]
        torch.cuda.synchronize()
        return outs + [w, c.k, c.v]

    for a, b in zip(steps(lambda: None), steps(torch.cuda.synchronize)):
        assert torch.equal(a, b)
    sync_ok()


def test_first_calls_in_a_capture():
    """In a process of its own: the operators' first calls are captured."""
    code = (
        "import torch\n"
        "from inferc_b200 import ops\n"
        "k = torch.randn(20, 2, 16, 64, device='cuda'); v = torch.randn_like(k)\n"
        "t = torch.randperm(20, device='cuda')[:16].view(2, 8).int()\n"
        "lens = torch.tensor([100, 7], dtype=torch.int32, device='cuda')\n"
        "q = torch.randn(2, 4, 64, device='cuda'); w = torch.zeros(2, 2, 128, device='cuda')\n"
        "kv = ops.PagedKV(k, v, t, lens)\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    x, _ = ops.QKNormRotary(q, q, torch.ones(64, device='cuda'))\n"
        "    ops.PagedKVAppend(kv, q[:, :2], q[:, 2:])\n"
        "    o = ops.PagedDecodeAttention(x, kv, weights=w)\n"
        "    n, kept, _ = ops.PagedKVEvict(kv, w, 40, 4)\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "# four query heads' weights of each sequence add up to 4; the first loses some to eviction\n"
        "s = w.sum((1, 2)).tolist()\n"
        "assert n.tolist() == [40, 7] and abs(s[1] - 4) < 1e-4 and 0.5 < s[0] < 4, (n, s)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT, timeout=300)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens,hk,group,d,page", [
    ([1], 12, 1, 64, 16), ([160], 12, 1, 64, 16), ([5001], 2, 4, 128, 16), ([70001], 1, 8, 128, 64),
    ([1000, 3, 0, 4097, 77, 2500], 4, 4, 128, 32), ([33000], 1, 2, 256, 128),
    ([37] * 300, 2, 2, 64, 16), ([20000, 1, 1, 1, 1, 1, 1], 3, 1, 64, 16)])
def test_attention_long(dtype, lens, hk, group, d, page):
    g = gen(sum(lens) + d)
    c = Cache(g, dtype, lens, hk, d, page)
    q = randn(g, len(lens), hk * group, d, dtype=dtype)
    check_attention(c, q, repeat=True)
    check_attention(c, q, weights=True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_peaked_scores(dtype):
    """One position far above the rest, first, in the middle or last; and a
    scale of zero and a negative one."""
    for at in (0, 700, 1499):
        g = gen(at)
        c = Cache(g, dtype, [1500], 2, 64, 16)
        q = randn(g, 1, 4, 64, dtype=dtype)
        p = c.table[0].long()[at // 16]
        c.k[p, :, at % 16] = 12 * q[0, ::2]
        check_attention(c, q, weights=True)
        check_attention(c, q, scale=0.0)
        check_attention(c, q, scale=-0.25)
        check_attention(c, q, scale=1.0)


def test_attention_wide_table_short_sequences():
    """The table's width says nothing about the lengths; unused entries are not
    read (they name no page)."""
    g = gen(5)
    c = Cache(g, BF16, [3, 40, 0], 2, 128, 16, wide=5000)
    check_attention(c, randn(g, 3, 8, 128, dtype=BF16), weights=True, repeat=True)


def test_attention_shared_pages():
    g = gen(6)
    c = Cache(g, F16, [200, 200, 130], 2, 128, 16)
    c.table[1, :8] = c.table[0, :8]
    c.table[2] = c.table[0]
    check_attention(c, randn(g, 3, 4, 128, dtype=F16), weights=True, repeat=True)


def test_attention_reports_and_leaves_out_what_points_outside():
    g = gen(7)
    for dtype in (F32, F16):
        c = Cache(g, dtype, [64, 64, 64, 64], 2, 64, 16)
        q = randn(g, 4, 4, 64, dtype=dtype)
        c.table[0, 1] = -1               # positions 16..31 are left out
        c.table[1, 3] = c.k.shape[0]     # positions 48..63
        c.lens[2] = 65                   # past the table: clamped to 64
        c.lens[3] = -2                   # none
        got = ops.PagedDecodeAttention(q, c.kv)
        assert sync_code() == 5
        for b, keep in ((0, list(range(16)) + list(range(32, 64))), (1, list(range(48))),
                        (2, list(range(64)))):
            at = torch.tensor(keep, device=DEV)
            t = c.table[b].long()[at // 16]
            k = c.k[t, :, at % 16].transpose(0, 1).double()
            v = c.v[t, :, at % 16].transpose(0, 1).double()
            qq = q[b].double().view(2, 2, 64)
            p = torch.softmax(0.125 * qq @ k.transpose(1, 2), -1)
            want = (p @ v).reshape(4, 64)
            close(got[b], want, half_step(dtype) * want.abs() + 1e-4)
        assert (got[3] == 0).all()
    sync_ok()


def test_attention_offsets_past_32_bits():
    """Pages that lie beyond 2^32 elements into the pool."""
    g = gen(8)
    pages = (1 << 32) // (16 * 128) + 64
    k = torch.empty(pages, 1, 16, 128, dtype=F16, device=DEV)
    v = torch.empty_like(k)
    c = Cache(g, F16, [300, 17], 1, 128, 16)
    for i in range(c.table.shape[0]):
        for j in range(-(-c.lens_list[i] // 16)):
            to = pages - 1 - (i * 32 + j)
            k[to], v[to] = c.k[c.table[i, j]], c.v[c.table[i, j]]
            c.table[i, j] = to
    c.k, c.v = k, v
    c.kv = ops.PagedKV(k, v, c.table, c.lens)
    check_attention(c, randn(g, 2, 4, 128, dtype=F16), weights=True)
    rows = randn(g, 2, 1, 128, dtype=F16)
    ops.PagedKVAppend(c.kv, rows, rows)
    assert torch.equal(c.rows(c.k, 0)[:, -1], rows[0].double())
    w = torch.rand(2, 1, c.kv.capacity, generator=g, device=DEV)
    before = [c.rows(c.k, b) for b in range(2)]
    lens, kept, _ = ops.PagedKVEvict(c.kv, w, 40, 3)
    sync_ok()
    assert torch.equal(c.rows(c.k, 0, 40), before[0][:, kept[0, 0].long()])


def test_attention_refusals():
    g = gen(9)
    c = Cache(g, F32, [20, 3], 2, 64, 16)
    q = randn(g, 2, 4, 64)
    for bad in (q.half(), q[:1], q[:, :3], randn(g, 2, 4, 32), q.transpose(0, 1), q.cpu(),
                q.double(), randn(g, 2, 4, 128)[..., ::2]):
        with pytest.raises(RuntimeError):
            ops.PagedDecodeAttention(bad, c.kv)
    for w in (torch.zeros(2, 2, c.kv.capacity - 1, device=DEV), torch.zeros(2, 4, 99, device=DEV),
              torch.zeros(2, 2, 99, device=DEV, dtype=F16)):
        with pytest.raises(RuntimeError):
            ops.PagedDecodeAttention(q, c.kv, weights=w)
    with pytest.raises(RuntimeError):
        ops.PagedKV(c.k, c.v.half(), c.table, c.lens)
    with pytest.raises(RuntimeError):
        ops.PagedKV(c.k, c.v, c.table.long(), c.lens)
    with pytest.raises(RuntimeError):
        ops.PagedKV(c.k, c.v, c.table, c.lens[:1])
    with pytest.raises(RuntimeError):
        ops.PagedDecodeAttention(q, ops.PagedKV(c.k[..., :60], c.v[..., :60], c.table, c.lens))


def test_caches_without_heads_or_positions_are_refused():
    table, lens = int32([[0]]), int32([0])
    for shape in ((2, 0, 16, 64), (2, 2, 0, 64)):
        x = torch.zeros(shape, device=DEV)
        with pytest.raises(RuntimeError, match="at least"):
            ops.PagedKV(x, x.clone(), table, lens)


def test_a_view_keeps_its_tensors():
    c = Cache(gen(31), F32, [20, 3], 2, 64, 16)
    for name in ("lens", "page_table", "k", "v"):
        with pytest.raises(RuntimeError, match="fixed"):
            setattr(c.kv, name, getattr(c.kv, name).clone())
    c.kv.lens += 1
    assert c.lens.tolist() == [21, 4] and c.kv.lens is c.lens


# ---------------------------------------------------------------- eviction


def keep64(w, n, keep, recent):
    if n <= keep:
        return torch.arange(n, device=w.device)
    old = torch.where(w.isnan(), torch.inf, w.double())[: n - recent]
    # NaN above every number, infinity included
    order = sorted(range(n - recent), key=lambda j: (-1 if w[j].isnan() else 0, -float(old[j]), j))
    best = sorted(order[: keep - recent]) + list(range(n - recent, n))
    return torch.tensor(best, device=w.device, dtype=torch.long)


def check_evict(c, w, keep, recent, dst=None, in_place_weights=True, fast=False):
    w0, n_of = w.clone(), c.lens_list
    old = [(c.rows(c.k, b), c.rows(c.v, b)) for b in range(len(n_of))]
    w_out = None if in_place_weights else torch.full_like(w, 3.0)
    lens, kept, got_w = ops.PagedKVEvict(c.kv, w, keep, recent, dst, w_out)
    sync_ok()
    assert lens.tolist() == [min(n, keep) for n in n_of]
    for b, n in enumerate(n_of):
        m = min(n, keep)
        new_k, new_v = c.rows(c.k, b, m, dst), c.rows(c.v, b, m, dst)
        for h in range(c.hk):
            if fast and n > keep:  # distinct weights
                best = torch.topk(w0[b, h, : n - recent], keep - recent).indices.sort().values
                want = torch.cat([best, torch.arange(n - recent, n, device=DEV)])
            else:
                want = keep64(w0[b, h].cpu(), n, keep, recent).to(DEV)
            assert torch.equal(kept[b, h, :m].long(), want), (b, h)
            assert (kept[b, h, m:] == -1).all()
            assert torch.equal(new_k[h], old[b][0][h, want])
            assert torch.equal(new_v[h], old[b][1][h, want])
            assert torch.equal(got_w[b, h, :m].nan_to_num(nan=-5.0),
                               w0[b, h, want].nan_to_num(nan=-5.0))
            assert (got_w[b, h, m:n] == 0).all()
        rest = w0 if in_place_weights else torch.full_like(w0, 3.0)
        assert torch.equal(got_w[b, :, n:], rest[b, :, n:])


@pytest.mark.parametrize("dtype,hk,d,page,token_major", [
    (F32, 2, 64, 16, False), (F16, 3, 128, 5, True), (BF16, 1, 256, 32, False),
    (F32, 1, 256, 7, False), (BF16, 2, 8, 1, False), (F16, 1, 80, 24, True)])
@pytest.mark.parametrize("keep,recent", [(40, 8), (1, 0), (1, 1), (64, 0), (64, 64), (129, 1),
                                         (5000, 10)])
def test_evict(dtype, hk, d, page, token_major, keep, recent):
    g = gen(keep * 10 + recent + d)
    lens = [0, 1, 39, 40, 41, 64, 65, 130, 333]
    for dst in (False, True):
        c = Cache(g, dtype, lens, hk, d, page, token_major=token_major, poison=False,
                  spare=len(lens) * -(-keep // page) if dst else 0)
        # few distinct values, so that most choices are ties; zeros of both signs
        w = torch.randint(0, 4, (len(lens), hk, c.kv.capacity), generator=g, device=DEV).float()
        w = torch.where(w == 0, torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.5,
                                            -0.0, 0.0), w)
        table = c.spare[: len(lens) * -(-keep // page)].view(len(lens), -1).contiguous() \
            if dst else None
        check_evict(c, w, keep, recent, table, in_place_weights=not dst)


def test_evict_special_weights():
    g = gen(11)
    c = Cache(g, F32, [200, 150], 2, 64, 16, poison=False)
    w = randn(g, 2, 2, c.kv.capacity)
    w[0, 0, 5:60:7] = float("nan")
    w[0, 0, 61:100:9] = float("inf")
    w[0, 1, 3:150:5] = -float("inf")
    w[1, 0, 10:20] = 1e-42  # subnormal
    w[1, 1, :] = 0.25
    check_evict(c, w, 100, 10)


@pytest.mark.parametrize("lens,keep,recent", [([70001], 20000, 100), ([9000, 4097, 8192], 4096, 256),
                                              ([3001] * 40, 1500, 3)])
def test_evict_long(lens, keep, recent):
    g = gen(sum(lens))
    c = Cache(g, BF16, lens, 2, 64, 16, poison=False)
    w = torch.empty(len(lens), 2, c.kv.capacity, device=DEV)
    for b in range(len(lens)):
        for h in range(2):  # distinct weights
            w[b, h] = torch.randperm(c.kv.capacity, generator=g, device=DEV).float()
    check_evict(c, w, keep, recent, fast=True)


def test_evict_refusals_and_bad_pages():
    g = gen(12)
    c = Cache(g, F32, [50, 50], 1, 64, 16, poison=False)
    w = torch.rand(2, 1, 64, generator=g, device=DEV)
    with pytest.raises(RuntimeError, match="lens"):
        ops.PagedKVEvict(c.kv, w, 20, 4, lens_out=c.lens)
    for keep, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(RuntimeError):
            ops.PagedKVEvict(c.kv, w, keep, recent)
    with pytest.raises(RuntimeError, match="too small"):
        ops.PagedKVEvict(c.kv, w, 20, 4, dst_table=int32([[0], [1]]))
    c.table[0, 1] = 1000
    c.table[1, 0] = -3
    k0 = c.k.clone()
    lens, kept, _ = ops.PagedKVEvict(c.kv, w, 20, 4)
    assert sync_code() == 5 and lens.tolist() == [20, 20]
    sync_ok()
    assert c.k.shape == k0.shape


# -------------------------------------------------------------- all of them


def test_streams_and_graphs():
    """On a side stream; and captured into graphs that are replayed in turn
    with other lengths, pages and values than they were captured with."""
    g = gen(13)
    wide = 60
    c = Cache(g, BF16, [700, 33, 5], 2, 128, 16, wide=wide, poison=False, spare=3 * wide)
    q = randn(g, 3, 8, 128, dtype=BF16)
    rows = randn(g, 3, 2, 128, dtype=BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_attention(c, q, weights=True)
    torch.cuda.current_stream().wait_stream(side)
    w = torch.zeros(3, 2, c.kv.capacity, device=DEV)
    steps = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.PagedKVAppend(c.kv, rows, rows)
            out = ops.PagedDecodeAttention(q, c.kv, weights=w)
        steps.append((graph, out))
    trim = torch.cuda.CUDAGraph()
    with torch.cuda.graph(trim):
        new_lens, kept, _ = ops.PagedKVEvict(c.kv, w, 300, 20)
    for turn, lens in enumerate(([900, 10, 301], [1, 1, 960], [960, 960, 960], [16, 299, 300])):
        c.lens_list = lens
        c.lens.copy_(int32(lens))
        c.table.copy_(torch.randperm(c.k.shape[0], generator=g, device=DEV)[: 3 * wide]
                      .view(3, wide))
        c.k.copy_(randn(g, *c.k.shape, dtype=BF16))
        rows.copy_(randn(g, *rows.shape, dtype=BF16))
        q.copy_(randn(g, *q.shape, dtype=BF16))
        w.zero_()
        graph, out = steps[turn % 2]
        graph.replay()
        sync_ok()
        for b, n in enumerate(lens):
            assert torch.equal(c.rows(c.k, b)[:, -1], rows[b].double())
            want, tol, p, ptol = attend64(c, q, 128 ** -0.5, b)
            close(out[b], want, tol)
            close(w[b, :, :n], p, ptol + 2 * U * p)
        old = [c.rows(c.k, b) for b in range(3)]
        w0 = w.clone()
        trim.replay()
        sync_ok()
        assert new_lens.tolist() == [min(n, 300) for n in lens]
        for b, n in enumerate(lens):
            m = min(n, 300)
            for i in range(2):
                at = keep64(w0[b, i].cpu(), n, 300, 20).to(DEV)
                assert torch.equal(kept[b, i, :m].long(), at)
                assert torch.equal(c.rows(c.k, b, m)[i], old[b][i, at])


def test_serving_run():
    """Steps of a small server: queries and keys normed, rotated and appended,
    attention with running sums, and eviction back to a budget, against a
    64-bit model that keeps each head's rows in lists."""
    g = gen(15)
    hk, group, d, page, keep, recent, eps = 2, 3, 64, 8, 24, 6, 1e-6
    lens = [20, 1, 9, 26]
    c = Cache(g, F32, lens, hk, d, page, wide=5, poison=False, spare=20)
    for b in range(4):  # pages for 40 positions each
        need = -(-lens[b] // page)
        c.table[b, need:] = c.spare[b * 5: b * 5 + 5 - need]
    h = hk * group
    w = torch.zeros(4, hk, 40, device=DEV)
    model = [[(list(c.rows(c.k, b)[i]), list(c.rows(c.v, b)[i]), [0.0] * lens[b])
              for i in range(hk)] for b in range(4)]
    gq, gk = 1 + 0.2 * randn(g, d), 1 + 0.2 * randn(g, d)
    cos, sin = ops.RotaryTable(4096, d)
    positions = c.lens.clone()
    for step in range(20):
        packed = randn(g, 4, (h + 2 * hk) * d)
        q = packed[:, : h * d].view(4, h, d)
        k = packed[:, h * d: (h + hk) * d].view(4, hk, d)
        v = packed[:, (h + hk) * d:].view(4, hk, d)
        c.lens.add_(1)
        qn = ops.QKNormRotaryAppend(c.kv, q, k, v, gq, gk, eps, cos, sin, positions)
        out = ops.PagedDecodeAttention(qn, c.kv, weights=w)
        q64, _ = turn64(q, gq, eps, cos, sin, positions.long(), False)
        k64, _ = turn64(k, gk, eps, cos, sin, positions.long(), False)
        for b in range(4):
            for i in range(hk):
                ks, vs, ws = model[b][i]
                ks.append(k64[b, i]), vs.append(v[b, i].double()), ws.append(0.0)
                kk, vv = torch.stack(ks), torch.stack(vs)
                p = torch.softmax(q64[b, i * group: (i + 1) * group] @ kk.T * d ** -0.5, -1)
                # fp32 norm, rotation and attention: |out| < 3, each step's errors below 1e-5
                assert (out[b, i * group: (i + 1) * group].double() - p @ vv).abs().max() < 3e-5
                for j, x in enumerate(p.sum(0).tolist()):
                    ws[j] += x
        positions.add_(1)
        if step % 5 == 4:
            new, kept, _ = ops.PagedKVEvict(c.kv, w, keep, recent)
            for b in range(4):
                for i in range(hk):
                    ks, vs, ws = model[b][i]
                    n = len(ks)
                    if n > keep:
                        order = sorted(range(n - recent), key=lambda j: (-ws[j], j))
                        at = sorted(order[: keep - recent]) + list(range(n - recent, n))
                        model[b][i] = tuple([x[j] for j in at] for x in (ks, vs, ws))
                        assert kept[b, i].tolist() == at
            c.lens.copy_(new)
    sync_ok()
