"""Eviction where pages of a table are no pages: rows from or to them are not
moved, the others are, nothing else is written, and it is reported."""
import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import (BF16, DEV, F32, Cache, gen, int32, keep64, sync_code, sync_ok)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hk,d,page", [(F32, 1, 64, 16), (BF16, 3, 128, 16), (F32, 2, 256, 7)])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("lens,keep,recent", [([50, 50], 20, 4), ([900, 333, 20], 300, 7)])
def test_rows_of_bad_pages_stay(dtype, hk, d, page, apart, lens, keep, recent):
    g = gen(sum(lens) + d)
    need = -(-keep // page)
    c = Cache(g, dtype, lens, hk, d, page, poison=False, spare=len(lens) * need if apart else 0)
    pages = c.k.shape[0]
    dst = c.spare[: len(lens) * need].view(-1, need).contiguous() if apart else None
    c.table[0, 1] = pages + 900
    c.table[1, 0] = -3
    c.table[1, 2] = pages
    if apart:
        dst[0, 0] = -1
    w = torch.randint(0, 30, (len(lens), hk, c.kv.capacity), generator=g, device=DEV).float()
    k0, v0, w0 = c.k.clone(), c.v.clone(), w.clone()
    want_k, want_v, want_w = k0.clone(), v0.clone(), w0.clone()
    kept_want = torch.full((len(lens), hk, keep), -1, dtype=torch.int32, device=DEV)
    to_table = (dst if apart else c.table).cpu().tolist()
    from_table = c.table.cpu().tolist()
    for b, n in enumerate(lens):
        for h in range(hk):
            at = keep64(w0[b, h].cpu(), n, keep, recent).tolist()
            kept_want[b, h, : len(at)] = int32(at)
            want_w[b, h, :n] = 0
            want_w[b, h, : len(at)] = w0[b, h, torch.tensor(at, device=DEV)]
            for i, j in enumerate(at):
                src, to = from_table[b][j // page], to_table[b][i // page]
                if 0 <= src < pages and 0 <= to < pages:
                    want_k[to, h, i % page] = k0[src, h, j % page]
                    want_v[to, h, i % page] = v0[src, h, j % page]
    sync_ok()
    got_lens, kept, _ = ops.PagedKVEvict(c.kv, w, keep, recent, dst)
    assert sync_code() == 5
    assert got_lens.tolist() == [min(n, keep) for n in lens]
    assert torch.equal(kept, kept_want) and torch.equal(w, want_w)
    assert torch.equal(c.k, want_k) and torch.equal(c.v, want_v)
    sync_ok()
