"""A PagedKV view holds addresses: a tensor of it that gets other memory is
refused by every operator, and one that nothing else holds stays alive."""
import gc

import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import DEV, F32, Cache, check_attention, gen, randn

pytestmark = pytest.mark.gpu


def calls(c):
    g = gen(1)
    q, rows = randn(g, 2, 4, 64), randn(g, 2, 2, 64)
    w = torch.zeros(2, 2, c.kv.capacity, device=DEV)
    return [lambda: ops.PagedDecodeAttention(q, c.kv), lambda: ops.PagedKVAppend(c.kv, rows, rows),
            lambda: ops.QKNormRotaryAppend(c.kv, q, rows, rows), lambda: ops.PagedKVEvict(c.kv, w, 9)]


def data(t):
    t.data = t.clone()


def set_(t):
    t.set_(t.clone())


def shrink(t):
    t.untyped_storage().resize_(0)


@pytest.mark.parametrize("name", ["k", "v", "page_table", "lens"])
@pytest.mark.parametrize("replace", [data, set_, shrink])
def test_replaced_memory_is_refused(name, replace):
    c = Cache(gen(2), F32, [20, 3], 2, 64, 16)
    replace(getattr(c.kv, name))
    for call in calls(c):
        with pytest.raises(RuntimeError, match="was replaced"):
            call()


def test_a_view_keeps_its_memory():
    c = Cache(gen(3), F32, [200, 30], 2, 64, 16)
    q = randn(gen(4), 2, 4, 64)
    want = check_attention(c, q)
    k, v, table, lens = (x.clone() for x in (c.k, c.v, c.table, c.lens))
    kv = ops.PagedKV(k, v, table, lens)
    for name in ("k", "v", "page_table", "lens"):
        delattr(kv, name)
    del k, v, table, lens
    gc.collect()
    junk = [torch.full_like(c.k, 7.0), torch.full_like(c.v, 7.0), torch.full_like(c.table, 10 ** 6),
            torch.full_like(c.lens, 99)]
    assert torch.equal(ops.PagedDecodeAttention(q, kv), want)
    assert len(junk) == 4
