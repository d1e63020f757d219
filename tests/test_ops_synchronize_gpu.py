"""ops.Synchronize: what kernels could not report when they were queued reaches a
Python caller as an InfercError, once, on whichever stream the work was."""
import pytest
import torch

from inferc_b200 import ops
from tests.test_paged_gpu import DEV, F32, Cache, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own_stream", [False, True])
def test_a_page_out_of_range_raises(own_stream):
    ops.Synchronize()
    c = Cache(gen(1), F32, [40, 40], 2, 64, 16)
    q = randn(gen(2), 2, 4, 64)
    c.table[1, 1] = c.k.shape[0]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if own_stream else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        ops.PagedDecodeAttention(q, c.kv)
    with pytest.raises(ops.InfercError, match="out of range") as e:
        ops.Synchronize(stream if own_stream else None)
    assert e.value.code == 5
    ops.Synchronize()
    c.table[1, 1] = c.table[1, 0]
    ops.PagedDecodeAttention(q, c.kv)
    ops.Synchronize()
