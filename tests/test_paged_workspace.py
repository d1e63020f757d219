"""The workspace size of a descriptor that the call refuses is -1, for each way a
descriptor can be wrong (CPU: nothing is followed)."""
import ctypes

import pytest

from inferc_b200 import lib
from tests.test_paged import BAD_KV, kv, message


@pytest.mark.parametrize("with_weights", [0, 1])
@pytest.mark.parametrize("over", BAD_KV, ids=lambda o: ",".join(map(str, o)))
def test_no_workspace_for_bad_descriptors(over, with_weights):
    size = lib.load().inferc_dev_paged_decode_attention_workspace
    assert size(ctypes.byref(kv()), 4, with_weights) >= 0
    assert size(ctypes.byref(kv(**over)), 4, with_weights) == -1 and message()
