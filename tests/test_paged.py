"""CPU checks of the paged-cache entry points: every refusal happens on the
host, before anything touches a device, so descriptors with made-up addresses
can be used; empty calls succeed without a device."""
import ctypes

import pytest
import torch

from inferc_b200 import lib, ops

A = 1 << 20  # a 16-byte aligned address that is never followed
INVALID = 1


def kv(**over):
    """A valid descriptor: 4 sequences, 2 key heads of 64, pages of 16."""
    d = dict(k=A, v=A, page_table=A, lens=A, k_page_stride=2048, k_head_stride=1024,
             k_token_stride=64, v_page_stride=2048, v_head_stride=1024, v_token_stride=64,
             num_pages=100, kv_heads=2, page_size=16, batch=4, max_pages=8, table_stride=8,
             head_dim=64, dtype=1)
    d.update(over)
    return lib.PagedKv(**d)


def rot(**over):
    d = dict(q_gamma=A, k_gamma=A, cos=A, sin=A, positions=None, table_len=64, table_stride=32,
             eps=1e-6, rotary_dim=64, interleaved=0)
    d.update(over)
    return lib.HeadRotary(**d)


def attend(k, q_heads=4, q=A, out=A, stride=64, ws=A, size=1 << 40, weights=None):
    return lib.load().inferc_dev_paged_decode_attention(
        ctypes.byref(k) if k else None, q, 256, stride, q_heads, 0.125, out, 256, 64, weights, 256,
        128, ws, size, None)


def append(k, r=None, q_heads=0, kn=A, vn=A, cu=None, tokens=4, stride=128):
    return lib.load().inferc_dev_paged_kv_append(
        ctypes.byref(k), ctypes.byref(r) if r else None, A, 256, 64, kn, stride, 64, vn, 128, 64,
        A, 256, 64, q_heads, cu, tokens, None)


def norm(r, dtype=1, dim=64, q=A, tokens=3, q_heads=2, kv_heads=2, stride=128):
    return lib.load().inferc_dev_qk_norm_rotary(
        ctypes.byref(r) if r else None, dtype, q, stride, 64, A, 128, 64, A, 128, 64, A, 128, 64,
        tokens, q_heads, kv_heads, dim, None)


def evict(k, keep=32, recent=8, dst=None, dst_pages=0, w=A, lens=2 * A, kept=A, w_out=None):
    return lib.load().inferc_dev_paged_kv_evict(
        ctypes.byref(k), dst, dst_pages, dst_pages, w, 256, 128, w_out, 256, 128, keep, recent,
        lens, kept, None)


def message():
    return lib.load().inferc_dev_last_error_string().decode()


BAD_KV = [dict(head_dim=60), dict(head_dim=0), dict(head_dim=264), dict(dtype=2), dict(k=None),
          dict(v=A + 8), dict(k_token_stride=62), dict(v_head_stride=1023), dict(k_page_stride=1),
          dict(kv_heads=0), dict(page_size=0), dict(batch=-1), dict(table_stride=7),
          dict(lens=None), dict(page_table=None), dict(num_pages=-1), dict(num_pages=1 << 31),
          dict(page_size=1 << 16, max_pages=1 << 15, table_stride=1 << 15),
          dict(page_size=(1 << 30) + 16, max_pages=1), dict(batch=(1 << 20) + 1)]


@pytest.mark.parametrize("over", BAD_KV, ids=lambda o: ",".join(map(str, o)))
def test_bad_cache_descriptors_are_refused(over):
    for call in (attend, append, evict):
        assert call(kv(**over)) == INVALID, call
        assert message()
    assert lib.load().inferc_dev_paged_decode_attention_workspace(
        ctypes.byref(kv(**over)), 4, 1) == -1 or "k" in over or "v" in over or any(
            s in "".join(over) for s in ("lens", "table", "stride"))


def test_attention_refusals():
    assert attend(None) == INVALID
    for over in (dict(q_heads=0), dict(q_heads=3), dict(q=None), dict(q=A + 4), dict(out=None),
                 dict(stride=66 - 1)):
        assert attend(kv(), **over) == INVALID, over
    need = lib.load().inferc_dev_paged_decode_attention_workspace(ctypes.byref(kv()), 4, 1)
    assert need > 0
    # weights of more positions than any device has room for (2^20 sequences of 2^30)
    huge = kv(page_size=1 << 20, max_pages=1 << 10, table_stride=1 << 10, batch=1 << 20)
    assert attend(huge, weights=A) == INVALID and "weights" in message()
    assert lib.load().inferc_dev_paged_decode_attention_workspace(ctypes.byref(huge), 4, 1) == -1
    assert lib.load().inferc_dev_paged_decode_attention_workspace(ctypes.byref(huge), 4, 0) > 0
    assert attend(kv(), weights=A, size=need - 1) == INVALID
    assert attend(kv(), weights=A, size=need, ws=None) == INVALID
    assert attend(kv(), weights=A, size=need, ws=A + 8) == INVALID
    assert "workspace" in message()


def test_append_refusals():
    assert append(kv(), tokens=3) == INVALID and "one token per sequence" in message()
    assert append(kv(), tokens=-1, cu=A) == INVALID
    assert append(kv(), kn=None) == INVALID
    assert append(kv(), vn=A + 2) == INVALID
    assert append(kv(), stride=127) == INVALID
    assert append(kv(), q_heads=2) == INVALID  # queries without a norm or rotation
    for over in (dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=-2), dict(cos=None),
                 dict(table_len=0), dict(table_stride=31), dict(eps=-1.0)):
        assert append(kv(), rot(**over)) == INVALID, over
        assert norm(rot(**over)) == INVALID, over


def test_norm_refusals():
    assert norm(None) == INVALID
    for over in (dict(dtype=11), dict(dim=68), dict(dim=512), dict(q=None), dict(tokens=-1),
                 dict(q_heads=-1), dict(kv_heads=1 << 17), dict(stride=126)):
        assert norm(rot(), **over) == INVALID, over


def test_evict_refusals():
    for over in (dict(keep=0), dict(recent=-1), dict(recent=33), dict(w=None), dict(kept=None),
                 dict(lens=None), dict(lens=A), dict(lens=A + 12), dict(lens=A - 12),
                 dict(dst=A + 4, dst_pages=1), dict(keep=(1 << 30) + 1), dict(keep=1 << 32)):
        assert evict(kv(), **over) == INVALID, over


def test_written_rows_that_overlap_are_refused():
    """Broadcast or interleaved outputs would get the values of several rows."""
    L = lib.load()
    c = kv()

    def attend_to(batch=256, head=64, w=None, wb=256, wh=128, d=c):
        return L.inferc_dev_paged_decode_attention(ctypes.byref(d), A, 256, 64, 4, 0.125, A, batch,
                                                   head, w, wb, wh, None, 0, None)

    for over in (dict(batch=0), dict(head=0), dict(head=60), dict(batch=252), dict(batch=64),
                 dict(batch=-64), dict(w=A, wb=0), dict(w=A, wh=0), dict(w=A, wh=127),
                 dict(w=A, wb=255)):
        assert attend_to(**over) == INVALID and "overlap" in message(), over
    # rows apart, head-major or with single rows: refused for the missing workspace alone
    long = kv(max_pages=128, table_stride=128)
    for over in (dict(batch=64, head=256, d=long), dict(w=A, wb=128, wh=512),
                 dict(batch=-256, d=long), dict(batch=0, w=A, wb=0, d=kv(batch=1))):
        assert attend_to(**over) == INVALID and "workspace" in message(), over
    for over in (dict(k_page_stride=0), dict(v_head_stride=0), dict(k_token_stride=0),
                 dict(v_page_stride=2048 - 64)):
        for call in (append, evict):
            assert call(kv(**over)) == INVALID and "overlap" in message(), (over, call)

    def norm_to(q=128, k=128, kh=64):
        return L.inferc_dev_qk_norm_rotary(ctypes.byref(rot()), 1, A, 128, 64, A, 128, 64, A, q, 64,
                                           A, k, kh, 3, 2, 2, 64, None)

    for over in (dict(q=0), dict(q=64), dict(k=124), dict(kh=0)):
        assert norm_to(**over) == INVALID and "overlap" in message(), over
    assert L.inferc_dev_paged_kv_append(
        ctypes.byref(kv()), ctypes.byref(rot()), A, 256, 64, A, 128, 64, A, 128, 64, A, 0, 64, 4,
        None, 4, None) == INVALID and "overlap" in message()

    def evict_to(w_out=None, wb=256, wh=128, dst=None, dst_stride=8):
        return L.inferc_dev_paged_kv_evict(ctypes.byref(kv()), dst, 8, dst_stride, A, 256, 128,
                                           w_out, wb, wh, 32, 8, 2 * A, A, None)

    for over in (dict(w_out=A + 64, wb=0), dict(w_out=A + 64, wh=64)):
        assert evict_to(**over) == INVALID and "overlap" in message(), over
    # the same place read and written in different orders
    assert evict_to(w_out=A, wb=128, wh=512) == INVALID and "other strides" in message()
    assert evict_to(dst=A, dst_stride=16) == INVALID and "another stride" in message()


def test_empty_calls_do_nothing():
    none = kv(batch=0)
    assert attend(none) == 0 and evict(none) == 0 and append(none, tokens=0) == 0
    assert norm(rot(), tokens=0) == 0


def test_python_checks_want_device_tensors():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.PagedKV(torch.zeros(2, 2, 16, 64), torch.zeros(2, 2, 16, 64),
                    torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.QKNormRotary(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64))


def test_rotary_table_is_formed_in_64_bits():
    c, s = ops.RotaryTable(1_000_001, 4, 10000.0, device="cpu")
    assert c.shape == (1_000_001, 2) and c.dtype == torch.float32
    # cos and sin of 10^6 and of 10^4 radians
    assert c[1_000_000, 0] == pytest.approx(0.93675212753314, abs=1e-7)
    assert s[1_000_000, 0] == pytest.approx(-0.34999350217129, abs=1e-7)
    assert s[1_000_000, 1] == pytest.approx(-0.30561438888825, abs=1e-7)
    with pytest.raises(RuntimeError):
        ops.RotaryTable(4, 3, device="cpu")
