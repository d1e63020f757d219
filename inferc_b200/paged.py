"""The paged cache of many requests and the operators on it, over device
tensors (inferc_dev_paged_*, inferc_dev_qk_norm_rotary). Re-exported by
inferc_b200.ops.

The reference keeps one dense cache per request, grown by Concat
(src/kernels/movement.cc:142-189, src/cli/main.cpp:831-836); these are the
batched forms a server needs. Checks raise RuntimeError as the other ops do;
an index found out of range on the device is reported by
inferc_dev_stream_synchronize (INFERC_ERR_RANGE) and never followed.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import lib as _lib
from .lib import HeadRotary as _Rotary
from .lib import PagedKv as _Kv

_DTYPES = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16}
_raw_stream = torch._C._cuda_getCurrentRawStream
_nothing = contextlib.nullcontext()


def _need(ok: bool, name: str, what: str) -> None:
    if not ok:
        raise RuntimeError(f"{name}: {what}")


def _on(device: torch.device):
    """The device's context, entered only when it is not the current one."""
    if device.index == torch.cuda.current_device():
        return _nothing
    return torch.cuda.device(device)


def _rows(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device,
          heads: int | None, dim: int, rows: int | None) -> tuple[int, int, int]:
    """(address, row stride, head stride) of a [rows, heads, dim] tensor."""
    if t.dtype != dtype or t.device != device:
        raise RuntimeError(f"{name}: {what} must be {dtype} on {device}")
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads) or \
            (rows is not None and t.shape[0] != rows):
        raise RuntimeError(f"{name}: {what} must be [{rows or 'rows'}, {heads or 'heads'}, {dim}],"
                           f" got {list(t.shape)}")
    a, b, c = t.stride()
    if c != 1:
        raise RuntimeError(f"{name}: the last dimension of {what} must be contiguous")
    return t.data_ptr(), a, b


def _ints(name: str, what: str, t: torch.Tensor, shape: tuple, device: torch.device) -> int:
    if t.dtype != torch.int32 or t.device != device or t.shape != shape or \
            not t.is_contiguous():
        raise RuntimeError(f"{name}: {what} must be a contiguous int32 tensor {list(shape)} on "
                           f"{device}")
    return t.data_ptr()


class PagedKV:
    """A batch's view of a paged cache; holds no data of its own.

    k_cache, v_cache: [pages, kv_heads, page, head_dim] of one floating type
    (any strides but the last, e.g. a transposed [pages, page, kv_heads,
    head_dim]); page_table: int32 [batch, max_pages]; lens: int32 [batch], the
    positions each sequence holds, tokens being appended by the current step
    included. The tensors are read when an operator runs, so they are updated
    in place between steps (lens.add_(1), new table entries) and must outlive
    the work queued on them."""

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 lens: torch.Tensor):
        n, dev = "PagedKV", k_cache.device
        _need(k_cache.is_cuda, n, "tensors must be on a CUDA device")
        _need(k_cache.dtype in _DTYPES, n, "caches must be float32, float16 or bfloat16")
        _need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape
              and v_cache.dtype == k_cache.dtype and v_cache.device == dev, n,
              "k_cache and v_cache must be alike, [pages, kv_heads, page, head_dim]")
        _need(k_cache.stride(3) == 1 and v_cache.stride(3) == 1, n,
              "the caches' last dimension must be contiguous")
        _need(page_table.dim() == 2 and page_table.dtype == torch.int32
              and page_table.device == dev
              and (page_table.shape[1] <= 1 or page_table.stride(1) == 1), n,
              "page_table must be int32 [batch, max_pages] with contiguous rows")
        _need(lens.dtype == torch.int32 and lens.device == dev and lens.dim() == 1
              and lens.shape[0] == page_table.shape[0] and lens.is_contiguous(), n,
              "lens must be a contiguous int32 tensor [batch]")
        self.k, self.v, self.page_table, self.lens = k_cache, v_cache, page_table, lens
        self.dtype, self.device = k_cache.dtype, dev
        pages, self.kv_heads, self.page, self.head_dim = k_cache.shape
        self.batch, self.max_pages = page_table.shape
        self.capacity = self.max_pages * self.page
        stride = max(page_table.stride(0), self.max_pages) if self.batch <= 1 else \
            page_table.stride(0)
        self.c = _Kv(k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
                     lens.data_ptr(), *k_cache.stride()[:3], *v_cache.stride()[:3], pages,
                     self.kv_heads, self.page, self.batch, self.max_pages, stride, self.head_dim,
                     _DTYPES[k_cache.dtype])
        self.ref = ctypes.byref(self.c)
        self._scratch: dict = {}

    def _workspace(self, q_heads: int, weights: bool) -> int:
        """Scratch bytes of one attention call (sizes only, so computed once)."""
        key = (q_heads, weights)
        if key not in self._scratch:
            got = _lib.load().inferc_dev_paged_decode_attention_workspace(self.ref, q_heads,
                                                                          int(weights))
            if got < 0:
                raise RuntimeError(_lib.load().inferc_dev_last_error_string().decode())
            self._scratch[key] = got
        return self._scratch[key]


def _weights(name: str, what: str, kv: PagedKV, w: torch.Tensor) -> tuple[int, int, int]:
    if w.dtype != torch.float32 or w.device != kv.device or w.dim() != 3 or \
            w.shape[0] != kv.batch or w.shape[1] != kv.kv_heads or w.shape[2] < kv.capacity or \
            (w.shape[2] > 1 and w.stride(2) != 1):
        raise RuntimeError(f"{name}: {what} must be float32 [{kv.batch}, {kv.kv_heads}, "
                           f">= {kv.capacity}] on {kv.device}, contiguous in its last dimension")
    return w.data_ptr(), w.stride(0), w.stride(1)


def _rotary(name: str, dev: torch.device, dim: int, tokens: int, q_gamma, k_gamma, eps: float,
            cos, sin, positions, interleaved: bool) -> _Rotary:
    gq = gk = c = s = p = None
    table_len = stride = rot = 0
    if q_gamma is not None:
        _need(q_gamma.dtype == torch.float32 and q_gamma.device == dev
              and q_gamma.shape == (dim,) and q_gamma.is_contiguous(), name,
              f"q_gamma must be float32 [{dim}] on {dev}")
        gq = q_gamma.data_ptr()
    if k_gamma is not None:
        _need(k_gamma.dtype == torch.float32 and k_gamma.device == dev
              and k_gamma.shape == (dim,) and k_gamma.is_contiguous(), name,
              f"k_gamma must be float32 [{dim}] on {dev}")
        gk = k_gamma.data_ptr()
    if (cos is None) != (sin is None):
        raise RuntimeError(f"{name}: cos and sin come together")
    if cos is not None:
        _need(cos.dim() == 2 and cos.dtype == torch.float32 and sin.dtype == torch.float32
              and cos.device == dev and sin.device == dev and cos.shape == sin.shape
              and cos.is_contiguous() and sin.is_contiguous(), name,
              "cos and sin must be contiguous float32 tables [positions, rotary_dim / 2]")
        table_len, half = cos.shape
        _need(half >= 1 and table_len >= 1 and 2 * half <= dim, name,
              "rotary_dim must be at most head_dim")
        c, s, stride, rot = cos.data_ptr(), sin.data_ptr(), half, 2 * half
        if positions is not None:
            p = _ints(name, "positions", positions, (tokens,), dev)
    return _Rotary(gq, gk, c, s, p, table_len, stride, eps, rot, int(interleaved))


def RotaryTable(positions: int, rotary_dim: int, base: float = 10000.0, device="cuda"
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), float32 [positions, rotary_dim / 2], of the angles
    p * base^(-2 i / rotary_dim), formed in 64 bits: in 32 an angle of position
    10^6 is off by a sixteenth of a radian."""
    _need(rotary_dim >= 2 and rotary_dim % 2 == 0 and positions >= 1, "RotaryTable",
          "rotary_dim must be even and positions at least 1")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * \
        base ** (-i / rotary_dim)
    return angle.cos().float(), angle.sin().float()


def QKNormRotary(q: torch.Tensor, k: torch.Tensor, q_gamma=None, k_gamma=None, eps: float = 1e-6,
                 cos=None, sin=None, positions=None, interleaved: bool = False, q_out=None,
                 k_out=None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head (gamma None: that side is left as
    it is) and its rotation by position in one pass. q [T, heads, d], k [T,
    kv_heads, d], e.g. column blocks of one projection; positions int32 [T]
    (None: 0..T-1). q_out / k_out may be q / k themselves."""
    name = "QKNormRotary"
    _need(q.is_cuda and q.dtype in _DTYPES and q.dim() == 3, name,
          "q must be [tokens, heads, head_dim], float32, float16 or bfloat16, on a CUDA device")
    tokens, heads, dim = q.shape
    dev, dt = q.device, q.dtype
    a = _rows(name, "q", q, dt, dev, None, dim, None)
    b = _rows(name, "k", k, dt, dev, None, dim, tokens)
    if q_out is None:
        q_out = torch.empty((tokens, heads, dim), dtype=dt, device=dev)
    if k_out is None:
        k_out = torch.empty((tokens, k.shape[1], dim), dtype=dt, device=dev)
    c = _rows(name, "q_out", q_out, dt, dev, heads, dim, tokens)
    e = _rows(name, "k_out", k_out, dt, dev, k.shape[1], dim, tokens)
    rot = _rotary(name, dev, dim, tokens, q_gamma, k_gamma, eps, cos, sin, positions, interleaved)
    with _on(dev):
        _lib.check(_lib.load().inferc_dev_qk_norm_rotary(
            ctypes.byref(rot), _DTYPES[dt], *a, *b, *c, *e, tokens, heads, k.shape[1], dim,
            _raw_stream(dev.index)))
    return q_out, k_out


def _cu(name: str, kv: PagedKV, cu_tokens, tokens: int):
    if cu_tokens is None:
        _need(tokens == kv.batch, name, "without cu_tokens there is one token per sequence")
        return None
    return _ints(name, "cu_tokens", cu_tokens, (kv.batch + 1,), kv.device)


def PagedKVAppend(kv: PagedKV, k: torch.Tensor, v: torch.Tensor,
                  cu_tokens: torch.Tensor | None = None) -> None:
    """Writes new rows k, v [T, kv_heads, d] as the last positions of their
    sequences: rows cu_tokens[b]..cu_tokens[b+1]-1 belong to sequence b (None:
    one row per sequence), whose lens count them already."""
    name = "PagedKVAppend"
    a = _rows(name, "k", k, kv.dtype, kv.device, kv.kv_heads, kv.head_dim, None)
    b = _rows(name, "v", v, kv.dtype, kv.device, kv.kv_heads, kv.head_dim, k.shape[0])
    cu = _cu(name, kv, cu_tokens, k.shape[0])
    with _on(kv.device):
        _lib.check(_lib.load().inferc_dev_paged_kv_append(
            kv.ref, None, None, 0, 0, *a, *b, None, 0, 0, 0, cu, k.shape[0],
            _raw_stream(kv.device.index)))


def QKNormRotaryAppend(kv: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       q_gamma=None, k_gamma=None, eps: float = 1e-6, cos=None, sin=None,
                       positions=None, interleaved: bool = False, cu_tokens=None,
                       q_out: torch.Tensor | None = None) -> torch.Tensor:
    """QKNormRotary of new rows with the keys and values going straight into
    the cache (PagedKVAppend); returns the queries. positions None: a token's
    slot in the cache (give them where earlier positions were evicted). Rows of
    q_out behind the last sequence are left as they are."""
    name = "QKNormRotaryAppend"
    dev, dt, dim = kv.device, kv.dtype, kv.head_dim
    a = _rows(name, "q", q, dt, dev, None, dim, None)
    tokens, heads = q.shape[0], q.shape[1]
    b = _rows(name, "k", k, dt, dev, kv.kv_heads, dim, tokens)
    c = _rows(name, "v", v, dt, dev, kv.kv_heads, dim, tokens)
    if q_out is None:
        q_out = torch.empty((tokens, heads, dim), dtype=dt, device=dev)
    e = _rows(name, "q_out", q_out, dt, dev, heads, dim, tokens)
    rot = _rotary(name, dev, dim, tokens, q_gamma, k_gamma, eps, cos, sin, positions, interleaved)
    cu = _cu(name, kv, cu_tokens, tokens)
    with _on(dev):
        _lib.check(_lib.load().inferc_dev_paged_kv_append(
            kv.ref, ctypes.byref(rot), *a, *b, *c, *e, heads, cu, tokens, _raw_stream(dev.index)))
    return q_out


def PagedDecodeAttention(q: torch.Tensor, kv: PagedKV, scale: float | None = None,
                         weights: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [batch, heads, d], over the
    positions its sequence holds; heads is a multiple of kv_heads (query head h
    reads key head h // (heads / kv_heads)); scale None: d ** -0.5. A sequence
    of length 0 gives zeros. weights: float32 [batch, kv_heads, >= max_pages *
    page], to which each position's softmax weight is added, summed over the
    query heads of its key head."""
    name = "PagedDecodeAttention"
    dev, dt, dim = kv.device, kv.dtype, kv.head_dim
    a = _rows(name, "q", q, dt, dev, None, dim, kv.batch)
    heads = q.shape[1]
    _need(heads >= 1 and heads % kv.kv_heads == 0, name,
          "the query heads must be a multiple of kv_heads")
    if out is None:
        out = torch.empty((kv.batch, heads, dim), dtype=dt, device=dev)
    b = _rows(name, "out", out, dt, dev, heads, dim, kv.batch)
    w = (None, 0, 0) if weights is None else _weights(name, "weights", kv, weights)
    size = kv._workspace(heads, weights is not None)
    with _on(dev):
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _lib.check(_lib.load().inferc_dev_paged_decode_attention(
            kv.ref, *a, heads, dim ** -0.5 if scale is None else scale, *b, *w,
            ws.data_ptr() if size else None, size, _raw_stream(dev.index)))
    return out


def PagedKVEvict(kv: PagedKV, weights: torch.Tensor, keep: int, recent: int = 0,
                 dst_table: torch.Tensor | None = None, weights_out: torch.Tensor | None = None,
                 lens_out: torch.Tensor | None = None, kept: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Trims every sequence longer than `keep` to `keep` positions per key head:
    its last `recent`, and of the others those with the largest weight (ties: the
    lower position). They move to the front in their order, in keys, values and
    weights. dst_table: int32 [batch, pages] of pages to put the result into
    (None: the sequence's own, which no other sequence may share); weights_out:
    like weights (None: in place). Returns (lens_out, kept, weights_out): the
    new lengths, a tensor apart from kv.lens; the old positions, int32 [batch,
    kv_heads, keep], -1 behind the last; and the weights."""
    name = "PagedKVEvict"
    dev = kv.device
    _need(keep >= 1 and 0 <= recent <= keep, name,
          "keep must be at least 1 and recent in [0, keep]")
    w = _weights(name, "weights", kv, weights)
    wo = (None, 0, 0)
    if weights_out is None:
        weights_out = weights
    else:
        wo = _weights(name, "weights_out", kv, weights_out)
    dst = (None, 0, 0)
    if dst_table is not None:
        _need(dst_table.dtype == torch.int32 and dst_table.device == dev and dst_table.dim() == 2
              and dst_table.shape[0] == kv.batch
              and (dst_table.shape[1] <= 1 or dst_table.stride(1) == 1), name,
              "dst_table must be int32 [batch, pages] with contiguous rows")
        pages = dst_table.shape[1]
        dst = (dst_table.data_ptr(), pages,
               max(dst_table.stride(0), pages) if kv.batch <= 1 else dst_table.stride(0))
    if lens_out is None:
        lens_out = torch.empty((kv.batch,), dtype=torch.int32, device=dev)
    if kept is None:
        kept = torch.empty((kv.batch, kv.kv_heads, keep), dtype=torch.int32, device=dev)
    a = _ints(name, "lens_out", lens_out, (kv.batch,), dev)
    b = _ints(name, "kept", kept, (kv.batch, kv.kv_heads, keep), dev)
    with _on(dev):
        _lib.check(_lib.load().inferc_dev_paged_kv_evict(
            kv.ref, *dst, *w, *wo, keep, recent, a, b, _raw_stream(dev.index)))
    return lens_out, kept, weights_out
