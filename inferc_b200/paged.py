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

import ctypes

import torch

from . import lib as _lib
from .lib import HeadRotary as _Rotary
from .lib import PagedKv as _Kv

_DTYPES = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16}
_F32, _I32 = torch.float32, torch.int32
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_call = _lib.load  # the library, loaded on first use

# These functions run once per layer and step, so their checks read each
# attribute once and build no message before it is needed.


def _run(dev: int, fn, *args) -> None:
    """Calls an entry point on the tensors' device and its current stream."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        _lib.check(rc)


def _rows(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, dev: int,
          heads: int | None, dim: int, rows: int | None) -> tuple[int, int, int]:
    """(address, row stride, head stride) of a [rows, heads, dim] tensor."""
    if t.dtype is not dtype or t.get_device() != dev:
        raise RuntimeError(f"{name}: {what} must be {dtype} on CUDA device {dev}")
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads) or \
            (rows is not None and shape[0] != rows):
        raise RuntimeError(f"{name}: {what} must be [{'rows' if rows is None else rows}, "
                           f"{'heads' if heads is None else heads}, {dim}], got {list(shape)}")
    a, b, c = t.stride()
    if c != 1:
        raise RuntimeError(f"{name}: the last dimension of {what} must be contiguous")
    return t.data_ptr(), a, b


def _flat(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple,
          dev: int) -> int:
    """Address of a contiguous tensor of the given type and shape."""
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape or \
            not t.is_contiguous():
        raise RuntimeError(f"{name}: {what} must be a contiguous {dtype} tensor {list(shape)} on "
                           f"CUDA device {dev}")
    return t.data_ptr()


def _need(ok: bool, name: str, what: str) -> None:
    if not ok:
        raise RuntimeError(f"{name}: {what}")


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
        self.dtype, self.dev = k_cache.dtype, k_cache.get_device()
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
        got = self._scratch.get((q_heads, weights))
        if got is None:
            got = _call().inferc_dev_paged_decode_attention_workspace(self.ref, q_heads,
                                                                      int(weights))
            if got < 0:
                raise RuntimeError(_call().inferc_dev_last_error_string().decode())
            self._scratch[(q_heads, weights)] = got
        return got


def _weights(name: str, what: str, kv: PagedKV, w: torch.Tensor) -> tuple[int, int, int]:
    shape, (a, b, c) = w.shape, w.stride() if w.dim() == 3 else (0, 0, 0)
    if w.dtype is not _F32 or w.get_device() != kv.dev or len(shape) != 3 or \
            shape[0] != kv.batch or shape[1] != kv.kv_heads or shape[2] < kv.capacity or \
            (shape[2] > 1 and c != 1):
        raise RuntimeError(f"{name}: {what} must be float32 [{kv.batch}, {kv.kv_heads}, "
                           f">= {kv.capacity}] on CUDA device {kv.dev}, contiguous in its last "
                           "dimension")
    return w.data_ptr(), a, b


def _rotary(name: str, dev: int, dim: int, tokens: int, q_gamma, k_gamma, eps: float, cos, sin,
            positions, interleaved: bool) -> _Rotary:
    gq = gk = c = s = p = None
    table_len = half = 0
    if q_gamma is not None:
        gq = _flat(name, "q_gamma", q_gamma, _F32, (dim,), dev)
    if k_gamma is not None:
        gk = _flat(name, "k_gamma", k_gamma, _F32, (dim,), dev)
    if cos is not None and sin is not None:
        shape = cos.shape
        if len(shape) != 2 or shape[0] < 1 or not 1 <= shape[1] <= dim // 2:
            raise RuntimeError(f"{name}: cos and sin must be [positions, rotary_dim / 2], with "
                               "rotary_dim at most head_dim")
        table_len, half = shape
        c = _flat(name, "cos", cos, _F32, shape, dev)
        s = _flat(name, "sin", sin, _F32, shape, dev)
        if positions is not None:
            p = _flat(name, "positions", positions, _I32, (tokens,), dev)
    elif cos is not None or sin is not None:
        raise RuntimeError(f"{name}: cos and sin come together")
    return _Rotary(gq, gk, c, s, p, table_len, half, eps, 2 * half, interleaved)


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
    dt, dev, shape = q.dtype, q.get_device(), q.shape
    if dev < 0 or dt not in _DTYPES or len(shape) != 3:
        raise RuntimeError(f"{name}: q must be [tokens, heads, head_dim], float32, float16 or "
                           "bfloat16, on a CUDA device")
    tokens, heads, dim = shape
    a = _rows(name, "q", q, dt, dev, None, dim, None)
    b = _rows(name, "k", k, dt, dev, None, dim, tokens)
    kv_heads = k.shape[1]
    if q_out is None:
        q_out = q.new_empty(shape)
        c = (q_out.data_ptr(), heads * dim, dim)
    else:
        c = _rows(name, "q_out", q_out, dt, dev, heads, dim, tokens)
    if k_out is None:
        k_out = k.new_empty((tokens, kv_heads, dim))
        e = (k_out.data_ptr(), kv_heads * dim, dim)
    else:
        e = _rows(name, "k_out", k_out, dt, dev, kv_heads, dim, tokens)
    rot = _rotary(name, dev, dim, tokens, q_gamma, k_gamma, eps, cos, sin, positions, interleaved)
    _run(dev, _call().inferc_dev_qk_norm_rotary, ctypes.byref(rot), _DTYPES[dt], *a, *b, *c, *e,
         tokens, heads, kv_heads, dim)
    return q_out, k_out


def _cu(name: str, kv: PagedKV, cu_tokens, tokens: int):
    if cu_tokens is None:
        _need(tokens == kv.batch, name, "without cu_tokens there is one token per sequence")
        return None
    return _flat(name, "cu_tokens", cu_tokens, _I32, (kv.batch + 1,), kv.dev)


def PagedKVAppend(kv: PagedKV, k: torch.Tensor, v: torch.Tensor,
                  cu_tokens: torch.Tensor | None = None) -> None:
    """Writes new rows k, v [T, kv_heads, d] as the last positions of their
    sequences: rows cu_tokens[b]..cu_tokens[b+1]-1 belong to sequence b (None:
    one row per sequence), whose lens count them already."""
    name = "PagedKVAppend"
    a = _rows(name, "k", k, kv.dtype, kv.dev, kv.kv_heads, kv.head_dim, None)
    tokens = k.shape[0]
    b = _rows(name, "v", v, kv.dtype, kv.dev, kv.kv_heads, kv.head_dim, tokens)
    cu = _cu(name, kv, cu_tokens, tokens)
    _run(kv.dev, _call().inferc_dev_paged_kv_append, kv.ref, None, None, 0, 0, *a, *b, None, 0, 0,
         0, cu, tokens)


def QKNormRotaryAppend(kv: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       q_gamma=None, k_gamma=None, eps: float = 1e-6, cos=None, sin=None,
                       positions=None, interleaved: bool = False, cu_tokens=None,
                       q_out: torch.Tensor | None = None) -> torch.Tensor:
    """QKNormRotary of new rows with the keys and values going straight into
    the cache (PagedKVAppend); returns the queries. positions None: a token's
    slot in the cache (give them where earlier positions were evicted). Rows of
    q_out behind the last sequence are left as they are."""
    name = "QKNormRotaryAppend"
    dev, dt, dim = kv.dev, kv.dtype, kv.head_dim
    a = _rows(name, "q", q, dt, dev, None, dim, None)
    tokens, heads, _ = q.shape
    b = _rows(name, "k", k, dt, dev, kv.kv_heads, dim, tokens)
    c = _rows(name, "v", v, dt, dev, kv.kv_heads, dim, tokens)
    if q_out is None:
        q_out = q.new_empty((tokens, heads, dim))
        e = (q_out.data_ptr(), heads * dim, dim)
    else:
        e = _rows(name, "q_out", q_out, dt, dev, heads, dim, tokens)
    rot = _rotary(name, dev, dim, tokens, q_gamma, k_gamma, eps, cos, sin, positions, interleaved)
    cu = _cu(name, kv, cu_tokens, tokens)
    _run(dev, _call().inferc_dev_paged_kv_append, kv.ref, ctypes.byref(rot), *a, *b, *c, *e, heads,
         cu, tokens)
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
    dev, dt, dim, batch = kv.dev, kv.dtype, kv.head_dim, kv.batch
    a = _rows(name, "q", q, dt, dev, None, dim, batch)
    heads = q.shape[1]
    if heads < 1 or heads % kv.kv_heads:
        raise RuntimeError(f"{name}: the query heads must be a multiple of kv_heads")
    if out is None:
        out = q.new_empty((batch, heads, dim))
        b = (out.data_ptr(), heads * dim, dim)
    else:
        b = _rows(name, "out", out, dt, dev, heads, dim, batch)
    w = (None, 0, 0) if weights is None else _weights(name, "weights", kv, weights)
    size = kv._workspace(heads, weights is not None)
    # scratch of this call alone, in stream order, so that calls on other streams may overlap
    ws = kv.lens.new_empty((size + 3) // 4) if size else None
    _run(dev, _call().inferc_dev_paged_decode_attention, kv.ref, *a, heads,
         dim ** -0.5 if scale is None else scale, *b, *w, ws.data_ptr() if size else None, size)
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
    dev, batch = kv.dev, kv.batch
    if keep < 1 or not 0 <= recent <= keep:
        raise RuntimeError(f"{name}: keep must be at least 1 and recent in [0, keep]")
    w = _weights(name, "weights", kv, weights)
    wo = (None, 0, 0)
    if weights_out is None:
        weights_out = weights
    else:
        wo = _weights(name, "weights_out", kv, weights_out)
    dst = (None, 0, 0)
    if dst_table is not None:
        shape = dst_table.shape
        if dst_table.dtype is not _I32 or dst_table.get_device() != dev or len(shape) != 2 or \
                shape[0] != batch or (shape[1] > 1 and dst_table.stride(1) != 1):
            raise RuntimeError(f"{name}: dst_table must be int32 [batch, pages] with contiguous "
                               f"rows on CUDA device {dev}")
        dst = (dst_table.data_ptr(), shape[1],
               max(dst_table.stride(0), shape[1]) if batch <= 1 else dst_table.stride(0))
    if lens_out is None:
        lens_out = kv.lens.new_empty(batch)
        a = lens_out.data_ptr()
    else:
        a = _flat(name, "lens_out", lens_out, _I32, (batch,), dev)
    if kept is None:
        kept = kv.lens.new_empty((batch, kv.kv_heads, keep))
        b = kept.data_ptr()
    else:
        b = _flat(name, "kept", kept, _I32, (batch, kv.kv_heads, keep), dev)
    _run(dev, _call().inferc_dev_paged_kv_evict, kv.ref, *dst, *w, *wo, keep, recent, a, b)
    return lens_out, kept, weights_out
