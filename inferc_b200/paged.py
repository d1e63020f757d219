"""The paged cache of many requests and the operators on it, over device
tensors (inferc_dev_paged_*, inferc_dev_qk_norm_rotary). Re-exported by
inferc_b200.ops.

The reference keeps one dense cache per request, grown by Concat
(src/kernels/movement.cc:142-189, src/cli/main.cpp:831-836); these are the
batched forms a server needs. Checks raise RuntimeError as the other ops do;
an index found out of range on the device is never followed, and the next
ops.Synchronize (inferc_dev_stream_synchronize) raises for it.
"""
from __future__ import annotations

import torch

_binding = None


def _x():
    """The binding (inferc_b200/_paged.so, built from csrc/torch_paged.cpp),
    loaded on first use: it checks the arguments, allocates outputs and scratch
    and calls the C ABI on the current stream of the tensors' device."""
    global _binding
    if _binding is None:
        from . import lib
        lib.load()  # one instance of the library, and its message when it is missing
        try:
            from . import _paged
        except ImportError as e:
            raise ImportError("inferc_b200/_paged.so is missing or does not load: build it with "
                              "`python -m inferc_b200.build`, torch installed") from e
        _binding = _paged
    return _binding


class PagedKV:
    """A batch's view of a paged cache; holds no data of its own.

    k_cache, v_cache: [pages, kv_heads, page, head_dim] of one floating type
    (any strides but the last, e.g. a transposed [pages, page, kv_heads,
    head_dim]); page_table: int32 [batch, max_pages]; lens: int32 [batch], the
    positions each sequence holds, tokens being appended by the current step
    included. The tensors are read when an operator runs, so they are updated
    in place between steps (lens.add_(1), new table entries) and must outlive
    the work queued on them. Giving one of them other memory (lens.data = ...,
    set_, resize_) ends the view: operators on it raise."""

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 lens: torch.Tensor):
        self._h = _x().make(k_cache, v_cache, page_table, lens)
        self.k, self.v, self.page_table, self.lens = k_cache, v_cache, page_table, lens
        self.batch, self.max_pages = page_table.shape
        _, self.kv_heads, self.page, self.head_dim = k_cache.shape
        self.capacity = self.max_pages * self.page

    def __setattr__(self, name, value):
        """Operators read the tensors given at first: another one (kv.lens = ...) would be
        ignored. kv.lens += 1 works in place and is the same tensor."""
        if name in self.__dict__ and self.__dict__[name] is not value:
            raise RuntimeError(f"PagedKV: {name} is fixed; update it in place or make another view")
        super().__setattr__(name, value)


def RotaryTable(positions: int, rotary_dim: int, base: float = 10000.0, device="cuda"
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), float32 [positions, rotary_dim / 2], of the angles
    p * base^(-2 i / rotary_dim), formed in 64 bits: in 32 an angle of position
    10^6 is off by a sixteenth of a radian."""
    if rotary_dim < 2 or rotary_dim % 2 or positions < 1:
        raise RuntimeError("RotaryTable: rotary_dim must be even and positions at least 1")
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
    return _x().norm(q, k, q_gamma, k_gamma, eps, cos, sin, positions, interleaved, q_out, k_out)


def PagedKVAppend(kv: PagedKV, k: torch.Tensor, v: torch.Tensor,
                  cu_tokens: torch.Tensor | None = None) -> None:
    """Writes new rows k, v [T, kv_heads, d] as the last positions of their
    sequences: rows cu_tokens[b]..cu_tokens[b+1]-1 belong to sequence b (None:
    one row per sequence), whose lens count them already."""
    _x().append(kv._h, k, v, cu_tokens)


def QKNormRotaryAppend(kv: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       q_gamma=None, k_gamma=None, eps: float = 1e-6, cos=None, sin=None,
                       positions=None, interleaved: bool = False, cu_tokens=None,
                       q_out: torch.Tensor | None = None) -> torch.Tensor:
    """QKNormRotary of new rows with the keys and values going straight into
    the cache (PagedKVAppend); returns the queries. positions None: a token's
    slot in the cache (give them where earlier positions were evicted). Rows of
    q_out behind the last sequence are left as they are."""
    return _x().norm_append(kv._h, q, k, v, q_gamma, k_gamma, eps, cos, sin, positions,
                            interleaved, cu_tokens, q_out)


def PagedDecodeAttention(q: torch.Tensor, kv: PagedKV, scale: float | None = None,
                         weights: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [batch, heads, d], over the
    positions its sequence holds; heads is a multiple of kv_heads (query head h
    reads key head h // (heads / kv_heads)); scale None: d ** -0.5. A sequence
    of length 0 gives zeros. weights: float32 [batch, kv_heads, >= max_pages *
    page], to which each position's softmax weight is added, summed over the
    query heads of its key head."""
    return _x().attend(kv._h, q, scale, weights, out)


def PagedKVEvict(kv: PagedKV, weights: torch.Tensor, keep: int, recent: int = 0,
                 dst_table: torch.Tensor | None = None, weights_out: torch.Tensor | None = None,
                 lens_out: torch.Tensor | None = None, kept: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Trims every sequence longer than `keep` to `keep` positions per key head:
    its last `recent`, and of the others those with the largest weight (ties: the
    lower position). They move to the front in their order, in keys, values and
    weights. dst_table: int32 [batch, pages] of pages to put the result into,
    none of them in kv.page_table (None: the sequence's own, which no other sequence may share); weights_out:
    like weights, apart from them (None: in place). Returns (lens_out, kept, weights_out): the
    new lengths, a tensor apart from kv.lens; the old positions, int32 [batch,
    kv_heads, keep], -1 behind the last; and the weights."""
    return _x().evict(kv._h, weights, keep, recent, dst_table, weights_out, lens_out, kept)
