"""A paged K/V cache held in 8 bits, and the operators over it, on gfx950.

The reference decodes against a contiguous bf16 StaticCache
(``src/gemma4_fa4/h100_torch_ops.py:479-846``); it has no counterpart of this
cache.  K and V are e4m3 with one fp32 scale, a power of two, for each block of
32 tokens of a page and KV head, so a token's element is ``value * scale``,
which bf16 holds exactly.  Token ``t`` of sequence ``b`` lies in row
``t % page_size`` of page ``page_table[b, t // page_size]``.

* ``PagedKVCache``: one layer's pages.
* ``paged_cache_append``: round the new tokens' K and V rows into the pages.
* ``paged_cache_attention``: attention of the sequences' last tokens over the pages,
  with a sliding window and sinks for local layers.
* ``paged_cache_gather``: read tokens back as packed bf16 rows.

The page table, lengths and cumulative arrays stay on the device: no call reads
them on the host, so every call can be captured in a graph.  A table entry
outside ``[0, num_pages)`` is no page: nothing is read or written for it.
Nothing here takes part in autograd.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import G4CacheAttn, G4Layout, G4PagedCache, G4PageTable
from .attention import (
    _MAX_SINKS,
    _check_real_operands,
    _empty_as,
    _is_python_int,
    _require_gfx950,
    _validate_layout,
)
from .errors import UnsupportedMI355XPath

CACHE_BLOCK = 32  # tokens that share a scale
PAGE_SIZES = (32, 64, 128, 256)
_E4M3 = torch.float8_e4m3fn
_INT32_MAX = 2**31 - 1


class PagedKVCache:
    """One layer's K and V pages: e4m3 tensors and their scales.

    ``k`` / ``v``: ``(num_pages, num_kv_heads, page_size, head_dim)`` float8_e4m3fn,
    ``k_scale`` / ``v_scale``: ``(num_pages, num_kv_heads, page_size // 32)`` fp32
    powers of two, all contiguous on one gfx950 device.  ``page_size`` is 32, 64,
    128 or 256, ``head_dim`` 256 or 512.  The tensors are used as they are, so
    several handles may share them; what they hold need not be initialised.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._pointers = None
        self.descriptor()

    def descriptor(self) -> G4PagedCache:
        """The tensors as the library takes them, checked anew where their memory changed."""
        pointers = (self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                    self.v_scale.data_ptr())
        if pointers != self._pointers:
            self._check()
            self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = self.k.shape
            self.device = self.k.device
            self._desc = G4PagedCache(*pointers, self.num_pages, self.num_kv_heads,
                                      self.head_dim, self.page_size)
            self._pointers = pointers
        return self._desc

    def _check(self) -> None:
        k, v = self.k, self.v
        for name, t in (("k", k), ("v", v)):
            if t.ndim != 4 or t.dtype != _E4M3:
                raise ValueError(f"cache {name} must be a rank-4 float8_e4m3fn tensor "
                                 "(num_pages, num_kv_heads, page_size, head_dim)")
        if v.shape != k.shape:
            raise ValueError("cache k and v must have the same shape")
        pages, heads, page_size, head_dim = k.shape
        if pages < 1 or heads < 1:
            raise ValueError("a cache needs at least one page and one head")
        if page_size not in PAGE_SIZES or head_dim not in (256, 512):
            raise UnsupportedMI355XPath(
                "the paged cache covers page sizes 32, 64, 128 and 256 and head dims 256 and 512")
        for name, t in (("k_scale", self.k_scale), ("v_scale", self.v_scale)):
            if t.dtype != torch.float32 or t.shape != (pages, heads, page_size // CACHE_BLOCK):
                raise ValueError(f"cache {name} must be a float32 tensor "
                                 "(num_pages, num_kv_heads, page_size // 32)")
        tensors = (k, v, self.k_scale, self.v_scale)
        if any(t.device != k.device for t in tensors):
            raise ValueError("the cache's tensors must share a device")
        if not all(t.is_contiguous() for t in tensors):
            raise ValueError("the cache's tensors must be contiguous")
        _check_real_operands((k, v), ("k", "v"), label="cache k and v")
        ends = sorted((t.data_ptr(), t.data_ptr() + t.nbytes) for t in tensors)
        if any(start < end for (_, end), (start, _) in zip(ends, ends[1:])):
            raise ValueError("the cache's tensors must be distinct, without memory in common")
        _require_gfx950(k.device)

    @classmethod
    def empty(cls, num_pages: int, *, num_kv_heads: int, head_dim: int, page_size: int = 64,
              device="cuda") -> "PagedKVCache":
        """A cache of uninitialised pages."""
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        scales = (num_pages, num_kv_heads, page_size // CACHE_BLOCK)
        return cls(*(torch.empty(shape, dtype=_E4M3, device=device) for _ in range(2)),
                   *(torch.empty(scales, dtype=torch.float32, device=device) for _ in range(2)))


def _ints(t: torch.Tensor, shape, device, name: str) -> None:
    if t.dtype != torch.int32 or t.shape != shape:
        raise ValueError(f"{name} must be an INT32 tensor of shape {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{name} must share the cache's device")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _table(page_table: torch.Tensor, seq_lens: torch.Tensor | None, device) -> G4PageTable:
    shape = page_table.shape
    if len(shape) != 2 or shape[0] < 1 or shape[1] < 1:
        raise ValueError("page_table must be a rank-2 (batch, width) tensor")
    batch, width = shape
    if batch * width > _INT32_MAX:
        raise UnsupportedMI355XPath("page_table must have fewer than 2^31 entries")
    _ints(page_table, shape, device, "page_table")
    if seq_lens is None:
        return G4PageTable(page_table.data_ptr(), page_table.data_ptr(), batch, width)
    _ints(seq_lens, (batch,), device, "seq_lens")
    return G4PageTable(page_table.data_ptr(), seq_lens.data_ptr(), batch, width)


def _rows_layout(t: torch.Tensor, name: str) -> G4Layout:
    """The layout of packed rows (T, H, 256 or 512), checked."""
    _, heads, head_dim = t.shape
    strides = t.stride()
    if strides != (heads * head_dim, head_dim, 1):  # (those of contiguous rows will do)
        _validate_layout(t, name=name)
    return G4Layout(0, strides[0], strides[1])


def _window(sliding_window: int | None) -> int:
    """The library's window: 0 for none, and no more than its int holds (which is all)."""
    if sliding_window is None:
        return 0
    if not _is_python_int(sliding_window):
        raise TypeError("sliding_window must be a Python integer")
    if sliding_window < 1:
        raise ValueError("sliding_window must be positive")
    return min(sliding_window, _INT32_MAX)


def _no_autograd(needed: bool) -> None:
    if needed and torch.is_grad_enabled():
        raise UnsupportedMI355XPath("the paged cache cannot participate in autograd")


def paged_cache_append(
    cache: PagedKVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
) -> None:
    """Round new K and V rows into the pages of their sequences.

    ``k`` / ``v`` are packed bf16 ``(T, num_kv_heads, head_dim)``; rows
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` are the last tokens of sequence ``b``,
    counted in ``seq_lens[b]``.  A block's scale is the smallest power of two ``s``
    with ``amax / s <= 448`` (at least 2^-64); a block that already holds earlier
    tokens keeps the larger of that and its own, and where it grows they are rounded
    again.  Infinities are stored as the block's largest value, NaN as zero.  Tokens
    without a page are dropped, rows past ``cu_seqlens[-1]`` are not read.  A page
    may receive tokens of one sequence only (``reserve_pages`` sees to that).
    """
    desc = cache.descriptor()
    if k.ndim != 3 or v.ndim != 3 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("k and v must be rank-3 BF16 (T, H, D) tensors")
    shape = k.shape
    if shape[1] != cache.num_kv_heads or shape[2] != cache.head_dim or v.shape != shape:
        raise ValueError("k and v must match each other and the cache's heads and head dim")
    if k.device != cache.device or v.device != cache.device:
        raise ValueError("k and v must share the cache's device")
    _no_autograd(k.requires_grad or v.requires_grad)
    table = _table(page_table, seq_lens, cache.device)
    _ints(cu_seqlens, (table.batch + 1,), cache.device, "cu_seqlens")
    if k.shape[0] == 0:
        return
    k_layout, v_layout = _rows_layout(k, "k"), _rows_layout(v, "v")
    _check_real_operands((k, v), ("k", "v"), label="k and v")
    with _lib.device_scope(cache.device):
        _lib.check(_lib.load().g4_cache_append(
            ctypes.byref(desc), ctypes.byref(table), cu_seqlens.data_ptr(), k.shape[0],
            k.data_ptr(), k_layout, v.data_ptr(), v_layout, _lib.raw_stream(cache.device)))


def paged_cache_gather(
    cache: PagedKVCache,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    total: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The sequences' tokens as packed bf16 ``(total, num_kv_heads, head_dim)`` K and V.

    Row ``cu_seqlens[b] + t`` is token ``t`` of sequence ``b`` (exactly what the cache
    stands for); rows of tokens past ``seq_lens[b]`` or without a page are zero.
    Rows past ``cu_seqlens[-1]`` are not written.
    """
    desc = cache.descriptor()
    if type(total) is not int or total < 0:
        raise ValueError("total must be a non-negative Python integer")
    table = _table(page_table, seq_lens, cache.device)
    _ints(cu_seqlens, (table.batch + 1,), cache.device, "cu_seqlens")
    k = torch.empty((total, cache.num_kv_heads, cache.head_dim), dtype=torch.bfloat16,
                    device=cache.device)
    v = _empty_as(k)
    if total:
        layout = G4Layout(0, k.stride(0), k.stride(1))
        with _lib.device_scope(cache.device):
            _lib.check(_lib.load().g4_cache_gather(
                ctypes.byref(desc), ctypes.byref(table), cu_seqlens.data_ptr(), total,
                k.data_ptr(), layout, v.data_ptr(), layout, _lib.raw_stream(cache.device)))
    return k, v


_MAX_LENGTH = 1 << 30


def paged_cache_attention(
    q: torch.Tensor,
    cache: PagedKVCache,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    *,
    max_seqlen_q: int,
    max_seqlen_k: int,
    sliding_window: int | None = None,
    num_sinks: int = 0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of each sequence's last tokens over its cached tokens (scale 1.0).

    ``q`` is packed bf16 ``(T, Hq, head_dim)``; rows ``cu_seqlens_q[b]`` to
    ``cu_seqlens_q[b + 1]`` are the last tokens of sequence ``b``, whose own K and V
    are already in the cache (``paged_cache_append``) and counted in ``seq_lens[b]``.
    A query at position ``a`` sees token ``j <= a``; with ``sliding_window`` W only
    ``j > a - W`` or ``j < num_sinks`` (up to 32), and pages that no query sees any more
    may be gone (``release_pages``).  Returns bf16 O like ``q`` and fp32 LSE ``(Hq, T)``:
    0 and -inf for a query that sees nothing, NaN in O where a visible token has no page;
    rows past ``cu_seqlens_q[-1]`` are not written.  ``max_seqlen_q`` and
    ``max_seqlen_k`` are bounds of the lengths on the device, which no call reads on the
    host; a batch beyond them gets unspecified rows.  Head dim 512 takes neither
    window nor sinks; query heads are 1, 2, 4 or 8 times the cache's.

    A few new tokens per sequence are computed from the pages as they lie; from more
    than 448 query rows per KV head on (192 at head dim 256, 320 of one or two
    sequences), what the batch can see is laid out as bf16 rows in a workspace (``4 * tokens * Hkv * head_dim`` bytes a
    sequence, as many sequences at a time as fit 8 GiB).
    """
    desc = cache.descriptor()
    if q.ndim != 3 or q.dtype != torch.bfloat16:
        raise ValueError("q must be a rank-3 BF16 (T, H, D) tensor")
    total, heads, head_dim = q.shape
    if head_dim != cache.head_dim:
        raise ValueError("q must have the cache's head dim")
    if heads < 1 or heads % cache.num_kv_heads:
        raise ValueError("q's heads must be a positive multiple of the cache's")
    if heads // cache.num_kv_heads not in (1, 2, 4, 8):
        raise UnsupportedMI355XPath("the validated GQA ratios are 1, 2, 4, and 8")
    if q.device != cache.device:
        raise ValueError("q must share the cache's device")
    if not (_is_python_int(max_seqlen_q) and _is_python_int(max_seqlen_k)):
        raise TypeError("max_seqlen_q and max_seqlen_k must be Python integers")
    if not (1 <= max_seqlen_q <= _MAX_LENGTH and 1 <= max_seqlen_k <= _MAX_LENGTH):
        raise ValueError("max_seqlen_q and max_seqlen_k must be in [1, 2^30]")
    window = _window(sliding_window)
    if not _is_python_int(num_sinks):
        raise TypeError("num_sinks must be a Python integer")
    if not 0 <= num_sinks <= _MAX_SINKS:
        raise UnsupportedMI355XPath(f"num_sinks must be in [0, {_MAX_SINKS}]")
    if sliding_window is None and num_sinks:
        raise ValueError("num_sinks needs a sliding_window")
    if head_dim == 512 and sliding_window is not None:
        raise UnsupportedMI355XPath("head dim 512 attends without a window and sinks")
    _no_autograd(q.requires_grad)
    table = _table(page_table, seq_lens, cache.device)
    _ints(cu_seqlens_q, (table.batch + 1,), cache.device, "cu_seqlens_q")
    out = _empty_as(q)
    lse = torch.empty((heads, total), dtype=torch.float32, device=q.device)
    if total == 0:
        return out, lse
    q_layout = _rows_layout(q, "q")
    _check_real_operands((q,), ("q",), label="q")
    lib = _lib.load()
    prob = G4CacheAttn(desc, table, cu_seqlens_q.data_ptr(), total, heads,
                       max_seqlen_q, max_seqlen_k, window, num_sinks)
    ref = ctypes.byref(prob)
    ws = torch.empty(lib.g4_cache_attn_workspace_bytes(ref), dtype=torch.uint8, device=q.device)
    with _lib.device_scope(q.device):
        _lib.check(lib.g4_cache_attn_fwd(
            ref, q.data_ptr(), q_layout, out.data_ptr(),
            G4Layout(0, heads * head_dim, head_dim), lse.data_ptr(),
            ws.data_ptr(), ws.numel(), _lib.raw_stream(q.device)))
    return out, lse
