"""Pages of a paged cache: handing out, sharing, taking back and moving, on gfx950.

The pages' bookkeeping is three device int32 tensors that every layer's
``PagedKVCache`` shares: ``page_table`` ``(batch, width)``, ``seq_lens``
``(batch,)`` and ``ref_counts`` ``(num_pages,)``.  A page is free when its count
is 0; a sequence uses the first ``ceil(seq_len / page_size)`` entries of its
row; -1 stands for no page.  The calls change the tensors in place on the
current stream, read nothing on the host (so all can be captured in a graph),
and their results do not depend on the order of atomics.

A step of a serving loop::

    src, dst, granted = reserve_pages(page_table, seq_lens, ref_counts, seq_lens + 1,
                                      page_size=cache.page_size)
    for cache in layers:            # pages that two conversations shared until now
        copy_pages(cache, src, dst)
    ...                             # per layer: paged_cache_append, paged_cache_attention

Bookkeeping that contradicts itself (a page in two rows with a count of 1, a
count below the rows that hold the page) is not detected; reads and writes stay
within the tensors all the same.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import _is_python_int, _require_gfx950
from .errors import UnsupportedMI355XPath
from .paged_cache import _INT32_MAX, PAGE_SIZES, PagedKVCache, _ints, _table, _window


def _pool(page_table, seq_lens, ref_counts, rows=None, name: str = ""):
    device = page_table.device
    # (without lengths, which compaction does not read, the entries stand in for them)
    table = _table(page_table, seq_lens, device)
    if ref_counts.ndim != 1 or ref_counts.shape[0] < 1:
        raise ValueError("ref_counts must be a rank-1 (num_pages,) tensor")
    if ref_counts.shape[0] > _INT32_MAX:
        raise UnsupportedMI355XPath("ref_counts must have fewer than 2^31 pages")
    _ints(ref_counts, (ref_counts.shape[0],), device, "ref_counts")
    if rows is not None:
        _ints(rows, (table.batch,), device, name)
    pointers = [t.data_ptr() for t in (page_table, seq_lens, ref_counts, rows) if t is not None]
    if len(set(pointers)) != len(pointers):
        raise ValueError("page_table, seq_lens, ref_counts and the rows' values must be distinct")
    return table, device


def _page_size(page_size: int) -> None:
    if page_size not in PAGE_SIZES:
        raise UnsupportedMI355XPath("page_size must be 32, 64, 128 or 256")


def _workspace(lib, num_pages: int, table, device) -> torch.Tensor:
    return torch.empty(lib.g4_pages_workspace_bytes(num_pages, table.batch, table.width),
                       dtype=torch.uint8, device=device)


def fork_pages(page_table, seq_lens, ref_counts, parents, *, page_size: int) -> None:
    """Row ``b`` becomes a copy of row ``parents[b]`` as it was before the call.

    The copies share their pages; ``reserve_pages`` parts them where they are written.
    ``parents[b] == b`` leaves a row alone, a value outside ``[0, batch)`` empties it.
    """
    table, device = _pool(page_table, seq_lens, ref_counts, parents, "parents")
    _page_size(page_size)
    _require_gfx950(device)
    lib = _lib.load()
    ws = _workspace(lib, ref_counts.shape[0], table, device)
    with _lib.device_scope(device):
        _lib.check(lib.g4_pages_fork(
            ctypes.byref(table), ref_counts.data_ptr(), ref_counts.shape[0], page_size,
            parents.data_ptr(), ws.data_ptr(), ws.numel(), _lib.raw_stream(device)))


def reserve_pages(page_table, seq_lens, ref_counts, new_lens, *, page_size: int):
    """Grow the rows to ``new_lens`` tokens; returns ``(src, dst, granted)``, int32 ``(batch,)``.

    Rows take the lowest free pages in their order.  A row whose last page is part full
    and shared gets a page of its own for it first: copy ``src[b]`` to ``dst[b]`` in
    every layer (``copy_pages``; -1 where there is nothing to copy) before the next
    append.  Where such rows hold all of a page's references, the first of them keeps
    it.  ``granted[b]`` is 0 where free pages or the table's width did not suffice; such
    a row, and one whose ``new_lens`` is not more than its length, stays as it was.
    """
    table, device = _pool(page_table, seq_lens, ref_counts, new_lens, "new_lens")
    _page_size(page_size)
    _require_gfx950(device)
    lib = _lib.load()
    ws = _workspace(lib, ref_counts.shape[0], table, device)
    src, dst, granted = torch.empty((3, table.batch), dtype=torch.int32, device=device).unbind(0)
    with _lib.device_scope(device):
        _lib.check(lib.g4_pages_reserve(
            ctypes.byref(table), ref_counts.data_ptr(), ref_counts.shape[0], page_size,
            new_lens.data_ptr(), src.data_ptr(), dst.data_ptr(), granted.data_ptr(),
            ws.data_ptr(), ws.numel(), _lib.raw_stream(device)))
    return src, dst, granted


def release_pages(page_table, seq_lens, ref_counts, keep_lens, *, page_size: int,
                  sliding_window: int | None = None, num_sinks: int = 0) -> None:
    """Cut the rows to ``keep_lens`` tokens (0 ends a sequence) and give back what they free.

    With ``sliding_window``, pages whose tokens are neither among the first
    ``num_sinks`` nor visible to a query at position ``keep_lens[b]`` or later go too.
    """
    table, device = _pool(page_table, seq_lens, ref_counts, keep_lens, "keep_lens")
    _page_size(page_size)
    window = _window(sliding_window)
    if not _is_python_int(num_sinks):
        raise TypeError("num_sinks must be a Python integer")
    if num_sinks < 0:
        raise ValueError("num_sinks must be >= 0")
    _require_gfx950(device)
    with _lib.device_scope(device):
        _lib.check(_lib.load().g4_pages_release(
            ctypes.byref(table), ref_counts.data_ptr(), ref_counts.shape[0], page_size,
            keep_lens.data_ptr(), window, min(num_sinks, _INT32_MAX), _lib.raw_stream(device)))


def compact_pages(page_table, ref_counts):
    """Move the ``n`` pages in use to the first ``n``; returns ``(src, dst)``.

    Tables and counts are rewritten; the pages' contents follow with ``copy_pages(cache,
    src, dst)`` for every layer.  The lists have ``max(num_pages // 2, 1)`` entries,
    padded with -1.
    """
    table, device = _pool(page_table, None, ref_counts)
    _require_gfx950(device)
    lib = _lib.load()
    ws = _workspace(lib, ref_counts.shape[0], table, device)
    src, dst = torch.empty((2, max(ref_counts.shape[0] // 2, 1)), dtype=torch.int32,
                           device=device).unbind(0)
    with _lib.device_scope(device):
        _lib.check(lib.g4_pages_compact(
            ctypes.byref(table), ref_counts.data_ptr(), ref_counts.shape[0], src.data_ptr(),
            dst.data_ptr(), ws.data_ptr(), ws.numel(), _lib.raw_stream(device)))
    return src, dst


def copy_pages(cache: PagedKVCache, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy pages ``src[i]`` to ``dst[i]`` of one layer's cache: K, V and scales, every head.

    Pairs with an entry that is no page (-1) are skipped.  A page may not be a
    destination twice, nor a source and a destination.
    """
    desc = cache.descriptor()
    if src.ndim != 1:
        raise ValueError("src must be a rank-1 tensor")
    if src.shape[0] > _INT32_MAX:
        raise UnsupportedMI355XPath("one call copies fewer than 2^31 pages")
    for name, t in (("src", src), ("dst", dst)):
        _ints(t, (src.shape[0],), cache.device, name)
    with _lib.device_scope(cache.device):
        _lib.check(_lib.load().g4_pages_copy(
            ctypes.byref(desc), src.data_ptr(), dst.data_ptr(), src.shape[0],
            _lib.raw_stream(cache.device)))
