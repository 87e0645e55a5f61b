"""Page operators of a paged cache: copy, fork, extend, free and compact.

They keep, on the device and without a host synchronisation, what a serving
program knows about its cache pages: block tables [rows, M] (a row holds a
sequence), context lengths [rows] (0: an empty row) and reference counts [NB]
(0: a free page), all int32.  The block tables are those that the paged
decodes take.  No counterpart in the reference; device work:
flydsl_amd/csrc/cache_pages.hip.

  * :func:`copy_cache_pages`     pages onto pages, in every layer
  * :func:`fork_cache_pages`     rows that share another row's pages
  * :func:`extend_cache_pages`   pages for a row's next tokens; a partial last
    page that other rows hold too is copied first
  * :func:`free_cache_pages`     a row's pages back, all or those behind a length
  * :func:`compact_cache_pages`  the held pages moved to the front of the cache

``caches`` is a sequence of tensors whose first dimension is the page: the key
and value caches of every layer, and their per-token scales where they have
any.  A page's bytes must lie together.

Every operator decides on the state before the call and returns (compact
aside) an int32 status a list entry: 1 carried out, 0 left out (an index or
length out of range, an entry named before, a pool that has run out; see each
function).  Pages are given out lowest index first in the order of the list,
so results depend on nothing but the state.  Calls on one state have to follow
each other on a stream.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

MAX_PAGES = 4 << 20
MAX_LIST = 65536
MAX_EXTEND = 4096


def _ints(name: str, t: torch.Tensor, dims: int, dev) -> None:
    if t.dtype != torch.int32:
        raise ValueError(f"`{name}` must be int32, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"`{name}` must have {dims} dimension{'s' if dims > 1 else ''}, got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"`{name}` must be on {dev}, got {t.device}")
    if t.dim() == 1 and not t.is_contiguous():
        raise ValueError(f"`{name}` must be contiguous")
    if t.dim() == 2 and t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"`{name}` must be contiguous in its last dimension")


def _on_gpu(dev, stream) -> None:
    if dev.type != "cuda" and stream is None:
        raise RuntimeError("the page operators need tensors on a GPU (they run only in libpa_fp8.so)")


def _lists(dev, most: int, **lists) -> int:
    n = None
    for name, t in lists.items():
        _ints(name, t, 1, dev)
        if n is None:
            n = int(t.shape[0])
        elif t.shape[0] != n:
            raise ValueError(f"`{name}` must have {n} entries, got {t.shape[0]}")
    if n > most:
        raise NotImplementedError(f"at most {most} entries a call, got {n}")
    return n


def _table(block_tables, context_lengths, ref_counts, block_size):
    dev = block_tables.device
    _ints("block_tables", block_tables, 2, dev)
    _ints("context_lengths", context_lengths, 1, dev)
    _ints("ref_counts", ref_counts, 1, dev)
    rows, width = block_tables.shape
    if context_lengths.shape[0] != rows:
        raise ValueError(f"`context_lengths` must have one entry a table row ({rows}), got {context_lengths.shape[0]}")
    if rows > 1 and block_tables.stride(0) < width:
        raise ValueError("rows of `block_tables` must not overlap")
    bs = int(block_size)
    if bs < 1 or bs > 1 << 20 or bs & (bs - 1):
        raise ValueError(f"block_size must be a power of two up to 2^20, got {block_size}")
    nb = int(ref_counts.shape[0])
    if nb > MAX_PAGES:
        raise NotImplementedError(f"at most {MAX_PAGES} pages, got {nb}")
    a = _lib.PageTableArgs()
    a.abi_version = _lib.ABI_VERSION
    a.block_tables, a.context_lengths = block_tables.data_ptr(), context_lengths.data_ptr()
    a.ref_counts = ref_counts.data_ptr()
    a.stride_bt_seq = block_tables.stride(0)
    a.num_rows, a.max_blocks_per_seq, a.num_blocks, a.block_size = rows, width, nb, bs
    return a, dev


def _caches(caches, dev, pages: Optional[int]):
    """(array of PageCache, pages)"""
    out = (_lib.PageCache * max(len(caches), 1))()
    for i, t in enumerate(caches):
        if t.dim() < 1:
            raise ValueError(f"caches[{i}] must have a page dimension")
        if t.device != dev:
            raise ValueError(f"caches[{i}] must be on {dev}, got {t.device}")
        if pages is None:
            pages = int(t.shape[0])
        if t.shape[0] != pages:
            raise ValueError(f"caches[{i}] must have {pages} pages, got {t.shape[0]}")
        size = t.element_size()
        nbytes = size * (t.numel() // pages if pages else 0)
        if pages and not t[0].is_contiguous():
            raise ValueError(f"caches[{i}] must be contiguous within a page")
        stride = t.stride(0) * size if pages > 1 else nbytes
        if stride < nbytes:
            raise ValueError(f"pages of caches[{i}] must not overlap")
        out[i].data, out[i].stride_bytes, out[i].page_bytes = t.data_ptr(), stride, nbytes
    return out, pages


def _run(name: str, dev, stream, *args) -> None:
    s = stream if stream is not None else torch.cuda.current_stream(dev)
    with torch.cuda.device(dev):
        _lib.check(getattr(_lib.load(), name)(*args, ctypes.c_void_p(s.cuda_stream)), name)


def _on(stream, dev):
    """Context in which buffers of a call on ``stream`` are allocated."""
    if stream is not None and not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(stream.cuda_stream, dev)
    return torch.cuda.stream(stream)


def copy_cache_pages(caches: Sequence[torch.Tensor], source_pages: torch.Tensor, target_pages: torch.Tensor, *,
                     stream=None) -> torch.Tensor:
    """Page ``target_pages[i]`` becomes a copy of page ``source_pages[i]`` in
    every cache.  An entry is left out where a later one has the same target,
    or where the target is another entry's source.  At most 65536 entries."""
    native = _lib.native()
    if native is not None and stream is None:
        status = native.copy_pages(caches, source_pages, target_pages)
        if status is not None:
            return status
    dev = source_pages.device
    n = _lists(dev, MAX_LIST, source_pages=source_pages, target_pages=target_pages)
    if not len(caches):
        raise ValueError("copy_cache_pages needs at least one cache")
    c, pages = _caches(caches, dev, None)
    _on_gpu(dev, stream)
    with _on(stream, dev):
        status = torch.empty(n, dtype=torch.int32, device=dev)
        ws = torch.empty(_lib.pages_workspace_bytes(_lib.PAGES_COPY, 0, n), dtype=torch.uint8, device=dev)
    if n:
        _run("pa_fp8_copy_pages", dev, stream, c, len(caches), pages, source_pages.data_ptr(), target_pages.data_ptr(), n,
             status.data_ptr(), ws.data_ptr(), ws.numel())
    return status


def fork_cache_pages(block_tables: torch.Tensor, context_lengths: torch.Tensor, ref_counts: torch.Tensor,
                     parents: torch.Tensor, children: torch.Tensor, block_size: int, *, stream=None) -> torch.Tensor:
    """Row ``children[i]`` becomes a sequence of the pages and the length of
    row ``parents[i]``; each of the pages gets one more holder.  The child's
    row must be empty.  An entry is left out where an earlier one has the same
    child, or where its parent is a child in the list.  At most 65536
    entries."""
    native = _lib.native()
    if native is not None and stream is None:
        status = native.fork_pages(block_tables, context_lengths, ref_counts, parents, children, block_size)
        if status is not None:
            return status
    a, dev = _table(block_tables, context_lengths, ref_counts, block_size)
    n = _lists(dev, MAX_LIST, parents=parents, children=children)
    _on_gpu(dev, stream)
    with _on(stream, dev):
        status = torch.empty(n, dtype=torch.int32, device=dev)
    if n:
        _run("pa_fp8_fork_pages", dev, stream, a, parents.data_ptr(), children.data_ptr(), n, status.data_ptr())
    return status


def extend_cache_pages(caches: Sequence[torch.Tensor], block_tables: torch.Tensor, context_lengths: torch.Tensor,
                       ref_counts: torch.Tensor, sequences: torch.Tensor, new_lengths: torch.Tensor, block_size: int, *,
                       stream=None) -> torch.Tensor:
    """Row ``sequences[i]`` grows to ``new_lengths[i]`` tokens: it gets free
    pages for them, and where its last page is part full and has other
    holders, a copy of that page (in every cache) to write them into -- unless
    every other holder is listed before it, with such a copy.  An entry is left
    out where an earlier one has the same row; from the first entry on that
    the free pages do not suffice for, all are.  At most 4096 entries."""
    native = _lib.native()
    if native is not None and stream is None:
        status = native.extend_pages(caches, block_tables, context_lengths, ref_counts, sequences, new_lengths,
                                     block_size)
        if status is not None:
            return status
    a, dev = _table(block_tables, context_lengths, ref_counts, block_size)
    n = _lists(dev, MAX_EXTEND, sequences=sequences, new_lengths=new_lengths)
    c, _ = _caches(caches, dev, a.num_blocks)
    _on_gpu(dev, stream)
    with _on(stream, dev):
        status = torch.empty(n, dtype=torch.int32, device=dev)
        ws = torch.empty(_lib.pages_workspace_bytes(_lib.PAGES_EXTEND, a.num_blocks, n), dtype=torch.uint8, device=dev)
    if n:
        _run("pa_fp8_extend_pages", dev, stream, a, c, len(caches), sequences.data_ptr(), new_lengths.data_ptr(), n,
             status.data_ptr(), ws.data_ptr(), ws.numel())
    return status


def free_cache_pages(block_tables: torch.Tensor, context_lengths: torch.Tensor, ref_counts: torch.Tensor,
                     sequences: torch.Tensor, block_size: int, *, new_lengths: Optional[torch.Tensor] = None,
                     stream=None) -> torch.Tensor:
    """Row ``sequences[i]`` keeps its first ``new_lengths[i]`` tokens (none
    without ``new_lengths``); the pages behind them lose a holder.  An entry is
    left out where an earlier one has the same row.  At most 65536 entries."""
    native = _lib.native()
    if native is not None and stream is None:
        status = native.free_pages(block_tables, context_lengths, ref_counts, sequences, block_size, new_lengths)
        if status is not None:
            return status
    a, dev = _table(block_tables, context_lengths, ref_counts, block_size)
    lists = {"sequences": sequences}
    if new_lengths is not None:
        lists["new_lengths"] = new_lengths
    n = _lists(dev, MAX_LIST, **lists)
    _on_gpu(dev, stream)
    with _on(stream, dev):
        status = torch.empty(n, dtype=torch.int32, device=dev)
    if n:
        _run("pa_fp8_free_pages", dev, stream, a, sequences.data_ptr(),
             new_lengths.data_ptr() if new_lengths is not None else None, n, status.data_ptr())
    return status


def compact_cache_pages(
    caches: Sequence[torch.Tensor], block_tables: torch.Tensor, context_lengths: torch.Tensor,
    ref_counts: torch.Tensor, block_size: int, *, stream=None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Moves the held pages to the front of every cache.

    Returns ``(block_tables, ref_counts, page_map, live)``, new tensors: the
    tables and counts after the move, each page's new index (-1 where it was
    free) and the number [1] of held pages, which then are pages 0 ..
    live - 1.  The k-th held page at or above ``live`` moves to the k-th free
    page below it; the others stay.  The old tables and the pages they name
    are left as they were, so work that reads them may still be running; once
    the caller has gone over to the new tables, the old ones' moved pages are
    free.  Table entries behind a row's tokens are copied as they are."""
    native = _lib.native()
    if native is not None and stream is None:
        out = native.compact_pages(caches, block_tables, context_lengths, ref_counts, block_size)
        if out is not None:
            return out
    a, dev = _table(block_tables, context_lengths, ref_counts, block_size)
    c, _ = _caches(caches, dev, a.num_blocks)
    _on_gpu(dev, stream)
    with _on(stream, dev):
        i32 = dict(dtype=torch.int32, device=dev)
        tables = torch.empty(block_tables.shape, **i32)
        refs, where = torch.empty(a.num_blocks, **i32), torch.empty(a.num_blocks, **i32)
        live = torch.empty(1, **i32)
        ws = torch.empty(_lib.pages_workspace_bytes(_lib.PAGES_COMPACT, a.num_blocks, 0), dtype=torch.uint8, device=dev)
    _run("pa_fp8_compact_pages", dev, stream, a, c, len(caches), tables.data_ptr(), tables.stride(0), refs.data_ptr(),
         where.data_ptr(), live.data_ptr(), ws.data_ptr(), ws.numel())
    return tables, refs, where, live
