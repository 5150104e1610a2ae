"""Page tables and slot maps of the paged cache, built on the device, on libsimsd_b200.

A pool's free pages are a stack: `free_pages` [P] int32, of which the lowest
free_count[0] entries are free.  Each sequence has a row of `page_table` [B, max_pages],
and `held` [B] of its places are the sequence's own.

* `paged_reserve(...)` — room for each sequence's next tokens: pages from the stack, and
  the tokens' slots and positions as `paged_append` takes them.
* `paged_release(...)` — pages past the tokens that a sequence keeps, back onto the stack.
* `page_pool(...)` — an empty pool and its tables.

Both are one launch that never waits for the host, so a decoding step that grows its
sequences can be captured in a CUDA graph.  The same lengths give the same pages.
CUDA tensors only (no CPU fallback).
"""
from __future__ import annotations

import torch

from . import _lib
from .paged_cache import _check_apart, _current_device, _current_stream


def page_pool(sequences: int, max_pages: int, pages: int, device=None):
    """(page_table, held, free_pages, free_count) with all `pages` free."""
    i32 = dict(dtype=torch.int32, device=device)
    return (torch.full((sequences, max_pages), -1, **i32), torch.zeros(sequences, **i32), torch.arange(pages, **i32).flip(0),
            torch.full((1,), pages, **i32))


def _check_state(what: str, page_table, free_pages, free_count, page_size, **rows) -> None:
    given = [page_table, free_pages, free_count, *(t for t in rows.values() if t is not None)]
    if any(t.dtype != torch.int32 for t in given):
        raise TypeError(f"{what}: tables, lengths and counts are int32")
    if page_table.ndim != 2 or free_pages.ndim != 1 or free_count.numel() != 1:
        raise ValueError(f"{what}: page_table must be [B, max_pages], free_pages [P] and free_count [1], got "
                         f"{tuple(page_table.shape)} / {tuple(free_pages.shape)} / {tuple(free_count.shape)}")
    B = page_table.shape[0]
    for name, t in rows.items():
        if t is not None and t.shape != (B,):
            raise ValueError(f"{what}: {name} must be [{B}], got {tuple(t.shape)}")
    if not 1 <= page_size <= 0x7fffffff:
        raise ValueError(f"{what}: page_size must be at least 1 and below 2^31, got {page_size}")
    written = {"page_table": page_table, "free_pages": free_pages, "held": rows["held"]}
    for name, t in written.items():
        if t.numel() > 1 and t.stride(-1) != 1:
            raise ValueError(f"{what}: {name}, which is written in place, must have a unit last stride")
    _check_apart(what, **written)
    _lib.require_cuda(*given)


def paged_reserve(page_table: torch.Tensor, lens: torch.Tensor, held: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, L: int, page_size: int, count: torch.Tensor | None = None):
    """(slots [B, L] int64, positions [B, L] int64, total [B] int32): room for count[b] (L when
    None; cut to 0 .. L) more tokens after the lens[b] of each sequence.

    A sequence that its held pages do not reach for gets pages from the top of the
    stack, sequence by sequence; page_table, held and free_count move on with that, lens
    does not.  Row b of slots and positions ends in the sequence's new tokens; before them stand
    slot -1, which `paged_append` skips, and position 0.  total: lens + count, the lengths that
    attention over the new tokens takes; total - lens is what was served, the `count` of
    `paged_append8`.

    From the first sequence on that the stack cannot serve, those that need a page get no tokens
    (slots -1, total = lens), and DEV_ERR_CAPACITY is raised in `_lib.device_error()`; so it
    is with one whose pages would not fit its row.  A negative length raises
    DEV_ERR_BAD_INDEX and gets none (total 0).
    """
    out = _lib.binding().paged_reserve(page_table, lens, held, free_pages, free_count, L, page_size, count)
    if out is not None:
        return out
    if not 0 <= L <= 0x7fffffff:
        raise ValueError(f"paged_reserve: L must be at least 0 and below 2^31, got {L}")
    _check_state("paged_reserve", page_table, free_pages, free_count, page_size, lens=lens, held=held, count=count)
    dev = page_table.get_device()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return paged_reserve(page_table, lens, held, free_pages, free_count, L, page_size, count)
    B = page_table.shape[0]
    lens = lens.contiguous()
    count = count.contiguous() if count is not None else None
    slots, positions = (torch.empty((B, L), dtype=torch.int64, device=page_table.device) for _ in range(2))
    total = torch.empty((B,), dtype=torch.int32, device=page_table.device)
    stream = _current_stream(dev)
    ws, ws_bytes, _owner = _lib.stream_scratch(dev, stream, _lib.PAGED_COUNTER_BYTES, _lib.PAGED_COUNTER_BYTES)
    rc = _lib.lib().simsd_paged_reserve(
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lens.data_ptr(),
        count.data_ptr() if count is not None else None, held.data_ptr(), free_pages.data_ptr(), free_pages.shape[0],
        free_count.data_ptr(), B, L, page_size, slots.data_ptr(), positions.data_ptr(), total.data_ptr(), ws, ws_bytes,
        _lib.error_ptr(dev), stream)
    _lib.check(rc, "paged_reserve")
    return slots, positions, total


def paged_release(page_table: torch.Tensor, held: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  keep: torch.Tensor, page_size: int) -> None:
    """Sequence b keeps the pages of its first keep[b] int32 tokens (0 or less: none, it is
    finished); its other held pages go back onto the stack.

    held, free_pages and free_count move on; the entries of page_table stay as they are.  A
    stack without room for a sequence's pages (they were never taken from it) takes none of them
    and raises DEV_ERR_CAPACITY in `_lib.device_error()`.
    """
    if _lib.binding().paged_release(page_table, held, free_pages, free_count, keep, page_size) is not None:
        return
    _check_state("paged_release", page_table, free_pages, free_count, page_size, held=held, keep=keep)
    dev = page_table.get_device()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return paged_release(page_table, held, free_pages, free_count, keep, page_size)
    keep = keep.contiguous()
    stream = _current_stream(dev)
    ws, ws_bytes, _owner = _lib.stream_scratch(dev, stream, _lib.PAGED_COUNTER_BYTES, _lib.PAGED_COUNTER_BYTES)
    rc = _lib.lib().simsd_paged_release(
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1], held.data_ptr(), free_pages.data_ptr(),
        free_pages.shape[0], free_count.data_ptr(), keep.data_ptr(), page_table.shape[0], page_size, ws, ws_bytes,
        _lib.error_ptr(dev), stream)
    _lib.check(rc, "paged_release")
