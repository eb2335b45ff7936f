"""Block tables and slot maps built on the GPU from request lengths.

What the store (``loc``, ``positions``), the readers (slot lists) and the decodes
(``block_table``, ``seqlens``, ``swa_indices``) take, without a round trip to the
host: a step's pages are taken from a list of free ones, and the lists of visible
slots are derived from the table. One launch a call, on the current stream of the
tensors' device; all of it can be captured in a HIP graph. No counterpart in the
reference's tree (its allocator and index builders live in the un-vendored forks).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, config
from .mx4 import _I32, _launch, _one_device


class SlotMap(NamedTuple):
    """The rows of a step: row ``row_starts[b] + i`` is record ``seqlens`` before the
    step plus i of request b."""
    loc: torch.Tensor          # int32 [rows]: pool slot, -1 past the step's records
    positions: torch.Tensor    # int32 [rows]: record number within its request
    row_starts: torch.Tensor   # int32 [batch + 1]
    seqlens: torch.Tensor      # int32 [batch]: records after the step
    pages_taken: torch.Tensor  # int32 [1]: pages needed; beyond the free list: it was short


def _vector(name, t, n):
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of {n} entries")


def _table(block_table):
    shape, strides = block_table.shape, block_table.stride()
    if block_table.dtype is not _I32 or len(shape) != 2 or (shape[1] > 1 and strides[1] != 1):
        raise ValueError("block_table must be int32 [batch, max_blocks] with unit inner stride")
    batch, width = shape
    stride = strides[0]
    if stride < width:
        if batch > 1:
            raise ValueError("block_table rows must not overlap")
        stride = width
    return batch, width, stride


def append_slots(block_table: torch.Tensor, old_lengths: torch.Tensor, new_lengths: torch.Tensor,
                 free_pages: torch.Tensor, *, ratio: int = 1, rows: int | None = None,
                 out=None) -> SlotMap:
    """Give a step's new records their pages and slots.

    Request b grows from ``old_lengths[b]`` to ``new_lengths[b]`` tokens (int32
    [batch], batch <= 8192), that is from old // ratio to new // ratio records
    (``ratio`` 4: the C4 pool; 1: one record a token; a request that does not grow
    adds none). The pages it lacks are taken, the requests in order, from the front of
    ``free_pages`` (int32 [n]) and written to the next columns of its row of
    ``block_table`` (int32 [batch, max_blocks], updated in place). Its new records are
    consecutive rows of the step, the requests in order: ``loc`` and ``positions`` are
    what ``pack_rows_fused`` / ``native_store_rows`` / ``mx4_store_rows`` take.

    ``rows`` is the capacity of the two row lists (in a captured graph: the largest
    step); rows past the step's records get slot -1, which the stores skip, and records
    past the capacity are left out. Where the free list or the table's columns run out,
    slots are -1; ``pages_taken`` tells how many pages were needed. ``out``: a
    ``SlotMap`` (or five tensors) to write to instead of new ones."""
    batch, width, stride = _table(block_table)
    if batch > config.MAX_SLOT_BATCH:
        raise ValueError(f"at most {config.MAX_SLOT_BATCH} requests a call")
    if type(ratio) is not int or not 1 <= ratio < 2 ** 31:
        raise ValueError("ratio must be a positive int")
    _vector("old_lengths", old_lengths, batch)
    _vector("new_lengths", new_lengths, batch)
    free = free_pages.shape
    if free_pages.dtype is not _I32 or len(free) != 1 or not free_pages.is_contiguous():
        raise ValueError("free_pages must be a contiguous int32 vector")
    if rows is None and out is not None:
        rows = out[0].shape[0] if out[0].dim() == 1 else 0
    elif type(rows) is not int or not 0 <= rows < 2 ** 31:
        raise ValueError("rows must be an int, the capacity of the row lists")
    if out is None:
        new = block_table.new_empty
        out = SlotMap(new(rows), new(rows), new(batch + 1), new(batch), new(1))
    else:
        if type(out) is not SlotMap:
            out = SlotMap(*out)
        _vector("loc", out.loc, rows)
        _vector("positions", out.positions, rows)
        _vector("row_starts", out.row_starts, batch + 1)
        _vector("seqlens", out.seqlens, batch)
        _vector("pages_taken", out.pages_taken, 1)
    loc, positions, row_starts, seqlens, taken = out
    device = _one_device(block_table, old_lengths, new_lengths, free_pages, loc, positions,
                         row_starts, seqlens, taken)
    _launch(device, "rm_append_slots", block_table.data_ptr(), stride, width,
            old_lengths.data_ptr(), new_lengths.data_ptr(), batch, ratio, free_pages.data_ptr(),
            free[0], rows, loc.data_ptr(), positions.data_ptr(), row_starts.data_ptr(),
            seqlens.data_ptr(), taken.data_ptr())
    return out


def window_slots(block_table: torch.Tensor, lengths: torch.Tensor, q_len: int, window: int, *,
                 first: int = 0, out=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Pool slots each query token may see: a sliding window and the request's first
    tokens.

    Query j of the last ``q_len`` tokens of request b (``lengths`` int32 [batch], the
    tokens held, the queries among them) sits at position p = lengths[b] - q_len + j and
    sees the ``first`` first tokens up to p, then the last ``window`` up to and with p,
    none twice. Returns (slots int32 [batch, q_len, first + window], counts int32
    [batch * q_len]): the slots of those tokens through ``block_table`` in ascending
    order, -1 behind them (and where no page is mapped), and their number -- the
    ``swa_indices`` and ``swa_lengths`` of the decodes, or, with a window as long as the
    history, the slot lists of the readers. ``out``: the two tensors to write to."""
    batch, width, stride = _table(block_table)
    if not (type(q_len) is type(window) is type(first) is int and 0 <= q_len < 2 ** 31
            and 0 <= window < 2 ** 31 and 0 <= first < 2 ** 31):
        raise ValueError("q_len, window and first must be non-negative ints")
    _vector("lengths", lengths, batch)
    shape = (batch, q_len, first + window)
    if out is None:
        out = block_table.new_empty(shape), block_table.new_empty(batch * q_len)
    slots, counts = out
    if slots.dtype is not _I32 or slots.shape != shape or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int32 {list(shape)} tensor")
    _vector("counts", counts, batch * q_len)
    if batch * q_len == 0:
        return slots, counts
    device = _one_device(block_table, lengths, slots, counts)
    _launch(device, "rm_window_slots", block_table.data_ptr(), stride, width, lengths.data_ptr(),
            batch, q_len, window, first, slots.data_ptr(), counts.data_ptr())
    return slots, counts
