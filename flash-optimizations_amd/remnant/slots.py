"""Block tables and slot maps built on the GPU from request lengths.

What the store (``loc``, ``positions``), the readers (slot lists) and the decodes
(``block_table``, ``seqlens``, ``swa_indices``) take, without a round trip to the
host: a step's pages are taken from a list of free ones, behind those that the steps
before have taken (a count on the GPU), and the lists of visible
slots are derived from the table. One launch a call, on the current stream of the
tensors' device; all of it can be captured in a HIP graph, which then stands for one
step a replay where lengths and count are carried on in it. No counterpart in the
reference's tree (its allocator and index builders live in the un-vendored forks).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class SlotMap(NamedTuple):
    """The rows of a step: row ``row_starts[b] + i`` is record ``seqlens`` before the
    step plus i of request b."""
    loc: torch.Tensor          # int32 [rows]: pool slot, -1 past the step's records
    positions: torch.Tensor    # int32 [rows]: record number within its request, 0 past them
    row_starts: torch.Tensor   # int32 [batch + 1]
    seqlens: torch.Tensor      # int32 [batch]: records after the step
    pages_taken: torch.Tensor  # int32 [1]: pages needed so far; beyond the free list: it was short


def append_slots(block_table: torch.Tensor, old_lengths: torch.Tensor, new_lengths: torch.Tensor,
                 free_pages: torch.Tensor, *, ratio: int = 1, rows: int | None = None,
                 out=None, taken: torch.Tensor | None = None) -> SlotMap:
    """Give a step's new records their pages and slots.

    Request b grows from ``old_lengths[b]`` to ``new_lengths[b]`` tokens (int32
    [batch], batch <= 8192), that is from old // ratio to new // ratio records
    (``ratio`` 4: the C4 pool; 1: one record a token; a request that does not grow
    adds none). The pages it lacks are taken, the requests in order, from the front of
    ``free_pages`` (int32 [n]) and written to the next columns of its row of
    ``block_table`` (int32 [batch, max_blocks], updated in place). Its new records are
    consecutive rows of the step, the requests in order: ``loc`` is what the stores take
    (``pack_rows_fused``, ``native_store_rows``, ``mx4_store_rows``), and ``positions``,
    numbers of records of ``ratio`` tokens each, what the rotating ones take with the same
    ``ratio`` (theirs is 4 unless given).

    ``rows`` is the capacity of the two row lists (in a captured graph: the largest
    step); rows past the step's records get slot -1, which the stores skip, and records
    past the capacity are left out. Where the free list or the table's columns run out,
    slots are -1; ``pages_taken`` tells how many pages were needed. ``out``: a
    ``SlotMap`` (or five tensors) to write to instead of new ones.

    ``taken`` (int32 [1]): pages that earlier steps have taken from the front of
    ``free_pages``, the ``pages_taken`` of the step before; this step takes those behind
    them and counts on. Without it every call starts at the front, each replay of a
    captured one too: the pages it took have to be off the list by then. A graph that is
    a step a replay ends with ``taken.copy_(map.pages_taken)`` (``taken`` is read while
    the outputs are written, and must not be one of them) and the same of the lengths."""
    append = _lib.ops().append
    if out is None:
        return SlotMap._make(append(block_table, old_lengths, new_lengths, free_pages, ratio, rows,
                                    None, taken))
    if type(out) is not SlotMap:
        out = SlotMap(*out)
    return append(block_table, old_lengths, new_lengths, free_pages, ratio, rows, out, taken)


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
    return _lib.ops().window(block_table, lengths, q_len, window, first, out)
