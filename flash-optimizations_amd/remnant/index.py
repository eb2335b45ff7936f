"""Index keys: what a sparse decode's lists are made of.

A small key of 128 coordinates stands beside each latent record; a query token scores
the keys of its request's records and attends the ``topk`` of the highest scores. The
keys are cached as E4M3 codes with one float32 scale a row, 132 bytes a record
(``LatentPool(..., fmt="index")``, or a uint8 [pages, 8448] page tensor), in the slots of
the records themselves: one block table and one ``SlotMap`` serve both pools. No
counterpart in the reference's tree (its indexer lives in the un-vendored forks).

The calls mirror their siblings' (``mx4_store_rows``, ``mx4_gather_bf16``): shape and type
mistakes raise ``ValueError`` before anything is launched (``TypeError`` where a tensor
or a number is something else altogether), empty inputs launch nothing, and work runs
asynchronously on the current stream of the tensors' device.
"""

from __future__ import annotations

import torch

from . import _lib, config


def index_store_rows(x: torch.Tensor, weight: torch.Tensor, eps: float, loc: torch.Tensor,
                     positions: torch.Tensor | None, freqs_cis: torch.Tensor | None, pool, *,
                     layer_id: int | None = None, ratio: int = config.C4_RATIO) -> None:
    """Write raw key rows ``x`` [n, 128] (float32 or bfloat16) as index records at pool
    slots ``loc`` [n] int32: RMSNorm with ``weight``, BF16 rounding, coordinates 64 to 127
    rotated with frequency row ``positions * ratio`` (as ``native_store_rows``;
    ``freqs_cis=None``: not rotated) and rounded to BF16, then E4M3 codes under the
    smallest power of two that holds the row. Slots outside the pool, and rows whose
    frequency row is outside the table, are skipped; those stored must differ. A row with
    an infinity or NaN reads back as NaN."""
    _lib.ops().index_store(x, weight, eps, loc, positions, freqs_cis, pool, layer_id, ratio)


def index_gather_bf16(pool, slots: torch.Tensor, lengths: torch.Tensor | None,
                      output: torch.Tensor | None = None, *,
                      layer_id: int | None = None) -> torch.Tensor:
    """Dense BF16 rows [queries * k, 128] of index records, as ``mx4_gather_bf16``: code
    times scale, rounded once (exact for the store's records)."""
    return _lib.ops().index_gather(pool, slots, lengths, output, layer_id)


def index_scores(q: torch.Tensor, weights: torch.Tensor, pool, block_table: torch.Tensor,
                 lengths: torch.Tensor, *, out: torch.Tensor | None = None,
                 layer_id: int | None = None) -> torch.Tensor:
    """What each query token gives the records of its request.

    ``q`` bfloat16 [batch, q_len, heads <= 128, 128], ``weights`` float32 [batch, q_len,
    heads]; ``lengths`` int32, an entry for each of the batch * q_len tokens: the records
    it may see, the first of its request's row of ``block_table``. Returns float32 [batch,
    q_len, records]: the record's scale times the sum over heads of weight * scale of q *
    max(0, codes of q . codes of the key), heads being coded as the store codes a key; for
    scales above zero, as the store's, that is the sum of weight * max(0, q . key) of the
    coded values. -inf past a token's length and where no page is mapped.
    ``out`` sets the number of records (without it the block table's capacity). A scale
    that belongs in the scores goes into ``weights``."""
    return _lib.ops().scores(q, weights, pool, block_table, lengths, out, layer_id)


def index_topk(scores: torch.Tensor, lengths: torch.Tensor | None, k: int, *,
               out=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Numbers of the ``k`` records with the highest scores, for each row of ``scores``
    (float32 [rows, records] or [batch, q_len, records], unit inner stride), among its
    first ``lengths[row]`` (int32; None: all).

    Returns (indices int32 [..., k], counts int32 [rows]), the ``indices`` and
    ``topk_length`` of the decodes: min(k, length) numbers in ascending order, -1 behind
    them. Equal scores go to the lowest numbers; NaN counts as -inf. ``out``: the two
    tensors to write to."""
    return _lib.ops().topk(scores, lengths, k, out)
