"""4-bit latent records: store, reader and sparse-MLA decode.

A third cache format beside Native (584 bytes a record) and Packed (328): every
coordinate of the normalised, rotated latent as an E2M1 code with one power-of-two
scale per 32 coordinates, 272 bytes a record (``LatentPool(..., fmt="mx4")``, or a
uint8 [pages, 17408] page tensor). The tail is stored rotated, as in Native records,
so readers take no positions. No counterpart in the reference.

The calls mirror their siblings' (``native_store_rows``, ``unpack_gather_bf16``,
``native_sparse_decode_fwd``): shape and type mistakes raise ``ValueError`` before
anything is launched (``TypeError`` where a tensor or a number is something else
altogether), empty inputs launch nothing, and work runs asynchronously on
the current stream of the tensors' device.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib, config


def mx4_store_rows(x: torch.Tensor, weight: torch.Tensor, eps: float, loc: torch.Tensor,
                   positions: torch.Tensor | None, freqs_cis: torch.Tensor | None, pool, *,
                   layer_id: int | None = None, ratio: int = config.C4_RATIO) -> None:
    """Write raw C4 rows ``x`` [n, 512] (float32 or bfloat16) as 4-bit records at pool
    slots ``loc`` [n] int32: RMSNorm with ``weight``, BF16 rounding, the tail rotated
    with frequency row ``positions * ratio`` (``ratio``: tokens a position stands for, as
    ``native_store_rows``; ``freqs_cis=None``: not rotated) and rounded
    to BF16, then E2M1 codes under one scale per 32 coordinates. Slots outside the
    pool, and rows whose frequency row is outside the table, are skipped; those stored
    must differ (two rows for one slot leave a mixture of both). A group of 32 with an
    infinity or NaN reads back as NaN."""
    _lib.ops().store(x, weight, eps, loc, positions, freqs_cis, pool, layer_id, ratio)


def mx4_gather_bf16(pool, slots: torch.Tensor, lengths: torch.Tensor | None,
                    output: torch.Tensor | None = None, *,
                    layer_id: int | None = None) -> torch.Tensor:
    """Dense BF16 rows of 4-bit records: row q * k + j of ``output`` is the record at
    pool slot ``slots[q, j]`` (int32 [queries, k], any strides), exactly dequantized.
    Entries at or past ``lengths[q]`` (int32 [queries]; None: all k count) and slots
    outside the pool give zero rows. ``output`` is caller-owned contiguous BF16 with at
    least queries * k rows of 512 (rows past them are left as they were); None
    allocates it."""
    return _lib.ops().gather(pool, slots, lengths, output, layer_id)


def get_mx4_decode_metadata(tokens: int, heads: int, topk: int,
                            swa_topk: int = 0) -> tuple[int, int]:
    """(num_splits, workspace_bytes) of a decode of ``tokens`` query tokens, as
    ``get_decode_metadata``."""
    return _plan(int(tokens), int(heads), int(topk), int(swa_topk))


@functools.lru_cache(maxsize=1024)  # a function of the four sizes alone
def _plan(tokens: int, heads: int, topk: int, swa_topk: int) -> tuple[int, int]:
    splits = ctypes.c_int32(0)
    nbytes = ctypes.c_size_t(0)
    _lib.check(_lib.load().rm_mx4_sparse_decode_workspace(
        tokens, heads, topk, swa_topk, ctypes.byref(splits), ctypes.byref(nbytes)),
        "rm_mx4_sparse_decode_workspace")
    return splits.value, nbytes.value


def mx4_sparse_decode_fwd(q, pool, block_table, indices, *, seqlens=None, topk_length=None,
                          sink=None, softmax_scale=None, out=None, lse=None, workspace=None,
                          layer_id=None, swa_pool=None, swa_indices=None, swa_lengths=None):
    """Sparse-MLA decode over 4-bit records: ``native_sparse_decode_fwd``'s contract
    (logical record indices through the block table, lengths, sink, window rows of a
    Native ``swa_pool`` in the same softmax; returns (out [B, Sq, H, 512] bf16, lse
    [B, Sq, H])) for any number of heads up to 1024. Scale bytes of up to 159 (2^32, the
    largest that ``mx4_store_rows`` writes) are read exactly; records written elsewhere
    with a larger one read as NaN, like those the store marks with 255, where
    ``mx4_gather_bf16`` gives their values."""
    return _lib.ops().decode(q, pool, block_table, indices, seqlens, topk_length, sink,
                             softmax_scale, out, lse, workspace, layer_id, swa_pool, swa_indices,
                             swa_lengths)
