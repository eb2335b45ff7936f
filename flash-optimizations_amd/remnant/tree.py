"""Attention of drafted trees: speculative decoding's verification step.

The nodes of a request's tree are its query tokens. All of them see the same committed
rows, which are read once for all nodes and heads, and each sees the drafted rows on its
own path. For the layers that have no list of selected records: those with a sliding
window alone, with a whole history, or with a dense history of compressed records beside
the window. No counterpart in the reference's tree.
"""

from __future__ import annotations

import ctypes
import functools

from . import _lib


def get_tree_decode_metadata(batch: int, nodes: int, heads: int, blocks: int, *,
                             window: int | None = None,
                             history_blocks: int = 0) -> tuple[int, int]:
    """(num_splits, workspace_bytes) of ``tree_decode_fwd`` with block tables of
    ``blocks`` and ``history_blocks`` columns."""
    return _plan(int(batch), int(nodes), int(heads), int(blocks),
                 0 if window is None else int(window), int(history_blocks))


@functools.lru_cache(maxsize=1024)  # a function of the sizes alone
def _plan(batch, nodes, heads, blocks, window, history_blocks):
    splits = ctypes.c_int32(0)
    nbytes = ctypes.c_size_t(0)
    _lib.check(_lib.load().rm_tree_decode_workspace(
        batch, nodes, heads, blocks, window, history_blocks, ctypes.byref(splits),
        ctypes.byref(nbytes)), "rm_tree_decode_workspace")
    return splits.value, nbytes.value


def tree_decode_fwd(q, pool, block_table, lengths, parents, *, window=None, history_pool=None,
                    history_table=None, history_lengths=None, sink=None, softmax_scale=None,
                    out=None, lse=None, workspace=None, layer_id=None, history_layer_id=None):
    """Attention of ``q`` bfloat16 [batch, nodes <= 64, heads, 512], the nodes of a drafted
    tree a request, over Native rows; returns (out [batch, nodes, heads, 512] bfloat16, lse
    [batch, nodes, heads]) as ``native_sparse_decode_fwd``.

    ``lengths`` int32 [batch]: committed rows, at positions 0 to lengths - 1 of the
    request's row of ``block_table`` (int32 [batch, max_blocks]) in ``pool`` (a Native
    ``LatentPool`` or its page tensor). Node j's own row is at position lengths + j:
    ``append_slots`` with ``ratio=1`` gives the slots, ``native_store_rows`` stores it with
    its position in the text, lengths + depth. ``parents`` int32 [batch, nodes]: the number
    of the node's parent, which comes before it, or -1 for a child of the committed text;
    other numbers are padding, as are the nodes below them: zeros, lse of the sink alone.

    A node sees the committed rows, the nodes on its path and itself, with ``window`` only
    those within the last ``window`` positions of its path, and, where given, the first
    ``history_lengths[b]`` records of ``history_table`` in ``history_pool`` (compressed
    records, also Native): one softmax over all of them and the ``sink`` (float32 [heads]).
    Rows whose page is not mapped are not seen. A row with an infinity or NaN makes outputs
    NaN for the nodes that see it, and for no other."""
    return _lib.ops().tree(q, pool, block_table, lengths, parents, window, history_pool,
                           history_table, history_lengths, sink, softmax_scale, out, lse,
                           workspace, layer_id, history_layer_id)
