"""4-bit latent records: store, reader and sparse-MLA decode.

A third cache format beside Native (584 bytes a record) and Packed (328): every
coordinate of the normalised, rotated latent as an E2M1 code with one power-of-two
scale per 32 coordinates, 272 bytes a record (``LatentPool(..., fmt="mx4")``, or a
uint8 [pages, 17408] page tensor). The tail is stored rotated, as in Native records,
so readers take no positions. No counterpart in the reference.

The calls mirror their siblings' (``native_store_rows``, ``unpack_gather_bf16``,
``native_sparse_decode_fwd``): shape and type mistakes raise ``ValueError`` before
anything is launched, empty inputs launch nothing, and work runs asynchronously on
the current stream of the tensors' device.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib, config
from .flash_mla import _swa_args
from .pool import LatentPool


# Small calls are bound by the host, so the checks below read each attribute once and
# compare shapes whole.
_I32, _BF16, _F32, _U8 = torch.int32, torch.bfloat16, torch.float32, torch.uint8
_get_device = torch._C._cuda_getDevice
_get_stream = torch._C._cuda_getCurrentRawStream


def _launch(device: int, name: str, *args) -> None:
    """Call a C entry point on the current stream of GPU ``device``."""
    fn = getattr(_lib.load(), name)
    if device == _get_device():
        status = fn(*args, _get_stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _get_stream(device))
    if status:
        _lib.check(status, name)


def _one_device(*tensors) -> int:
    """Index of the GPU that all of ``tensors`` (None left out) live on."""
    device = tensors[0].get_device()
    if device < 0:
        raise ValueError("tensors must live on the GPU")
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError("tensors must live on the same GPU")
    return device


def _pages(pool, layer_id) -> tuple[torch.Tensor, int, int]:
    """(buffer, address of the layer's pages, page count) of a 4-bit pool."""
    if isinstance(pool, LatentPool):
        if pool.fmt != "mx4":
            raise ValueError("this operator takes a 4-bit (mx4) pool")
        layer = 0 if layer_id is None else layer_id
        buf = pool.buffer
        layers, pages, page_bytes = buf.shape
        if type(layer) is not int or not 0 <= layer < layers:
            raise ValueError("layer_id out of range")
        return buf, buf.data_ptr() + layer * pages * page_bytes, pages
    if isinstance(pool, torch.Tensor):
        shape = pool.shape
        if pool.dtype is not _U8 or len(shape) != 2 or shape[1] != config.MX4_PAGE_BYTES \
                or not pool.is_contiguous():
            raise ValueError("pool must be a contiguous uint8 [pages, 17408] tensor")
        return pool, pool.data_ptr(), shape[0]
    raise ValueError("pool must be a LatentPool or a uint8 page tensor")


def mx4_store_rows(x: torch.Tensor, weight: torch.Tensor, eps: float, loc: torch.Tensor,
                   positions: torch.Tensor | None, freqs_cis: torch.Tensor | None, pool, *,
                   layer_id: int | None = None) -> None:
    """Write raw C4 rows ``x`` [n, 512] (float32 or bfloat16) as 4-bit records at pool
    slots ``loc`` [n] int32: RMSNorm with ``weight``, BF16 rounding, the tail rotated
    with frequency row ``positions * 4`` (``freqs_cis=None``: not rotated) and rounded
    to BF16, then E2M1 codes under one scale per 32 coordinates. Slots outside the
    pool, and rows whose frequency row is outside the table, are skipped; those stored
    must differ (two rows for one slot leave a mixture of both). A group of 32 with an
    infinity or NaN reads back as NaN."""
    buf, pages, n_pages = _pages(pool, layer_id)
    shape, strides, dtype = x.shape, x.stride(), x.dtype
    if len(shape) != 2 or shape[1] != config.HEAD_DIM or strides[1] != 1:
        raise ValueError("x must be [rows, 512] with unit inner stride")
    if dtype is not _F32 and dtype is not _BF16:
        raise ValueError("x must be float32 or bfloat16")
    rows = shape[0]
    if loc.dtype is not _I32 or loc.shape != (rows,) or not loc.is_contiguous():
        raise ValueError("loc must be a contiguous int32 [rows] tensor")
    if weight.dtype is not _F32 or weight.shape != (config.HEAD_DIM,) \
            or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous float32 [512] tensor")
    freq_ptr, freq_rows, pos_ptr = None, 0, None
    if freqs_cis is None:
        positions = None
    else:
        if freqs_cis.dtype != torch.complex64 or not freqs_cis.is_contiguous() \
                or freqs_cis.is_conj():
            raise ValueError("freqs_cis must be a contiguous complex64 tensor")
        if positions is None or positions.dtype is not _I32 or positions.shape != (rows,) \
                or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32 [rows] tensor when freqs_cis "
                             "is given")
        freq_ptr, freq_rows = freqs_cis.data_ptr(), freqs_cis.numel() // (config.ROPE_DIM // 2)
        pos_ptr = positions.data_ptr()
    if rows == 0 or (freqs_cis is not None and freq_rows == 0):
        return
    _launch(_one_device(x, weight, loc, positions, freqs_cis, buf), "rm_mx4_store_rows",
            x.data_ptr(), 1 if dtype is _BF16 else 0, strides[0], weight.data_ptr(),
            float(eps), loc.data_ptr(), pos_ptr, freq_ptr, freq_rows, rows, pages, n_pages)


def mx4_gather_bf16(pool, slots: torch.Tensor, lengths: torch.Tensor | None,
                    output: torch.Tensor | None = None, *,
                    layer_id: int | None = None) -> torch.Tensor:
    """Dense BF16 rows of 4-bit records: row q * k + j of ``output`` is the record at
    pool slot ``slots[q, j]`` (int32 [queries, k], any strides), exactly dequantized.
    Entries at or past ``lengths[q]`` (int32 [queries]; None: all k count) and slots
    outside the pool give zero rows. ``output`` is caller-owned contiguous BF16 with at
    least queries * k rows of 512 (rows past them are left as they were); None
    allocates it."""
    buf, pages, n_pages = _pages(pool, layer_id)
    shape = slots.shape
    if slots.dtype is not _I32 or len(shape) != 2:
        raise ValueError("slots must be int32 [queries, k]")
    queries, k = shape
    length_ptr, length_stride = None, 0
    if lengths is not None:
        if lengths.dtype is not _I32 or lengths.shape != (queries,):
            raise ValueError("lengths must be int32 [queries]")
        length_ptr, length_stride = lengths.data_ptr(), lengths.stride()[0]
    if output is None:
        output = torch.empty((queries * k, config.HEAD_DIM), dtype=_BF16, device=slots.device)
    shape = output.shape
    if output.dtype is not _BF16 or len(shape) != 2 or shape[1] != config.HEAD_DIM \
            or not output.is_contiguous():
        raise ValueError("output must be a contiguous bfloat16 [rows, 512] tensor")
    if shape[0] < queries * k:
        raise ValueError("output has fewer rows than queries * k")
    if queries * k == 0:
        return output
    _launch(_one_device(buf, slots, lengths, output), "rm_mx4_gather_bf16", pages, n_pages,
            slots.data_ptr(), *slots.stride(), length_ptr, length_stride, queries, k,
            output.data_ptr())
    return output


def get_mx4_decode_metadata(tokens: int, heads: int, topk: int,
                            swa_topk: int = 0) -> tuple[int, int]:
    """(num_splits, workspace_bytes) of a decode of ``tokens`` query tokens, as
    ``get_decode_metadata``."""
    return _plan(int(tokens), int(heads), int(topk), int(swa_topk))


_SCALE = 1.0 / math.sqrt(config.HEAD_DIM)


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
    [B, Sq, H])) for any number of heads up to 1024."""
    buf, pages, n_pages = _pages(pool, layer_id)
    shape = q.shape
    if len(shape) != 4 or shape[3] != config.HEAD_DIM or q.dtype is not _BF16 \
            or not q.is_contiguous():
        raise ValueError("q must be a contiguous bfloat16 [batch, q_len, heads, 512] tensor")
    batch, q_len, heads, _ = shape
    tokens = batch * q_len
    listed = indices.shape
    if indices.dtype is not _I32 or len(listed) != 3 or listed[0] != batch or listed[1] != q_len \
            or not indices.is_contiguous():
        raise ValueError("indices must be a contiguous int32 [batch, q_len, topk] tensor")
    topk = listed[2]
    table, bt_strides = block_table.shape, block_table.stride()
    if block_table.dtype is not _I32 or len(table) != 2 or table[0] != batch \
            or bt_strides[1] != 1:
        raise ValueError("block_table must be int32 [batch, max_blocks] with unit inner stride")
    # a single request's table may be a broadcast view (stride 0 in dim 0)
    bt_stride = bt_strides[0] if batch > 1 else max(bt_strides[0], table[1])
    seq_ptr = length_ptr = sink_ptr = None
    if seqlens is not None:
        if seqlens.dtype is not _I32 or seqlens.numel() != batch or not seqlens.is_contiguous():
            raise ValueError(f"seqlens must be a contiguous int32 tensor of {batch} entries")
        seq_ptr = seqlens.data_ptr()
    if topk_length is not None:
        if topk_length.dtype is not _I32 or topk_length.numel() != tokens \
                or not topk_length.is_contiguous():
            raise ValueError(f"topk_length must be a contiguous int32 tensor of {tokens} entries")
        length_ptr = topk_length.data_ptr()
    if sink is not None:
        if sink.dtype is not _F32 or sink.shape != (heads,) or not sink.is_contiguous():
            raise ValueError("sink must be a contiguous float32 [heads] tensor")
        sink_ptr = sink.data_ptr()
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype is not _BF16 or not out.is_contiguous():
        raise ValueError("out must be a contiguous bfloat16 tensor shaped like q")
    if lse is None:
        lse = torch.empty((batch, q_len, heads), dtype=_F32, device=q.device)
    elif lse.shape != (batch, q_len, heads) or lse.dtype is not _F32 or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous float32 [batch, q_len, heads] tensor")
    sbuf = sidx = slen = None
    sbuf_ptr, s_pages, sidx_ptr, width, slen_ptr = None, 0, None, 0, None
    if swa_pool is not None or swa_indices is not None:
        sbuf, sidx, slen, width = _swa_args(swa_pool, swa_indices, swa_lengths, batch, q_len)
        sbuf_ptr, s_pages, sidx_ptr = sbuf.data_ptr(), sbuf.shape[0], sidx.data_ptr()
        slen_ptr = None if slen is None else slen.data_ptr()
    need = _plan(tokens, heads, topk, width)[1]
    if workspace is not None and (workspace.dtype is not _U8 or not workspace.is_contiguous()):
        raise ValueError("workspace must be a contiguous uint8 tensor on the GPU")
    if tokens * heads == 0:
        return out, lse
    if need:
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(need, dtype=_U8, device=q.device)
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel()
    else:
        ws_ptr, ws_bytes = None, 0
    device = _one_device(q, buf, block_table, indices, seqlens, topk_length, sink, out, lse, sbuf,
                         sidx, slen, workspace)
    _launch(device, "rm_mx4_sparse_decode_fwd", q.data_ptr(), batch, q_len, heads, pages, n_pages,
            block_table.data_ptr(), bt_stride, table[1], seq_ptr, indices.data_ptr(), topk,
            length_ptr, sbuf_ptr, s_pages, sidx_ptr, width, slen_ptr, sink_ptr,
            _SCALE if softmax_scale is None else float(softmax_scale), out.data_ptr(),
            lse.data_ptr(), ws_ptr, ws_bytes)
    return out, lse
