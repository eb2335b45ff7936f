"""MI355X-native Remnant packed-KV hot path.

Store (pack), reconstruct (unpack + tail RoPE) and Direct packed sparse-MLA
decode, each a hand-written gfx950 HIP kernel reached through the C ABI in
``include/remnant_mi355x.h``. Operator names mirror the reference's fork
(``srt/remnant/packed.py``, ``sgl_kernel/flash_mla.py``) so callers can switch.
"""

from . import config
from .config import configure_cache_format, packed_profile
from .flash_mla import (get_decode_metadata, native_sparse_decode_fwd, remnant_buffers,
                        remnant_sparse_decode_fwd, sparse_decode_fwd)
from .packed import (RemnantBuffers, native_store_rows, pack_rows_fused, packed_to_native,
                     unpack_gather_bf16, unpack_rows)
from .host_cache import HostLatentPool, copy_records
from .index import index_gather_bf16, index_scores, index_store_rows, index_topk
from .mx4 import (get_mx4_decode_metadata, mx4_gather_bf16, mx4_sparse_decode_fwd,
                  mx4_store_rows)
from .pool import LatentPool, records_fitting
from .slots import SlotMap, append_slots, window_slots
from .tree import get_tree_decode_metadata, tree_decode_fwd

__all__ = [
    "config", "configure_cache_format", "packed_profile", "get_decode_metadata",
    "native_sparse_decode_fwd", "remnant_sparse_decode_fwd", "sparse_decode_fwd",
    "remnant_buffers", "RemnantBuffers",
    "native_store_rows", "pack_rows_fused", "packed_to_native", "unpack_gather_bf16",
    "unpack_rows",
    "LatentPool", "records_fitting", "HostLatentPool", "copy_records",
    "get_mx4_decode_metadata", "mx4_gather_bf16", "mx4_sparse_decode_fwd", "mx4_store_rows",
    "SlotMap", "append_slots", "window_slots",
    "index_gather_bf16", "index_scores", "index_store_rows", "index_topk",
    "get_tree_decode_metadata", "tree_decode_fwd",
]
