"""Loader for the C-ABI library ``libremnant_mi355x.so`` (include/remnant_mi355x.h).

The library is built in-tree by ``flash-optimizations_amd/csrc/Makefile``
(``__graft_entry__.build()``). There is no fallback: when the library is
missing, every operator raises instead of computing anything on the CPU.
"""

from __future__ import annotations

import ctypes
import importlib.util
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_lib", "libremnant_mi355x.so")
OPS_PATH = os.path.join(_HERE, "_lib", "remnant_ops.so")

STATUS = {
    0: "ok",
    -1: "required pointer missing",
    -2: "size or stride out of range",
    -3: "pointer not aligned",
    -4: "unsupported dtype",
    -5: "workspace too small",
    -6: "HIP launch failed",
}

# (name, restype, argtypes) for every symbol declared in include/remnant_mi355x.h
_i64, _i32, _f32, _vp, _sz = (ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_void_p,
                              ctypes.c_size_t)
SIGNATURES = {
    "rm_version": (_i32, []),
    "rm_pack_rows": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _i64, _vp, _i64, _vp]),
    "rm_pack_rows_k": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _i64, _vp, _i64, _i32, _vp]),
    "rm_pack_rows_planes": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _i64, _vp, _vp, _vp, _i64,
                                   _i32, _vp]),
    "rm_native_store_rows": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _vp, _vp, _i64, _i64, _vp,
                                    _i64, _vp]),
    "rm_native_store_rows_ratio": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _vp, _vp, _i64, _i64,
                                          _i64, _vp, _i64, _vp]),
    "rm_unpack_gather_bf16_planes": (_i32, [_vp, _vp, _vp, _i64, _i32, _vp, _i64, _i64, _vp,
                                            _i64, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp,
                                            _vp]),
    "rm_packed_to_native_planes": (_i32, [_vp, _vp, _vp, _i64, _vp, _i64, _i64, _vp, _i64, _i64,
                                          _vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp]),
    "rm_remnant_sparse_decode_planes_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _vp, _vp, _i64,
                                                   _vp, _i64, _i64, _vp, _vp, _i64, _vp, _vp,
                                                   _i64, _vp, _i64, _vp, _vp, _vp, _i64, _vp,
                                                   _f32, _vp, _vp, _vp, _sz, _vp]),
    "rm_unpack_gather_bf16": (_i32, [_vp, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64,
                                     _i64, _i64, _vp, _i64, _vp, _vp]),
    "rm_unpack_gather_bf16_k": (_i32, [_vp, _i64, _i32, _vp, _i64, _i64, _vp, _i64, _i64, _vp,
                                       _i64, _i64, _i64, _vp, _i64, _vp, _vp]),
    "rm_packed_to_native": (_i32, [_vp, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64,
                                   _i64, _i64, _vp, _i64, _vp, _i64, _vp]),
    "rm_copy_records": (_i32, [_vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _i32,
                               _i32, _vp]),
    "rm_sparse_decode_workspace": (_i32, [_i64, _i64, _i64, ctypes.POINTER(ctypes.c_int32),
                                          ctypes.POINTER(ctypes.c_size_t)]),
    "rm_remnant_sparse_decode_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _i64,
                                            _vp, _vp, _i64, _vp, _vp, _vp, _i64, _vp, _f32, _vp,
                                            _vp, _vp, _sz, _vp]),
    "rm_native_sparse_decode_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _i64,
                                           _vp, _vp, _i64, _vp, _vp, _f32, _vp, _vp, _vp, _sz,
                                           _vp]),
    "rm_sparse_decode_workspace_swa": (_i32, [_i64, _i64, _i64, _i64,
                                              ctypes.POINTER(ctypes.c_int32),
                                              ctypes.POINTER(ctypes.c_size_t)]),
    "rm_remnant_sparse_decode_swa_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64,
                                                _i64, _vp, _vp, _i64, _vp, _vp, _i64, _vp, _i64,
                                                _vp, _vp, _vp, _i64, _vp, _f32, _vp, _vp, _vp,
                                                _sz, _vp]),
    "rm_remnant_sparse_decode_swa_noalloc_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp,
                                                        _i64, _i64, _vp, _vp, _i64, _vp, _vp,
                                                        _i64, _vp, _i64, _vp, _vp, _vp, _i64,
                                                        _vp, _f32, _vp, _vp, _vp]),
    "rm_native_sparse_decode_swa_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64,
                                               _i64, _vp, _vp, _i64, _vp, _vp, _i64, _vp, _i64,
                                               _vp, _vp, _f32, _vp, _vp, _vp, _sz, _vp]),
    "rm_mx4_store_rows": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _vp, _vp, _i64, _i64, _vp,
                                 _i64, _vp]),
    "rm_mx4_store_rows_ratio": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _vp, _vp, _i64, _i64,
                                       _i64, _vp, _i64, _vp]),
    "rm_mx4_gather_bf16": (_i32, [_vp, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp]),
    "rm_mx4_sparse_decode_workspace": (_i32, [_i64, _i64, _i64, _i64,
                                              ctypes.POINTER(ctypes.c_int32),
                                              ctypes.POINTER(ctypes.c_size_t)]),
    "rm_mx4_sparse_decode_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _vp,
                                        _vp, _i64, _vp, _vp, _i64, _vp, _i64, _vp, _vp, _f32,
                                        _vp, _vp, _vp, _sz, _vp]),
    "rm_append_slots": (_i32, [_vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp,
                               _vp, _vp, _vp, _vp]),
    "rm_append_slots_after": (_i32, [_vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _vp, _i64,
                                     _vp, _vp, _vp, _vp, _vp, _vp]),
    "rm_window_slots": (_i32, [_vp, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _vp]),
    "rm_index_store_rows": (_i32, [_vp, _i32, _i64, _vp, _f32, _vp, _vp, _vp, _i64, _i64, _i64,
                                   _vp, _i64, _vp]),
    "rm_index_gather_bf16": (_i32, [_vp, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp,
                                    _vp]),
    "rm_index_scores": (_i32, [_vp, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _i64, _i64, _vp, _i64,
                               _vp, _vp]),
    "rm_index_topk": (_i32, [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _vp]),
    "rm_tree_decode_workspace": (_i32, [_i64, _i64, _i64, _i64, _i64, _i64,
                                        ctypes.POINTER(ctypes.c_int32),
                                        ctypes.POINTER(ctypes.c_size_t)]),
    "rm_tree_decode_fwd": (_i32, [_vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp,
                                  _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp, _f32, _vp, _vp, _vp,
                                  _sz, _vp]),
}

_lib = None


class RemnantLibraryMissing(RuntimeError):
    pass


def load() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RemnantLibraryMissing(
                f"{LIB_PATH} is not built; run __graft_entry__.build() "
                "(or make -C flash-optimizations_amd/csrc)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


_ops = None


def ops():
    """Module of csrc/ops.cpp: checks and launches of the 4-bit and index operators, the
    tree attention and the slot maps, over the entry points of ``load()``."""
    return _ops or _load_ops()


def _load_ops():
    global _ops
    import torch

    from .flash_mla import _native_pages
    from .pool import LatentPool
    lib = load()
    if not os.path.exists(OPS_PATH):
        raise RemnantLibraryMissing(f"{OPS_PATH} is not built; run __graft_entry__.build() "
                                    "(or make -C flash-optimizations_amd/csrc)")
    spec = importlib.util.spec_from_file_location("remnant_ops", OPS_PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.setup(tuple(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
        "rm_mx4_store_rows_ratio", "rm_mx4_gather_bf16", "rm_mx4_sparse_decode_workspace",
        "rm_mx4_sparse_decode_fwd", "rm_append_slots_after", "rm_window_slots",
        "rm_index_store_rows", "rm_index_gather_bf16", "rm_index_scores", "rm_index_topk",
        "rm_tree_decode_workspace", "rm_tree_decode_fwd")),
        LatentPool, torch._C._cuda_getCurrentRawStream, check, _native_pages)
    _ops = module
    return module


def check(status: int, what: str) -> None:
    if status != 0:
        raise RuntimeError(f"{what}: {STATUS.get(status, 'error')} (status {status})")
