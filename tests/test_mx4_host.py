"""CPU tests of the 4-bit record and slot-map operators: the codec's plain definition
against torch casts and closed forms, and the calls that are refused before anything
is launched. No kernel runs here."""

import ctypes
import sys

import numpy as np
import pytest
import torch

import mx4_reference as ref
import remnant
from remnant import _lib, config

I32 = torch.int32


def buf(n=64, align=256):
    raw = ctypes.create_string_buffer(n + align)
    addr = ctypes.addressof(raw)
    return raw, addr + (-addr % align)


# ---- the definition itself ----

def test_levels_round_to_nearest_even_code():
    v = np.zeros((1, 512), np.float32)
    vals = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.26, 0.74, 5.01, -0.25, -0.75, -5.0, -6.0]
    want = [0, 1, 1, 2, 2, 4, 4, 6, 0.5, 0.5, 6, 0, -1, -4, -6]
    v[0, :15] = vals
    rec = ref.encode(v)
    assert rec[0, 256] == 127 and rec[0, 257] == 127 - 15
    assert np.array_equal(ref.decode_rows(rec)[0, :15], want)
    assert rec[0, 5] >> 4 == 8  # the -0.25 of coordinate 11 keeps its sign: code 8


@pytest.mark.parametrize("amax,e", [(6.0, 0), (6.03125, 1), (3.0, -1), (3.015625, 0), (1e-4, -15),
                                    (1e-6, -15), (0.0, -15), (6 * 2.0 ** 32, 32), (3e38, 32)])
def test_scale_is_the_smallest_that_holds_the_largest(amax, e):
    v = np.zeros((1, 512), np.float32)
    v[0, 40] = ref.bf16(np.float32([amax]))[0]
    assert ref.encode(v)[0, 257] == e + 127


def test_a_group_with_infinity_or_nan_reads_as_nan():
    v = np.ones((2, 512), np.float32)
    v[0, 33], v[1, 511] = np.inf, np.nan
    rec = ref.encode(v)
    out = ref.decode_rows(rec)
    assert rec[0, 257] == 255 and np.isnan(out[0, 32:64]).all() and (out[0, 64:] == 1).all()
    assert np.isnan(out[1, 480:]).all() and (out[1, :480] == 1).all()


def test_values_are_bf16_and_reencode_to_themselves():
    rng = np.random.default_rng(1)
    v = ref.bf16((rng.standard_normal((64, 512)) * 2.0 ** rng.integers(-12, 12, (64, 1))))
    out = ref.decode_rows(ref.encode(v))
    assert np.array_equal(ref.bf16(out), out)
    # a coded row needs no rounding: a scale not larger than its own holds it exactly
    assert np.array_equal(ref.decode_rows(ref.encode(out.astype(np.float32))), out)
    group = np.abs(v).reshape(-1, 16, 32).max(-1).repeat(32, 1)
    # steps at the top of a group are 2 * 2^e < 2/3 of its largest (amax > 3 * 2^e)
    assert (np.abs(out - v) <= np.maximum(group / 3, 2.0 ** -16)).all()


def test_window_definition_against_a_mask():
    table = np.arange(20).reshape(2, 10)[:, ::-1]
    for length, q_len, win, first in ((0, 1, 4, 2), (1, 2, 4, 2), (7, 3, 4, 0), (300, 2, 65, 3),
                                      (5, 1, 0, 2), (5, 1, 100, 100)):
        slots, counts = ref.window(table, np.array([length, 3]), q_len, win, first)
        for j in range(q_len):
            p = length - q_len + j
            t = np.arange(640)
            seen = t[(t <= p) & ((t < first) | (p - t < win))]
            want = table[0, seen // 64] * 64 + seen % 64
            n = counts[j]
            assert n == len(seen) <= first + win
            assert np.array_equal(slots[0, j, :n], want) and (slots[0, j, n:] == -1).all()


# ---- geometry, configuration ----

def test_geometry():
    text = open(_header()).read()
    assert f"#define RM_MX4_RECORD_BYTES {config.MX4_RECORD_BYTES}" in text
    assert f"#define RM_MX4_PAGE_BYTES {config.MX4_PAGE_BYTES}" in text
    assert f"#define RM_MAX_SLOT_BATCH {config.MAX_SLOT_BATCH}" in text
    pool = remnant.LatentPool(3, layers=2, fmt="mx4", device="cpu")
    assert pool.buffer.shape == (2, 3, 17408) and pool.rows == 192 and pool.record_bytes == 272
    pool.buffer.copy_(torch.randint(0, 256, pool.buffer.shape, dtype=torch.uint8))
    rec = pool.buffer[1].view(192, 272)
    assert torch.equal(pool.values(1).reshape(192, 256), rec[:, :256])
    assert torch.equal(pool.scales(1).reshape(192, 16), rec[:, 256:])
    assert torch.equal(pool.records(torch.tensor([5, 130]), 1), rec[[5, 130]])
    with pytest.raises(ValueError, match="bitmap"):
        pool.bitmaps()
    with pytest.raises(ValueError):
        remnant.LatentPool(1, fmt="mx4", device="cpu", keep_count=128)
    assert remnant.records_fitting(17408 * 5 + 17407, "mx4") == 320


def _header():
    import os
    return os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                        "remnant_mi355x.h")


def test_cache_format_selection():
    import argparse
    p = argparse.ArgumentParser()
    config.add_cli_arguments(p)
    try:
        got = config.configure_from_args(p.parse_args(["--kv-cache-format", "mx4"]))
        assert got.fmt == "mx4" and not got.packed
        assert got.record_bytes == 272 and got.page_bytes == 17408
        for bad in (dict(keep_count=128), dict(decode_impl="triton"),
                    dict(layer_keep_counts={2: 128}, compression_ratios=(0, 0, 4))):
            with pytest.raises(ValueError):
                remnant.configure_cache_format("mx4", **bad)
        assert config.current() == got
        with pytest.raises(ValueError):
            config.configure_from_args(p.parse_args(["--kv-cache-format", "mx4",
                                                     "--dsv4-c4-cache-format", "remnant"]))
    finally:
        remnant.configure_cache_format("native")


def test_other_operators_refuse_4bit_pools():
    pool = remnant.LatentPool(1, fmt="mx4", device="cpu")
    x, w, loc = torch.zeros(1, 512), torch.ones(512), torch.zeros(1, dtype=I32)
    out = torch.empty(1, 512, dtype=torch.bfloat16)
    q, idx, bt = torch.zeros(1, 1, 16, 512, dtype=torch.bfloat16), loc.view(1, 1, 1), loc.view(1, 1)
    for p in (pool, pool.layer()):
        for call in (lambda: remnant.pack_rows_fused(x, w, 1e-6, loc, p),
                     lambda: remnant.native_store_rows(x, w, 1e-6, loc, None, None, p),
                     lambda: remnant.unpack_gather_bf16(p, loc.view(1, 1), None, loc, None, out),
                     lambda: remnant.packed_to_native(p, loc.view(1, 1), None, loc, None, p),
                     lambda: remnant.remnant_sparse_decode_fwd(q, p, bt, idx),
                     lambda: remnant.native_sparse_decode_fwd(q, p, bt, idx),
                     lambda: remnant.remnant_buffers(p)):
            with pytest.raises(ValueError):
                call()


def test_host_cache_geometry():
    dev = remnant.LatentPool(2, layers=3, fmt="mx4", device="cpu")
    host = remnant.HostLatentPool.like(dev, pin_memory=False)
    assert host.buffer.shape == (3, 2, 17408)
    packed = remnant.LatentPool(2, layers=3, device="cpu")
    idx = torch.zeros(4, dtype=I32)
    with pytest.raises(ValueError, match="different record formats"):
        remnant.copy_records(packed, idx, host, idx)
    lib = _lib.load()
    _, a = buf(20000)
    _, s = buf()
    assert lib.rm_copy_records(a, 1, 0, s, a, 1, 0, s, 0, 1, 4, 256, None) == 0
    assert lib.rm_copy_records(a, 1, 100, s, a, 1, 17408, s, 4, 2, 4, 0, None) == -2
    assert lib.rm_copy_records(a + 4, 1, 0, s, a, 1, 0, s, 4, 1, 4, 0, None) == -3


# ---- refusals ----

def test_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    hold = [buf(4096) for _ in range(4)]
    x, w, s, pool = [a for _, a in hold]
    store, gather = lib.rm_mx4_store_rows, lib.rm_mx4_gather_bf16
    ok = [x, 1, 512, w, 1e-6, s, s, w, 8, 4, pool, 1, None]
    for at, value, status in ((9, 0, 0), (9, -1, -2), (0, None, -1), (3, None, -1), (5, None, -1),
                              (6, None, -1), (10, None, -1), (1, 7, -4), (0, x + 2, -3),
                              (2, 100, -2), (2, 513, -3), (3, w + 4, -3), (7, w + 8, -3),
                              (10, pool + 8, -3), (11, -1, -2), (11, (1 << 25) + 1, -2),
                              (8, -1, -2)):
        args = list(ok)
        args[at] = value
        if status or at == 9:
            assert store(*args) == status, (at, value)
    ok = [pool, 1, s, 5, 1, s, 1, 2, 5, x, None]
    for at, value, status in ((7, 0, 0), (8, 0, 0), (7, -1, -2), (8, -1, -2), (0, None, -1),
                              (2, None, -1), (9, None, -1), (9, x + 8, -3), (0, pool + 8, -3),
                              (2, s + 2, -3), (5, s + 1, -3), (1, -1, -2), (1, 1 << 26, -2)):
        args = list(ok)
        args[at] = value
        assert gather(*args) == status, (at, value)
    plan = lib.rm_mx4_sparse_decode_workspace
    n, size = ctypes.c_int32(), ctypes.c_size_t()
    for sizes, status in (((1, 16, 64, 0), 0), ((0, 0, 0, 0), 0), ((-1, 16, 64, 0), -2),
                          ((65536, 16, 64, 0), -2), ((1, 1025, 64, 0), -2), ((1, -1, 64, 0), -2),
                          ((1, 16, (1 << 20) + 1, 0), -2), ((1, 16, 64, 513), -2),
                          ((1, 16, -1, 0), -2), ((1, 16, 1, -1), -2)):
        assert plan(*sizes, ctypes.byref(n), ctypes.byref(size)) == status, sizes
    #     0  1  2  3   4     5  6  7  8  9 10 11 12 13    14 15 16 17  18    19 20 21   22 23  24
    ok = [x, 1, 1, 16, pool, 1, s, 4, 4, s, s, 8, s, None, 0, None, 0, None, None, 1.0, x, x, None,
          0, None]
    decode = lib.rm_mx4_sparse_decode_fwd
    for at, value, status in ((1, 0, 0), (2, 0, 0), (3, 0, 0), (1, -1, -2), (1, 65536, -2),
                              (3, 1025, -2), (3, -4, -2), (11, -1, -2), (11, (1 << 20) + 1, -2),
                              (7, 3, -2), (8, -1, -2), (5, -1, -2), (5, 1 << 26, -2),
                              (16, 513, -2), (14, -1, -2), (0, None, -1), (4, None, -1),
                              (6, None, -1), (10, None, -1), (20, None, -1), (21, None, -1),
                              (16, 4, -1), (0, x + 8, -3), (4, pool + 8, -3), (20, x + 2, -3),
                              (21, x + 2, -3), (6, s + 2, -3), (9, s + 2, -3), (10, s + 1, -3),
                              (12, s + 2, -3), (15, s + 2, -3), (17, s + 2, -3), (18, s + 2, -3)):
        args = list(ok)
        args[at] = value
        assert decode(*args) == status, (at, value)


def test_c_slot_entries_refuse_bad_arguments():
    lib = _lib.load()
    raw, base = buf(8192)
    t, old, new, free, loc, pos, starts, lens, taken = (base + 512 * i for i in range(9))
    #     0  1  2  3    4    5  6  7     8  9  10   11   12      13    14
    ok = [t, 8, 8, old, new, 4, 4, free, 8, 8, loc, pos, starts, lens, taken, None]
    for at, value, status in ((5, -1, -2), (5, 8193, -2), (6, 0, -2), (6, -4, -2), (1, 7, -2),
                              (2, -1, -2), (8, -1, -2), (9, -1, -2), (9, 1 << 31, -2),
                              (0, None, -1), (3, None, -1), (4, None, -1), (7, None, -1),
                              (10, None, -1), (11, None, -1), (12, None, -1), (13, None, -1),
                              (14, None, -1), (10, loc + 2, -3), (3, old + 1, -3),
                              # an output over an input, or over another output
                              (13, old, -2), (13, new + 4, -2), (12, free, -2), (10, pos, -2),
                              (14, lens + 8, -2), (11, t + 4 * 20, -2), (14, t + 4 * 31, -2)):
        args = list(ok)
        args[at] = value
        assert lib.rm_append_slots(*args) == status, (at, value)
    #     0  1  2  3    4  5  6  7  8    9
    ok = [t, 8, 8, old, 4, 1, 4, 2, loc, pos, None]
    for at, value, status in ((4, 0, 0), (5, 0, 0), (4, -1, -2), (5, -1, -2), (6, -1, -2),
                              (7, -1, -2), (1, 7, -2), (5, 1 << 30, -2), (0, None, -1),
                              (3, None, -1), (8, None, -1), (9, None, -1), (8, loc + 2, -3),
                              (8, t, -2), (9, old, -2), (9, loc + 4, -2)):
        args = list(ok)
        args[at] = value
        assert lib.rm_window_slots(*args) == status, (at, value)


def _decode_args():
    return dict(q=torch.zeros(2, 1, 16, 512, dtype=torch.bfloat16),
                pool=remnant.LatentPool(1, fmt="mx4", device="cpu"),
                block_table=torch.zeros(2, 1, dtype=I32), indices=torch.zeros(2, 1, 4, dtype=I32))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 16, 512, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 1, 16, 512)),
    dict(q=torch.zeros(2, 1, 16, 256, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 1, 32, 512, dtype=torch.bfloat16)[:, :, ::2]),
    dict(pool=remnant.LatentPool(1, device="cpu")), dict(pool=torch.zeros(1, 20992, dtype=torch.uint8)),
    dict(pool=torch.zeros(1, 17408)), dict(pool=None), dict(layer_id=1), dict(layer_id=-1),
    dict(indices=torch.zeros(2, 1, 4)), dict(indices=torch.zeros(2, 2, 4, dtype=I32)),
    dict(indices=torch.zeros(2, 1, 8, dtype=I32)[..., ::2]),
    dict(block_table=torch.zeros(3, 1, dtype=I32)), dict(block_table=torch.zeros(2, 1)),
    dict(block_table=torch.zeros(2, 4, dtype=I32)[:, ::2]),
    dict(seqlens=torch.zeros(3, dtype=I32)), dict(topk_length=torch.zeros(2)),
    dict(sink=torch.zeros(8)), dict(out=torch.zeros(2, 1, 16, 512)), dict(lse=torch.zeros(2, 16)),
    dict(workspace=torch.zeros(64)), dict(swa_indices=torch.zeros(2, 1, 4, dtype=I32)),
    dict(swa_pool=remnant.LatentPool(1, fmt="mx4", device="cpu"),
         swa_indices=torch.zeros(2, 1, 4, dtype=I32)),
    dict(swa_pool=remnant.LatentPool(1, fmt="native", device="cpu"),
         swa_indices=torch.zeros(2, 1, 513, dtype=I32)),
    dict()], ids=lambda c: "+".join(c) or "cpu")
def test_decode_refuses(change):
    args = _decode_args() | change
    with pytest.raises(ValueError):
        remnant.mx4_sparse_decode_fwd(args.pop("q"), args.pop("pool"), args.pop("block_table"),
                                      args.pop("indices"), **args)


def test_decode_of_nothing_returns_without_a_launch():
    args = _decode_args()
    out, lse = remnant.mx4_sparse_decode_fwd(args["q"][:0], args["pool"], args["block_table"][:0],
                                             args["indices"][:0])
    assert out.shape == (0, 1, 16, 512) and lse.shape == (0, 1, 16)


def test_store_and_gather_refuse():
    pool = remnant.LatentPool(2, fmt="mx4", device="cpu")
    x, w, loc = torch.zeros(4, 512), torch.ones(512), torch.zeros(4, dtype=I32)
    f = torch.zeros(8, 32, dtype=torch.complex64)
    good = dict(x=x, weight=w, eps=1e-6, loc=loc, positions=loc, freqs_cis=f, pool=pool)
    for change in (dict(x=x.half()), dict(x=x[:, :256]), dict(x=torch.zeros(512, 4).t()),
                   dict(weight=w[:100]), dict(weight=w.double()), dict(loc=loc.long()),
                   dict(loc=loc[:3]), dict(positions=None), dict(positions=loc[:2]),
                   dict(positions=loc.float()), dict(freqs_cis=f.to(torch.complex128)),
                   dict(freqs_cis=f.conj()), dict(freqs_cis=torch.zeros(8, 64)),
                   dict(pool=remnant.LatentPool(2, fmt="native", device="cpu")), dict()):
        with pytest.raises(ValueError):
            remnant.mx4_store_rows(**(good | change))
    remnant.mx4_store_rows(x[:0], w, 1e-6, loc[:0], None, None, pool)  # nothing to do
    out = torch.empty(8, 512, dtype=torch.bfloat16)
    slots, n = torch.zeros(2, 4, dtype=I32), torch.zeros(2, dtype=I32)
    good = dict(pool=pool, slots=slots, lengths=n, output=out)
    for change in (dict(slots=slots.long()), dict(slots=loc), dict(lengths=n.float()),
                   dict(lengths=loc), dict(output=out[:7]), dict(output=out.float()),
                   dict(output=torch.empty(8, 1024, dtype=torch.bfloat16)[:, ::2]),
                   dict(pool=remnant.LatentPool(2, device="cpu")), dict()):
        with pytest.raises(ValueError):
            remnant.mx4_gather_bf16(**(good | change))
    assert remnant.mx4_gather_bf16(pool, slots[:, :0], None).shape == (0, 512)


def test_lazily_negated_and_sparse_tensors_are_refused():
    """Views whose memory does not hold their values."""
    negated = torch.zeros(4, 512, dtype=torch.complex64).conj().imag
    assert negated.is_neg()
    pool = remnant.LatentPool(2, fmt="mx4", device="cpu")
    loc, w = torch.zeros(4, dtype=I32), torch.ones(512)
    for x in (negated, torch.zeros(4, 512).to_sparse()):
        with pytest.raises(ValueError, match="strided"):
            remnant.mx4_store_rows(x, w, 1e-6, loc, None, None, pool)
    with pytest.raises(TypeError):
        remnant.mx4_store_rows(None, w, 1e-6, loc, None, None, pool)
    with pytest.raises(TypeError):
        remnant.mx4_store_rows(torch.zeros(4, 512), w, "1e-6", loc, None, None, pool)


def test_calls_hold_no_references():
    pool = remnant.LatentPool(2, fmt="mx4", device="cpu")
    slots = torch.zeros(2, 0, dtype=I32)
    t, n = torch.zeros(3, 4, dtype=I32), torch.zeros(3, dtype=I32)
    held = [pool, pool.buffer, slots, t, n]
    counts = [sys.getrefcount(x) for x in held]
    for _ in range(50):
        out = remnant.mx4_gather_bf16(pool, slots, None)
        assert remnant.mx4_gather_bf16(pool, slots, None, out) is out
        assert sys.getrefcount(out) == 2
        a, b = remnant.window_slots(t, n, 0, 4)
        assert sys.getrefcount(a) == 2 and sys.getrefcount(b) == 2
        with pytest.raises(ValueError):
            remnant.append_slots(t, n, n, n, rows=4)
        with pytest.raises(ValueError):
            remnant.mx4_gather_bf16(pool, t, n[:2])
    del a, b, out
    assert [sys.getrefcount(x) for x in held] == counts


def test_slot_maps_refuse():
    t, n, f = torch.zeros(3, 4, dtype=I32), torch.zeros(3, dtype=I32), torch.zeros(5, dtype=I32)
    good = dict(block_table=t, old_lengths=n, new_lengths=n, free_pages=f, rows=8)
    big = torch.zeros(8193, dtype=I32)
    for change in (dict(block_table=t.long()), dict(block_table=n), dict(block_table=t.t()),
                   dict(block_table=t[:1].expand(3, 4)), dict(old_lengths=n[:2]),
                   dict(new_lengths=n.long()), dict(free_pages=torch.zeros(5)),
                   dict(free_pages=torch.zeros(10, dtype=I32)[::2]), dict(ratio=0),
                   dict(ratio=2.0), dict(rows=None), dict(rows=-1),
                   dict(block_table=big[:, None], old_lengths=big, new_lengths=big),
                   dict(out=(f, f, f[:4], n, n[:1]), rows=8), dict(out=(f, f, f, n, n[:1]), rows=5),
                   dict()):
        with pytest.raises(ValueError):
            remnant.append_slots(**(good | change))
    good = dict(block_table=t, lengths=n, q_len=2, window=4, first=1)
    for change in (dict(block_table=t.t()), dict(lengths=n[:1]), dict(q_len=-1), dict(window=1.5),
                   dict(first=-1), dict(out=(torch.zeros(3, 2, 4, dtype=I32), f)), dict()):
        with pytest.raises(ValueError):
            remnant.window_slots(**(good | change))
    slots, counts = remnant.window_slots(t, n, 0, 4)
    assert slots.shape == (3, 0, 4) and counts.shape == (0,)


def test_stores_refuse_ratios():
    """Frequency rows a position: a positive int of 31 bits."""
    x, w, loc = torch.zeros(4, 512), torch.ones(512), torch.zeros(4, dtype=I32)
    f = torch.zeros(8, 32, dtype=torch.complex64)
    for store, fmt in ((remnant.mx4_store_rows, "mx4"), (remnant.native_store_rows, "native")):
        pool = remnant.LatentPool(2, fmt=fmt, device="cpu")
        for ratio in (0, -4, 2 ** 31, 2.0, True, None):
            with pytest.raises(ValueError, match="ratio"):
                store(x, w, 1e-6, loc, loc, f, pool, ratio=ratio)
        with pytest.raises(ValueError, match="GPU"):
            store(x, w, 1e-6, loc, loc, f, pool, ratio=2 ** 31 - 1)
    lib = _lib.load()
    hold = [buf(4096) for _ in range(4)]
    x, w, s, pool = [a for _, a in hold]
    for store in (lib.rm_mx4_store_rows_ratio, lib.rm_native_store_rows_ratio):
        ok = [x, 1, 512, w, 1e-6, s, s, w, 8, 1, 4, pool, 1, None]
        for at, value, status in ((10, 0, 0), (9, 0, -2), (9, -1, -2), (9, 1 << 31, -2),
                                  (6, None, -1), (11, None, -1), (2, 100, -2)):
            args = list(ok)
            args[at] = value
            assert store(*args) == status, (at, value)


def test_empty_tables_have_no_strides_to_refuse():
    """A batch of nothing, its table's strides whatever they are (numpy's are zero)."""
    none = torch.zeros(0, dtype=I32)
    for strides in ((0, 0), (9, 1), (1, 2)):
        table = torch.empty_strided((0, 9), strides, dtype=I32)
        slots, counts = remnant.window_slots(table, none, 2, 4)
        assert slots.shape == (0, 2, 4) and counts.shape == (0,)


def test_slot_maps_refuse_counts_of_taken_pages():
    t, n, f = torch.zeros(3, 4, dtype=I32), torch.zeros(3, dtype=I32), torch.zeros(5, dtype=I32)
    for taken in (f, f[:0], f[0], f[:1].long(), f[:1].float(), f.view(1, 5)[:, :1]):
        with pytest.raises(ValueError, match="taken"):
            remnant.append_slots(t, n, n, f, rows=8, taken=taken)
    with pytest.raises(TypeError):
        remnant.append_slots(t, n, n, f, rows=8, taken=3)
    with pytest.raises(ValueError, match="GPU"):
        remnant.append_slots(t, n, n, f, rows=8, taken=f[:1])
    raw, base = buf(8192)
    t, old, new, free, loc, pos, starts, lens, pages, taken = (base + 512 * i for i in range(10))
    #     0  1  2  3    4    5  6  7     8  9      10 11   12   13      14    15
    ok = [t, 8, 8, old, new, 4, 4, free, 8, taken, 8, loc, pos, starts, lens, pages, None]
    for at, value, status in ((9, taken + 2, -3), (9, pages, -2), (9, t + 4, -2), (9, loc + 28, -2),
                              (9, lens, -2), (9, starts + 16, -2), (8, -1, -2), (7, None, -1),
                              (10, -1, -2)):
        args = list(ok)
        args[at] = value
        assert _lib.load().rm_append_slots_after(*args) == status, (at, value)
