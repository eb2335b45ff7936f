"""CPU tests of the index operators and the tree attention: the plain definitions against
torch casts, closed forms and each other, and the calls that are refused before anything
is launched. No kernel runs here."""

import ctypes
import os

import numpy as np
import pytest
import torch

import index_reference as ref
import remnant
from remnant import _lib, config

I32 = torch.int32


def buf(n=64, align=256):
    raw = ctypes.create_string_buffer(n + align)
    addr = ctypes.addressof(raw)
    return raw, addr + (-addr % align)


# ---- the definitions ----

def test_codes_are_torch_casts_under_the_smallest_scale():
    rng = np.random.default_rng(0)
    n = ref.bf16(rng.standard_normal((500, 128)) * 2.0 ** rng.integers(-20, 20, (500, 1)))
    n[0] = 0
    n[1, 3] = 448.0
    n[2] = ref.bf16(np.float32(449))
    code, scale = ref.codes_of(n)
    assert scale[0] == 2.0 ** -22
    for i in range(500):
        amax = max(float(np.abs(n[i]).max()), 1e-4)
        assert amax <= 448 * float(scale[i]) and (scale[i] == 2.0 ** -22 or amax > 224 * float(scale[i]))
    want = torch.from_numpy(n / scale[:, None]).to(torch.float8_e4m3fn)
    assert np.array_equal(code, want.view(torch.uint8).numpy())
    lv = ref.levels()
    assert np.array_equal(lv[code], want.double().numpy())
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(lv, every, equal_nan=True)


def test_rows_with_an_infinity_or_nan_read_as_nan():
    n = np.ones((3, 128), np.float32)
    n[0, 5], n[1, 127] = np.inf, np.nan
    code, scale = ref.codes_of(n)
    assert np.isnan(scale[:2]).all() and scale[2] == 2.0 ** -8 and (code[:2] == 0).all()


def test_topk_definition():
    x = np.array([[3, 1, 3, -np.inf, 3, np.nan, 2, 0, -0.0]], np.float32)
    for k, want in ((1, [0]), (2, [0, 2]), (3, [0, 2, 4]), (4, [0, 2, 4, 6]), (5, [0, 1, 2, 4, 6]),
                    (6, [0, 1, 2, 4, 6, 7]), (7, [0, 1, 2, 4, 6, 7, 8]),
                    (8, [0, 1, 2, 3, 4, 6, 7, 8]), (9, list(range(9)))):
        idx, counts = ref.topk(x, None, k)
        assert idx[0].tolist() == want and counts[0] == k
    idx, counts = ref.topk(x, np.array([2]), 4)
    assert idx[0].tolist() == [0, 1, -1, -1] and counts[0] == 2


def test_tree_definition_is_causal_attention_for_a_chain():
    """A chain of nodes with no window is a causal prefix, one with a window a band."""
    rng = np.random.default_rng(3)
    pool = ref.random_native(2, 1)
    table = np.array([[1, 0]])
    held, nodes = 50, 6
    q = torch.from_numpy(rng.standard_normal((1, nodes, 2, 512)).astype(np.float32)).bfloat16()
    parents = np.arange(nodes)[None] - 1
    rows = torch.from_numpy(ref.native_rows(pool, np.concatenate([np.arange(64, 128), np.arange(64)])))
    for window in (None, 1, 7, 1000):
        out, lse, _, _ = ref.tree(q, pool, table, [held], parents, window)
        for j in range(nodes):
            lo = 0 if window is None else max(0, held + j + 1 - window)
            k = rows[lo:held + j + 1]
            logits = q[0, j].double() @ k.t() / 512 ** 0.5
            assert np.allclose(lse[0, j], torch.logsumexp(logits, 1))
            assert np.allclose(out[0, j], torch.softmax(logits, 1) @ k)


def test_paths():
    assert ref.paths([-1, 0, 0, 2, -1, -2, 5, 7, 9, 3]) == \
        [[0], [0, 1], [0, 2], [0, 2, 3], [4], None, None, None, None, [0, 2, 3, 9]]


# ---- geometry ----

def test_geometry():
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                             "include", "remnant_mi355x.h")).read()
    assert f"#define RM_INDEX_RECORD_BYTES {config.INDEX_RECORD_BYTES}" in text
    assert f"#define RM_INDEX_PAGE_BYTES {config.INDEX_PAGE_BYTES}" in text
    pool = remnant.LatentPool(3, layers=2, fmt="index", device="cpu")
    assert pool.buffer.shape == (2, 3, 8448) and pool.rows == 192 and pool.record_bytes == 132
    pool.buffer.copy_(torch.randint(0, 256, pool.buffer.shape, dtype=torch.uint8))
    page = pool.buffer[1]
    assert torch.equal(pool.values(1), page[:, :8192].reshape(3, 64, 128))
    assert torch.equal(pool.scales(1), page[:, 8192:].reshape(3, 64, 4))
    assert torch.equal(pool.records(torch.tensor([70]), 1)[0],
                       torch.cat([page[1, 6 * 128:7 * 128], page[1, 8192 + 24:8192 + 28]]))
    with pytest.raises(ValueError, match="bitmap"):
        pool.bitmaps()
    with pytest.raises(ValueError):
        remnant.LatentPool(1, fmt="index", device="cpu", keep_count=128)
    assert remnant.records_fitting(8448 * 5 + 8447, "index") == 320
    with pytest.raises(ValueError):
        remnant.configure_cache_format("index")


def test_other_operators_refuse_index_pools():
    pool = remnant.LatentPool(1, fmt="index", device="cpu")
    x, w, loc = torch.zeros(1, 512), torch.ones(512), torch.zeros(1, dtype=I32)
    out = torch.empty(1, 512, dtype=torch.bfloat16)
    q, idx, bt = torch.zeros(1, 1, 16, 512, dtype=torch.bfloat16), loc.view(1, 1, 1), loc.view(1, 1)
    native = remnant.LatentPool(1, fmt="native", device="cpu")
    for p in (pool, pool.layer()):
        for call in (lambda: remnant.pack_rows_fused(x, w, 1e-6, loc, p),
                     lambda: remnant.native_store_rows(x, w, 1e-6, loc, None, None, p),
                     lambda: remnant.mx4_store_rows(x, w, 1e-6, loc, None, None, p),
                     lambda: remnant.mx4_gather_bf16(p, bt, None),
                     lambda: remnant.unpack_gather_bf16(p, loc.view(1, 1), None, loc, None, out),
                     lambda: remnant.packed_to_native(p, loc.view(1, 1), None, loc, None, p),
                     lambda: remnant.remnant_sparse_decode_fwd(q, p, bt, idx),
                     lambda: remnant.native_sparse_decode_fwd(q, p, bt, idx),
                     lambda: remnant.mx4_sparse_decode_fwd(q, p, bt, idx),
                     lambda: remnant.tree_decode_fwd(q, p, bt, loc, bt),
                     lambda: remnant.tree_decode_fwd(q, native, bt, loc, bt, history_pool=p,
                                                     history_table=bt, history_lengths=loc),
                     lambda: remnant.remnant_buffers(p)):
            with pytest.raises(ValueError):
                call()


def test_host_cache_geometry():
    dev = remnant.LatentPool(2, layers=3, fmt="index", device="cpu")
    host = remnant.HostLatentPool.like(dev, pin_memory=False)
    assert host.buffer.shape == (3, 2, 8448)
    idx = torch.zeros(4, dtype=I32)
    with pytest.raises(ValueError, match="different record formats"):
        remnant.copy_records(remnant.LatentPool(2, layers=3, fmt="native", device="cpu"), idx,
                             host, idx)
    lib = _lib.load()
    _, a = buf(20000)
    _, s = buf()
    assert lib.rm_copy_records(a, 1, 0, s, a, 1, 0, s, 0, 1, 5, 0, None) == 0
    assert lib.rm_copy_records(a, 1, 100, s, a, 1, 8448, s, 4, 2, 5, 0, None) == -2
    assert lib.rm_copy_records(a + 4, 1, 0, s, a, 1, 0, s, 4, 1, 5, 0, None) == -3
    assert lib.rm_copy_records(a, 1, 0, s, a, 1, 0, s, 4, 1, 6, 0, None) == -4


# ---- refusals ----

def test_c_index_entries_refuse_bad_arguments():
    lib = _lib.load()
    hold = [buf(4096) for _ in range(4)]
    x, w, s, pool = [a for _, a in hold]
    #     0  1  2    3  4     5  6  7  8  9  10 11   12 13
    ok = [x, 1, 128, w, 1e-6, s, s, w, 8, 4, 4, pool, 1, None]
    for at, value, status in ((10, 0, 0), (10, -1, -2), (9, 0, -2), (9, 1 << 31, -2), (0, None, -1),
                              (3, None, -1), (5, None, -1), (6, None, -1), (11, None, -1),
                              (1, 7, -4), (0, x + 2, -3), (2, 100, -2), (2, 129, -3), (3, w + 4, -3),
                              (7, w + 8, -3), (11, pool + 8, -3), (12, -1, -2),
                              (12, (1 << 25) + 1, -2), (8, -1, -2), (5, s + 2, -3), (6, s + 1, -3)):
        args = list(ok)
        args[at] = value
        assert lib.rm_index_store_rows(*args) == status, (at, value)
    ok = [pool, 1, s, 5, 1, s, 1, 2, 5, x, None]
    for at, value, status in ((7, 0, 0), (8, 0, 0), (7, -1, -2), (8, -1, -2), (0, None, -1),
                              (2, None, -1), (9, None, -1), (9, x + 8, -3), (0, pool + 8, -3),
                              (2, s + 2, -3), (5, s + 1, -3), (1, -1, -2), (1, 1 << 26, -2)):
        args = list(ok)
        args[at] = value
        assert lib.rm_index_gather_bf16(*args) == status, (at, value)
    #     0  1  2  3   4  5     6  7  8  9  10 11  12 13
    ok = [x, 1, 1, 16, w, pool, 1, s, 4, 4, s, 64, x, None]
    for at, value, status in ((1, 0, 0), (2, 0, 0), (11, 0, 0), (1, -1, -2), (1, 65536, -2),
                              (2, (1 << 20) + 1, -2), (2, -1, -2), (3, 129, -2), (3, -1, -2),
                              (6, -1, -2), (6, 1 << 26, -2), (8, 3, -2), (9, -1, -2),
                              (9, 1 << 26, -2), (11, -1, -2), (11, 1 << 31, -2), (0, None, -1),
                              (4, None, -1), (5, None, -1), (7, None, -1), (10, None, -1),
                              (12, None, -1), (0, x + 8, -3), (5, pool + 8, -3), (4, w + 2, -3),
                              (7, s + 2, -3), (10, s + 1, -3), (12, x + 2, -3)):
        args = list(ok)
        args[at] = value
        assert lib.rm_index_scores(*args) == status, (at, value)
    #     0  1   2  3  4   5  6  7  8
    ok = [x, 64, s, 2, 64, 8, s, s, None]
    for at, value, status in ((3, 0, 0), (3, -1, -2), (1, 63, -2), (4, -1, -2), (4, (1 << 20) + 1, -2),
                              (5, -1, -2), (5, (1 << 20) + 1, -2), (3, 1 << 31, -2), (0, None, -1),
                              (6, None, -1), (7, None, -1), (0, x + 2, -3), (2, s + 2, -3),
                              (6, s + 1, -3), (7, s + 2, -3)):
        args = list(ok)
        args[at] = value
        assert lib.rm_index_topk(*args) == status, (at, value)


def test_c_tree_entries_refuse_bad_arguments():
    lib = _lib.load()
    n, size = ctypes.c_int32(), ctypes.c_size_t()
    for sizes, status in (((1, 8, 16, 4, 0, 0), 0), ((0, 0, 0, 0, 0, 0), 0), ((-1, 8, 16, 4, 0, 0), -2),
                          ((1, 65, 16, 4, 0, 0), -2), ((1, -1, 16, 4, 0, 0), -2),
                          ((1, 8, 1025, 4, 0, 0), -2), ((1, 8, -1, 4, 0, 0), -2),
                          ((65536, 1, 16, 4, 0, 0), -2), ((2048, 64, 16, 4, 0, 0), -2),
                          ((1, 8, 16, -1, 0, 0), -2), ((1, 8, 16, (1 << 24) + 1, 0, 0), -2),
                          ((1, 8, 16, 4, -1, 0), -2), ((1, 8, 16, 4, 1 << 31, 0), -2),
                          ((1, 8, 16, 4, 0, -1), -2), ((1, 8, 16, 4, 0, (1 << 24) + 1), -2)):
        assert lib.rm_tree_decode_workspace(*sizes, ctypes.byref(n), ctypes.byref(size)) == status
    hold = [buf(4096) for _ in range(4)]
    x, s, pool, past = [a for _, a in hold]
    #     0  1  2  3   4     5  6  7  8  9  10 11 12    13 14 15 16 17 18    19   20 21 22    23 24
    ok = [x, 1, 2, 16, pool, 1, s, 1, 1, s, s, 0, past, 1, s, 1, 1, s, None, 1.0, x, x, None, 0, None]
    for at, value, status in ((1, 0, 0), (2, 0, 0), (3, 0, 0), (1, -1, -2), (2, 65, -2), (3, 1025, -2),
                              (5, -1, -2), (5, 1 << 26, -2), (7, 0, -2), (8, -1, -2), (11, -1, -2),
                              (13, -1, -2), (13, 1 << 26, -2), (15, 0, -2), (16, -1, -2),
                              (0, None, -1), (4, None, -1), (6, None, -1), (9, None, -1),
                              (10, None, -1), (12, None, -1), (14, None, -1), (17, None, -1),
                              (20, None, -1), (21, None, -1), (0, x + 8, -3), (4, pool + 8, -3),
                              (12, past + 8, -3), (20, x + 8, -3), (21, x + 2, -3), (6, s + 2, -3),
                              (9, s + 1, -3), (10, s + 2, -3), (14, s + 2, -3), (17, s + 2, -3),
                              (18, s + 2, -3)):
        args = list(ok)
        args[at] = value
        assert lib.rm_tree_decode_fwd(*args) == status, (at, value)
    args = list(ok)
    args[8] = args[7] = 1000  # more rows: several splits, and no workspace
    assert lib.rm_tree_decode_fwd(*args) == -5
    args[22], args[23] = x + 8, 1 << 40
    assert lib.rm_tree_decode_fwd(*args) == -3


def test_tree_metadata():
    splits, need = remnant.get_tree_decode_metadata(1, 8, 16, 128)
    assert splits > 1 and need >= splits * 8 * 16 * 513 * 4
    assert remnant.get_tree_decode_metadata(64, 64, 16, 128) == (1, 0)
    assert remnant.get_tree_decode_metadata(1, 8, 16, 1 << 20, window=64)[0] <= 2
    with pytest.raises(RuntimeError):
        remnant.get_tree_decode_metadata(1, 65, 16, 128)


def test_store_and_gather_refuse():
    pool = remnant.LatentPool(2, fmt="index", device="cpu")
    x, w, loc = torch.zeros(4, 128), torch.ones(128), torch.zeros(4, dtype=I32)
    f = torch.zeros(8, 32, dtype=torch.complex64)
    good = dict(x=x, weight=w, eps=1e-6, loc=loc, positions=loc, freqs_cis=f, pool=pool)
    for change in (dict(x=x.half()), dict(x=torch.zeros(4, 512)), dict(x=torch.zeros(128, 4).t()),
                   dict(weight=torch.ones(512)), dict(weight=w.double()), dict(loc=loc.long()),
                   dict(loc=loc[:3]), dict(positions=None), dict(positions=loc[:2]),
                   dict(freqs_cis=f.to(torch.complex128)), dict(freqs_cis=f.conj()),
                   dict(pool=remnant.LatentPool(2, fmt="mx4", device="cpu")),
                   dict(pool=torch.zeros(2, 17408, dtype=torch.uint8)), dict(pool=None),
                   dict(layer_id=1), dict(ratio=0), dict(ratio=2.0), dict()):
        with pytest.raises(ValueError):
            remnant.index_store_rows(**(good | change))
    remnant.index_store_rows(x[:0], w, 1e-6, loc[:0], None, None, pool)  # nothing to do
    out = torch.empty(8, 128, dtype=torch.bfloat16)
    slots, n = torch.zeros(2, 4, dtype=I32), torch.zeros(2, dtype=I32)
    good = dict(pool=pool, slots=slots, lengths=n, output=out)
    for change in (dict(slots=slots.long()), dict(slots=loc), dict(lengths=n.float()),
                   dict(lengths=loc), dict(output=out[:7]), dict(output=out.float()),
                   dict(output=torch.empty(8, 256, dtype=torch.bfloat16)[:, ::2]),
                   dict(pool=remnant.LatentPool(2, fmt="native", device="cpu")), dict()):
        with pytest.raises(ValueError):
            remnant.index_gather_bf16(**(good | change))
    assert remnant.index_gather_bf16(pool, slots[:, :0], None).shape == (0, 128)


def test_scores_refuse():
    q = torch.zeros(2, 3, 8, 128, dtype=torch.bfloat16)
    w, t, n = torch.zeros(2, 3, 8), torch.zeros(2, 4, dtype=I32), torch.zeros(6, dtype=I32)
    pool = remnant.LatentPool(2, fmt="index", device="cpu")
    good = dict(q=q, weights=w, pool=pool, block_table=t, lengths=n)
    for change in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[:, 0]), dict(q=q[:, ::2]),
                   dict(q=torch.zeros(2, 3, 129, 128, dtype=torch.bfloat16),
                        weights=torch.zeros(2, 3, 129)),
                   dict(weights=w.bfloat16()), dict(weights=w[..., :4]), dict(weights=w.transpose(0, 1)),
                   dict(block_table=t[:1]), dict(block_table=t.long()), dict(block_table=t[:, ::2]),
                   dict(block_table=t[:1].expand(2, 4)), dict(lengths=n[:5]), dict(lengths=n.long()),
                   dict(lengths=torch.zeros(12, dtype=I32)[::2]), dict(out=torch.zeros(2, 3)),
                   dict(out=torch.zeros(2, 3, 64, dtype=torch.float64)), dict(out=torch.zeros(3, 2, 64)),
                   dict(out=torch.zeros(2, 3, 128)[..., ::2]), dict(layer_id=1),
                   dict(pool=remnant.LatentPool(2, fmt="native", device="cpu")), dict()):
        with pytest.raises(ValueError):
            remnant.index_scores(**(good | change))
    assert remnant.index_scores(q[:0], w[:0], pool, t[:0], n[:0]).shape == (0, 3, 256)
    assert remnant.index_scores(q, w, pool, t[:, :0], n).shape == (2, 3, 0)


def test_topk_refuses():
    x, n = torch.zeros(2, 3, 10), torch.zeros(6, dtype=I32)
    good = dict(scores=x, lengths=n, k=4)
    for change in (dict(scores=x.double()), dict(scores=x[0, 0]), dict(scores=x[None]),
                   dict(scores=torch.zeros(2, 3, 20)[..., ::2]), dict(scores=torch.zeros(2, 10, 3).transpose(1, 2)),
                   dict(scores=torch.zeros(2, 6, 10)[:, :3]), dict(scores=x[:, :1].expand(2, 3, 10)),
                   dict(lengths=n[:5]), dict(lengths=n.long()), dict(k=-1), dict(k=2.0), dict(k=None),
                   dict(k=(1 << 20) + 1), dict(out=(torch.zeros(2, 3, 4, dtype=I32),)),
                   dict(out=(torch.zeros(2, 3, 5, dtype=I32), n)), dict(out=(torch.zeros(6, 4, dtype=I32), n)),
                   dict(out=(torch.zeros(2, 3, 4, dtype=I32), n[:5])), dict()):
        with pytest.raises(ValueError):
            remnant.index_topk(**(good | change))
    idx, counts = remnant.index_topk(x[:0], None, 4)
    assert idx.shape == (0, 3, 4) and counts.shape == (0,)


def _tree_args():
    return dict(q=torch.zeros(2, 3, 16, 512, dtype=torch.bfloat16),
                pool=remnant.LatentPool(1, fmt="native", device="cpu"),
                block_table=torch.zeros(2, 1, dtype=I32), lengths=torch.zeros(2, dtype=I32),
                parents=torch.zeros(2, 3, dtype=I32))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 48, 512, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 3, 16, 512)),
    dict(q=torch.zeros(2, 3, 16, 256, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 3, 32, 512, dtype=torch.bfloat16)[:, :, ::2]),
    dict(q=torch.zeros(2, 65, 1, 512, dtype=torch.bfloat16), parents=torch.zeros(2, 65, dtype=I32)),
    dict(pool=remnant.LatentPool(1, device="cpu")), dict(pool=torch.zeros(1, 17408, dtype=torch.uint8)),
    dict(pool=None), dict(layer_id=1), dict(layer_id=-1),
    dict(block_table=torch.zeros(3, 1, dtype=I32)), dict(block_table=torch.zeros(2, 1)),
    dict(block_table=torch.zeros(2, 4, dtype=I32)[:, ::2]), dict(lengths=torch.zeros(3, dtype=I32)),
    dict(lengths=torch.zeros(2)), dict(parents=torch.zeros(2, 2, dtype=I32)),
    dict(parents=torch.zeros(2, 3)), dict(parents=torch.zeros(3, 2, dtype=I32).t()),
    dict(window=0), dict(window=-1), dict(window=2.0), dict(window=1 << 31),
    dict(history_pool=remnant.LatentPool(1, fmt="native", device="cpu")),
    dict(history_table=torch.zeros(2, 1, dtype=I32), history_lengths=torch.zeros(2, dtype=I32)),
    dict(history_pool=remnant.LatentPool(1, device="cpu"),
         history_table=torch.zeros(2, 1, dtype=I32), history_lengths=torch.zeros(2, dtype=I32)),
    dict(history_pool=remnant.LatentPool(1, fmt="native", device="cpu"),
         history_table=torch.zeros(1, 1, dtype=I32), history_lengths=torch.zeros(2, dtype=I32)),
    dict(history_pool=remnant.LatentPool(1, fmt="native", device="cpu"),
         history_table=torch.zeros(2, 1, dtype=I32), history_lengths=torch.zeros(3, dtype=I32)),
    dict(history_pool=remnant.LatentPool(1, fmt="native", device="cpu"), history_layer_id=1,
         history_table=torch.zeros(2, 1, dtype=I32), history_lengths=torch.zeros(2, dtype=I32)),
    dict(sink=torch.zeros(8)), dict(sink=torch.zeros(16, dtype=torch.float64)),
    dict(out=torch.zeros(2, 3, 16, 512)), dict(lse=torch.zeros(2, 48)),
    dict(workspace=torch.zeros(64)), dict()], ids=lambda c: "+".join(c) or "cpu")
def test_tree_refuses(change):
    args = _tree_args() | change
    with pytest.raises(ValueError):
        remnant.tree_decode_fwd(args.pop("q"), args.pop("pool"), args.pop("block_table"),
                                args.pop("lengths"), args.pop("parents"), **args)


def test_tree_of_nothing_returns_without_a_launch():
    a = _tree_args()
    out, lse = remnant.tree_decode_fwd(a["q"][:0], a["pool"], a["block_table"][:0], a["lengths"][:0],
                                       a["parents"][:0])
    assert out.shape == (0, 3, 16, 512) and lse.shape == (0, 3, 16)
    out, lse = remnant.tree_decode_fwd(a["q"][:, :0], a["pool"], a["block_table"], a["lengths"],
                                       a["parents"][:, :0])
    assert out.shape == (2, 0, 16, 512) and lse.shape == (2, 0, 16)


def test_wrong_kinds_of_arguments():
    pool = remnant.LatentPool(2, fmt="index", device="cpu")
    a = _tree_args()
    with pytest.raises(TypeError):
        remnant.index_topk(None, None, 4)
    with pytest.raises(TypeError):
        remnant.index_scores(a["q"], None, pool, a["block_table"], a["lengths"])
    with pytest.raises(TypeError):
        remnant.tree_decode_fwd(a["q"], a["pool"], a["block_table"], 5, a["parents"])
    with pytest.raises(TypeError):
        remnant.tree_decode_fwd(a["q"], a["pool"], a["block_table"], a["lengths"], a["parents"],
                                softmax_scale="1")
    negated = torch.zeros(2, 10, dtype=torch.complex64).conj().imag
    with pytest.raises(ValueError, match="strided"):
        remnant.index_topk(negated, None, 4)
