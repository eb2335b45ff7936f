"""GPU tests of the 4-bit records: store bit-exact, reader exact and decode within
derived tolerances (mx4_reference.py) of the plain definitions; a serving step that
runs slot maps, store, window lists and decode together; graphs, streams."""

import ctypes
import os

import numpy as np
import pytest
import torch

import mx4_reference as ref
import remnant
from remnant import synthetic as syn

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = torch.int32


def banner(msg):
    print(f"[gpu-mx4] {msg}", flush=True)


def gpu(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype).to(DEV)


def random_pool(pages, seed, sigma=1.0):
    """uint8 [pages, 17408] of coded unit-RMS rows (numpy)."""
    rng = np.random.default_rng(seed)
    scale = np.exp(rng.uniform(np.log(0.1), np.log(10), 512))
    x = rng.standard_normal((pages * 64, 512)) * scale
    x = sigma * x / np.sqrt((x * x).mean(1, keepdims=True))
    return ref.encode(ref.bf16(x)).reshape(pages, -1)


def native_pool(pages, seed):
    pool = remnant.LatentPool(pages, fmt="native", device=DEV)
    x = syn.latents(pages * 64, seed=seed)
    remnant.native_store_rows(x.to(DEV), torch.ones(512, device=DEV), 1e-6,
                              torch.arange(pages * 64, dtype=I32, device=DEV), None, None, pool)
    return pool


# ---- the conversions ----

@pytest.fixture(scope="module")
def selftest():
    path = os.path.join(os.path.dirname(remnant.__file__), "_lib", "libremnant_selftest.so")
    if not os.path.exists(path):
        pytest.fail(f"{path} is not built (make -C flash-optimizations_amd/csrc)")
    lib = ctypes.CDLL(path)
    vp, i32 = ctypes.c_void_p, ctypes.c_int
    lib.rmt_fp4_encode_table.argtypes = [i32, i32, vp, vp, vp]
    lib.rmt_fp4_decode_table.argtypes = [vp, vp, vp]
    return lib


def test_fp4_encode_every_bf16_input_and_scale(selftest):
    """v_cvt_scalef32_pk_fp4_bf16 at the scales a store writes: the nearest level, a
    midpoint to the even code, magnitudes above 6 to 6."""
    banner("fp4 encode: all bf16 x scales -15..32")
    lo, hi = -15, 32
    out = torch.empty((hi - lo + 1) * 65536, dtype=torch.uint8, device=DEV)
    result = torch.tensor([0, -1], dtype=torch.int64, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert selftest.rmt_fp4_encode_table(lo, hi, out.data_ptr(), result.data_ptr(), stream) == 0
    assert result[0].item() == 0, "the codes of one dword differ"
    table = out.cpu().numpy().reshape(-1, 65536)
    bits = np.arange(65536, dtype=np.uint32)
    with np.errstate(invalid="ignore"):
        n = (bits << 16).view(np.float32).astype(np.float64)
    finite = np.isfinite(n)
    mid = (ref.LEVELS[1:] + ref.LEVELS[:-1]) / 2
    for e in range(lo, hi + 1):
        v = np.abs(n[finite]) * 2.0 ** -e
        code = np.searchsorted(mid, v, side="left")  # a midpoint to the lower level ...
        tie = np.isin(v, mid)
        code = np.where(tie & (code % 2 == 1), code + 1, code)  # ... unless that is odd
        assert np.array_equal(table[e - lo][finite], code + 8 * np.signbit(n[finite])), e


def test_fp4_decode_every_byte_and_scale(selftest):
    """v_cvt_scalef32_pk_bf16_fp4 at the scale bytes a store writes, 255 among them."""
    banner("fp4 decode: all bytes x scales")
    out = torch.empty(65536, dtype=torch.int32, device=DEV)
    result = torch.tensor([0, -1], dtype=torch.int64, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert selftest.rmt_fp4_decode_table(out.data_ptr(), result.data_ptr(), stream) == 0
    got = out.view(torch.bfloat16).double().cpu().numpy().reshape(256, 256, 2)
    level = np.concatenate([ref.LEVELS, -ref.LEVELS])
    codes = np.arange(256)
    want = np.stack([level[codes & 15], level[codes >> 4]], -1)
    assert np.isnan(got[255]).all()
    scales = np.arange(112, 160)
    assert np.array_equal(got[scales], want * 2.0 ** (scales - 127.0)[:, None, None])


# ---- store ----

def store(x, slots, pages, weight=None, eps=1e-6, positions=None, freqs=None, fill=0x5A):
    pool = remnant.LatentPool(pages, fmt="mx4", device=DEV)
    pool.buffer.fill_(fill)
    w = torch.ones(512) if weight is None else weight
    remnant.mx4_store_rows(x.to(DEV), w.float().to(DEV), eps, gpu(slots, I32),
                           None if positions is None else gpu(positions, I32),
                           None if freqs is None else freqs.to(DEV), pool)
    torch.cuda.synchronize()
    return pool.layer().cpu().numpy()


def expect(x, slots, pages, weight=None, eps=1e-6, positions=None, freqs=None, fill=0x5A):
    pool = np.full((pages * 64, 272), fill, np.uint8)
    slots = np.asarray(slots, np.int64)
    ok = (slots >= 0) & (slots < pages * 64)
    if freqs is not None:
        row = np.asarray(positions, np.int64) * 4
        ok &= (row >= 0) & (row < freqs.shape[0])
        positions = np.asarray(positions)[ok]
    w = np.ones(512, np.float32) if weight is None else weight.float().numpy()
    pool[slots[ok]] = ref.store_rows(x[torch.from_numpy(ok)], w, eps, positions, freqs)
    return pool.reshape(pages, -1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 64, 1000, 16385, 70001])
def test_store_is_bit_exact(rows, dtype):
    banner(f"store {rows} {dtype}")
    rng = np.random.default_rng(rows)
    x = syn.latents(rows, seed=rows).float()
    x = (x * torch.pow(2.0, torch.randint(-20, 20, (rows, 1)).float())).to(dtype)
    pages = rows // 64 + 2
    slots = rng.permutation(pages * 64)[:rows].astype(np.int32)
    slots[2::17] = -1
    slots[5::31] = pages * 64 + 3
    weight = torch.linspace(0.5, 1.5, 512)
    freqs = syn.rope_freqs(4 * 500)
    positions = rng.integers(-1, 501, rows)
    args = dict(weight=weight, positions=positions, freqs=freqs)
    assert np.array_equal(store(x, slots, pages, **args), expect(x, slots, pages, **args))
    assert np.array_equal(store(x, slots, pages, weight), expect(x, slots, pages, weight))


def test_store_above_the_streaming_limit_equals_smaller_calls():
    banner("store 131073")
    n = 131073
    x = syn.latents(n, seed=8).to(DEV)
    w = torch.linspace(0.5, 1.5, 512, device=DEV)
    slots = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(I32).to(DEV)
    pages = (n + 63) // 64
    pools = [torch.zeros(pages, 17408, dtype=torch.uint8, device=DEV) for _ in range(2)]
    remnant.mx4_store_rows(x, w, 1e-6, slots, None, None, pools[0])
    for at in range(0, n, 50000):
        remnant.mx4_store_rows(x[at:at + 50000], w, 1e-6, slots[at:at + 50000].contiguous(), None,
                               None, pools[1])
    assert torch.equal(*pools)


def test_store_special_rows():
    """Zeros, ties of every level, the largest and smallest magnitudes, infinities and
    NaN in some groups, a weight that saturates the scale; strided rows."""
    banner("store special rows")
    rows = torch.zeros(16, 512)
    rows[1] = 1.0
    rows[2] = torch.arange(512) % 25 * 0.25
    rows[3] = -rows[2]
    rows[4] = 3e38
    rows[5] = 1e-38
    rows[6, 7] = float("inf")
    rows[7, 7] = float("nan")
    rows[8] = torch.where(torch.arange(512) == 3, 1e30, 1e-30)
    rows[9] = torch.where(torch.arange(512) % 32 == 0, 6.0, 0.25)
    rows[10] = -0.0
    rows[11:] = torch.randn(5, 512, generator=torch.Generator().manual_seed(3))
    wide = torch.zeros(16, 1024)
    wide[:, :512] = rows
    big = torch.ones(512)
    big[32:64] = 1e12
    big[64:96] = 1e-12
    big[96] = float("inf")
    for x in (rows, rows.bfloat16(), wide[:, :512]):
        for weight in (None, big):
            for eps in (1e-6, 0.0, 1e-30):
                got = store(x, np.arange(16), 1, weight, eps)
                assert np.array_equal(got, expect(x, np.arange(16), 1, weight, eps)), eps


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [4097, 4112, 65537, 65552])
def test_store_special_rows_in_large_calls(rows, dtype):
    """Each form of the store writes the same record for the same row, also next to an
    infinity, to rows left out and at the end of the call."""
    banner(f"store special rows x {rows} {dtype}")
    base = syn.latents(23, seed=9).float()
    base[3] = 0.0
    base[5, 100] = float("inf")
    base[6, 511] = float("nan")
    base[8] *= 1e18
    base[9] *= 1e-18
    base[10] = torch.arange(512) % 25 * 0.25
    base = base.to(dtype)
    freqs = syn.rope_freqs(4 * 23).to(DEV)
    weight = torch.linspace(0.5, 1.5, 512, device=DEV)
    ids = torch.arange(rows) % 23
    pages = rows // 64 + 1
    slots = torch.arange(rows, dtype=I32)
    slots[(torch.arange(rows) % 29 == 7) | (torch.arange(rows) // 64 % 5 == 3)] = -1
    pools = []
    for take, where in ((ids, slots), (torch.arange(23), torch.arange(23, dtype=I32))):
        pool = torch.full((pages, 17408), 0x5A, dtype=torch.uint8, device=DEV)
        remnant.mx4_store_rows(base[take].to(DEV), weight, 1e-6, where.to(DEV),
                               take.to(I32).to(DEV), freqs, pool)
        pools.append(pool.cpu().reshape(-1, 272))
    want = pools[1][:23][ids]
    want[slots < 0] = 0x5A
    assert torch.equal(pools[0][:rows], want)
    assert (pools[0][rows:] == 0x5A).all()


def test_store_keeps_bytes_past_4_gib_apart():
    """A pool of 4.6 GB: the last slots' records, beyond 32-bit offsets."""
    banner("store far slots")
    pages = 265000
    pool = remnant.LatentPool(pages, fmt="mx4", device=DEV)
    x = syn.latents(40, seed=5)
    slots = np.concatenate([np.arange(20), pages * 64 - 1 - np.arange(20)])
    remnant.mx4_store_rows(x.to(DEV), torch.ones(512, device=DEV), 1e-6, gpu(slots, I32), None,
                           None, pool)
    want = ref.store_rows(x, np.ones(512), 1e-6)
    assert np.array_equal(pool.records(gpu(slots)).cpu().numpy(), want)
    out = remnant.mx4_gather_bf16(pool, gpu(slots, I32)[None], None)
    assert np.array_equal(out.double().cpu().numpy(), ref.decode_rows(want))
    # and a decode through a block table that names the last pages
    q = torch.randn(1, 1, 16, 512, generator=torch.Generator().manual_seed(1)).bfloat16()
    table = np.array([[pages - 1, 0]], np.int32)
    idx = np.concatenate([63 - np.arange(20), 64 + np.arange(20)]).astype(np.int32)[None, None]
    got = remnant.mx4_sparse_decode_fwd(q.to(DEV), pool, gpu(table), gpu(idx))
    small = np.zeros((2, 17408), np.uint8)
    small.reshape(-1, 272)[np.concatenate([64 + 63 - np.arange(20), np.arange(20)])] = want[
        np.concatenate([20 + np.arange(20), np.arange(20)])]
    check(got, ref.decode(q, small, np.array([[1, 0]]), idx))


# ---- reader ----

@pytest.mark.parametrize("queries,k", [(1, 1), (1, 700), (3, 37), (5, 5), (2, 20000), (70000, 1)])
def test_gather_is_exact(queries, k):
    banner(f"gather {queries} x {k}")
    rng = np.random.default_rng(k)
    pages = 7
    pool = random_pool(pages, k)
    pool.reshape(-1, 272)[::5, 256 + 3] = 255  # a NaN group
    slots = rng.integers(-2, pages * 64 + 2, (queries, k)).astype(np.int32)
    lengths = rng.integers(-1, k + 2, queries).astype(np.int32)
    wide = torch.zeros(queries, 2 * k, dtype=I32)
    wide[:, ::2] = torch.from_numpy(slots)
    out = torch.full((queries * k + 2, 512), -91.0, dtype=torch.bfloat16, device=DEV)
    two = torch.zeros(queries, 2, dtype=I32, device=DEV)
    two[:, 1] = gpu(lengths)
    remnant.mx4_gather_bf16(gpu(pool), wide.to(DEV)[:, ::2], two[:, 1], out)
    ok = (np.arange(k) < lengths[:, None]) & (slots >= 0) & (slots < pages * 64)
    values = ref.decode_rows(pool.reshape(-1, 272))[slots.clip(0, pages * 64 - 1)]
    want = np.where(ok[..., None], values, 0).reshape(-1, 512)
    assert np.array_equal(out[:-2].double().cpu().numpy(), want, equal_nan=True)
    assert (out[-2:] == -91).all()  # rows behind the last query
    plain = remnant.mx4_gather_bf16(gpu(pool), gpu(slots), None)
    ok = (slots >= 0) & (slots < pages * 64)
    want = np.where(ok[..., None], values, 0).reshape(-1, 512)
    assert np.array_equal(plain.double().cpu().numpy(), want, equal_nan=True)


# ---- decode ----

def check(got, want, where=""):
    out, lse = (t.double().cpu().numpy() for t in got)
    ref_out, ref_lse, tol, ltol = want
    inf = np.isinf(ref_lse)
    assert np.array_equal(lse[inf], ref_lse[inf]), where
    with np.errstate(invalid="ignore"):
        off, loff = np.abs(out - ref_out) - tol, np.where(inf, 0, np.abs(lse - ref_lse) - ltol)
    assert not np.isnan(off).any() and not np.isnan(loff).any(), where
    print(f"  out {np.max(np.abs(out - ref_out) / np.maximum(tol, 1e-30)):.3f} of its tolerance, "
          f"lse {np.max(np.where(inf, 0, np.abs(lse - np.where(inf, 0, ref_lse))) / np.maximum(ltol, 1e-30)):.3f}",
          flush=True)
    assert (off <= 1e-30).all() and (loff <= 0).all(), where


class Case:
    """A paged request batch with ragged lists; everything numpy, `run` sends it."""

    def __init__(self, heads, topk, *, batch=3, q_len=1, context=500, seed=0, window=0, q=0.5,
                 full=False, sigma=1.0):
        rng = np.random.default_rng(seed * 7 + heads * 31 + topk)
        contexts = [context] + [int(c) for c in rng.integers(0, context + 1, batch - 1)]
        self.table, pages = syn.paged_requests([max(c, 1) for c in contexts], seed, None)
        self.pool = random_pool(pages + 1, seed, sigma)
        tokens = batch * q_len
        self.q = (torch.randn(batch, q_len, heads, 512, generator=torch.Generator()
                              .manual_seed(seed)) * q).bfloat16()
        # entries at random (twice the same among them), padding and records past the request
        self.indices = rng.integers(0, context, (batch, q_len, topk)).astype(np.int32)
        if not full:
            self.indices[rng.random(self.indices.shape) < 0.1] = -1
            self.indices[rng.random(self.indices.shape) < 0.05] = 2 ** 31 - 1
        self.kw = dict(seqlens=np.array(contexts, np.int32),
                       topk_length=rng.integers(0, topk + 1, tokens).astype(np.int32),
                       sink=rng.standard_normal(heads).astype(np.float32))
        if full:
            self.kw["topk_length"][:] = topk
        if window:
            self.kw["swa_pool"] = native_pool(4, seed)
            w = rng.integers(-1, 4 * 64 + 2, (batch, q_len, window)).astype(np.int32)
            self.kw |= dict(swa_indices=w,
                            swa_lengths=rng.integers(0, window + 1, tokens).astype(np.int32))

    def run(self, **more):
        kw = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in self.kw.items()}
        return remnant.mx4_sparse_decode_fwd(self.q.to(DEV), gpu(self.pool), gpu(self.table),
                                             gpu(self.indices), **(kw | more))

    def want(self, **more):
        kw = dict(self.kw)
        if "swa_pool" in kw and kw["swa_pool"] is not None:
            kw["swa_pool"] = kw["swa_pool"].layer().cpu().numpy()
        return ref.decode(self.q, self.pool, self.table, self.indices, **(kw | more))


@pytest.mark.parametrize("topk", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257,
                                  511, 513, 1024, 2049])
@pytest.mark.parametrize("heads", [16, 1, 24])
def test_decode_list_lengths(heads, topk):
    banner(f"decode heads {heads} topk {topk}")
    case = Case(heads, topk, seed=topk)
    check(case.run(), case.want())
    full = Case(heads, topk, seed=topk + 1, full=True, batch=2)
    check(full.run(), full.want())


@pytest.mark.parametrize("heads", [2, 8, 15, 17, 32, 48, 64, 128])
def test_decode_head_counts(heads):
    banner(f"decode heads {heads}")
    case = Case(heads, 150, batch=2, q_len=2, seed=heads, window=20)
    check(case.run(), case.want())


@pytest.mark.parametrize("window", [1, 15, 16, 17, 63, 64, 65, 128, 300, 512])
@pytest.mark.parametrize("topk", [0, 40, 600])
def test_decode_window(topk, window):
    banner(f"decode topk {topk} window {window}")
    case = Case(16, topk, q_len=2, seed=window, window=window)
    check(case.run(), case.want())
    case.kw["swa_lengths"] = None
    case.kw["sink"] = None
    check(case.run(), case.want())


@pytest.mark.parametrize("batch,q_len,topk", [(40, 1, 300), (128, 2, 70), (1, 4, 5000), (2, 1, 20000),
                                              (9, 3, 1111), (300, 1, 33)])
def test_decode_batches(batch, q_len, topk):
    banner(f"decode batch {batch} x {q_len} topk {topk}")
    case = Case(16, topk, batch=batch, q_len=q_len, seed=batch, context=2000)
    check(case.run(), case.want())


@pytest.mark.parametrize("batch,heads,topk,window", [
    (128, 16, 2048, 0),    # records past the caches
    (64, 64, 5000, 0),     # the same, forty rounds a workgroup, each record for four of them
    (32, 128, 5000, 40),   # forty rounds through the caches, the window behind them
    (260, 16, 200, 100),   # more tokens than workgroups at once, the window behind the list
    (300, 16, 1000, 0), (300, 16, 1000, 30), (90, 48, 700, 5),  # the last of them split
    (20, 16, 2000, 512),   # splits, and the window in a workgroup of its own
    (3, 1000, 70, 20), (1, 1024, 300, 0)])
def test_decode_forms(batch, heads, topk, window):
    """Sizes at which the kernel shares its work out in another way, some tokens of each
    against the definition."""
    banner(f"decode batch {batch} heads {heads} topk {topk} window {window}")
    case = Case(heads, topk, batch=batch, seed=batch, window=window, context=40)
    rng = np.random.default_rng(batch)
    case.pool = random_pool(90, 5)
    case.table = rng.integers(0, 90, (batch, 31)).astype(np.int32)
    case.kw["seqlens"] = rng.integers(1500, 31 * 64 + 1, batch).astype(np.int32)
    case.kw["topk_length"][:] = rng.integers(topk * 3 // 4, topk + 1, batch)
    case.indices = rng.integers(-20, 31 * 64, case.indices.shape).astype(np.int32)
    out, lse = case.run()
    assert out.isfinite().all() and lse.isfinite().all()
    some = sorted({0, batch // 2, batch - 1})
    part = {k: v if k in ("sink", "swa_pool") or v is None else v[some] for k, v in case.kw.items()}
    if window:
        part["swa_pool"] = case.kw["swa_pool"].layer().cpu().numpy()
    check((out[some], lse[some]),
          ref.decode(case.q[some], case.pool, case.table[some], case.indices[some], **part))


@pytest.mark.parametrize("copies", [1, 3, 40, 700])
def test_decode_of_one_record_is_that_record(copies):
    """Weights of one record alone, also many times over, cancel: its values, exactly."""
    banner(f"decode one record x {copies}")
    case = Case(16, copies, batch=2, seed=copies, full=True, q=1.0)
    case.kw["seqlens"][:] = 500
    case.indices[:] = 37
    case.kw["sink"] = None
    out, lse = case.run()
    rec = case.pool.reshape(-1, 272)[case.table[:, 0] * 64 + 37]
    want = np.broadcast_to(ref.decode_rows(rec)[:, None, None], out.shape)
    assert np.array_equal(out.double().cpu().numpy(), want)
    check((out, lse), case.want())


def test_decode_wide_block_table():
    """More columns than the kernel keeps at hand, lists that use the last of them."""
    banner("decode wide table")
    for columns in (1024, 1025, 3000):
        case = Case(16, 700, batch=2, seed=columns, context=40, window=30)
        rng = np.random.default_rng(columns)
        case.pool = random_pool(40, 6)
        case.table = rng.integers(0, 40, (2, columns)).astype(np.int32)
        case.table[:, rng.integers(0, columns, 50)] = -1
        case.kw["seqlens"][:] = [columns * 64, columns * 64 - 70]
        case.kw["topk_length"][:] = 700
        case.indices = rng.integers(0, columns * 64 + 40, case.indices.shape).astype(np.int32)
        case.indices[..., 5] = columns * 64 - 1
        check(case.run(), case.want(), f"{columns} columns")


@pytest.mark.parametrize("pages", [130000, 246723, 246724, 300000])
def test_decode_and_reader_far_in_the_pool(pages):
    """Records past 2 and 4 GiB, by either way of forming their addresses: the bits of the
    same records in a small pool."""
    banner(f"decode far, {pages} pages")
    case = Case(16, 400, batch=2, seed=11, context=2000, full=True)
    near = case.pool.shape[0]
    pool = torch.zeros(pages, 17408, dtype=torch.uint8, device=DEV)
    pool[pages - near:] = gpu(case.pool)
    want = case.run()
    check(want, case.want())
    kw = {k: gpu(v) for k, v in case.kw.items()}
    table = gpu(np.where(case.table >= 0, case.table + pages - near, -1))
    got = remnant.mx4_sparse_decode_fwd(case.q.to(DEV), pool, table, gpu(case.indices), **kw)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    slots = torch.arange(near * 64, dtype=I32, device=DEV)[None]
    far = remnant.mx4_gather_bf16(pool, slots + (pages - near) * 64, None)
    assert torch.equal(far, remnant.mx4_gather_bf16(gpu(case.pool), slots, None))


def test_decode_rows_with_nothing():
    """Lists and windows that leave no row: zeros, the sink alone, or -inf."""
    banner("decode empty rows")
    case = Case(16, 64, seed=3, window=8)
    for sink in (case.kw["sink"], None, np.full(16, -np.inf, np.float32)):
        case.kw["sink"] = sink
        case.kw["topk_length"][:] = 0
        case.kw["swa_lengths"][:] = 0
        check(case.run(), case.want())
        case.kw["topk_length"][:] = -5
        case.kw["swa_lengths"][:] = 99  # past the list's end: all of it
        check(case.run(), case.want())
        case.kw["topk_length"][:] = 1 << 30
        case.kw["seqlens"][:] = 0
        check(case.run(), case.want())
        case.kw["seqlens"][:] = -1
        case.kw["swa_lengths"][:] = 0
        out, lse = case.run()
        assert (out == 0).all()
        # the sink times log2(e) and ln(2): two rounded constants, two rounded products,
        # half a step (2^-24) each
        alone = gpu(np.full(16, -np.inf, np.float32) if sink is None else sink)
        assert torch.allclose(lse, alone.expand(3, 1, 16), rtol=2.0 ** -22, atol=0)
    empty = Case(16, 0, seed=4)
    check(empty.run(), empty.want())


def test_decode_unmapped_pages_and_short_tables():
    banner("decode unmapped")
    case = Case(16, 300, seed=6)
    case.table[0, 2] = -1
    case.table[1, 0] = 1 << 26
    case.table[2, 0] = case.pool.shape[0]  # one past the pool
    check(case.run(), case.want())
    case.kw["seqlens"] = None
    case.table = case.table[:, :3]
    check(case.run(), case.want())
    wide = torch.zeros(3, 9, dtype=I32, device=DEV)
    wide[:, :3] = gpu(case.table)
    kw = {k: gpu(v) for k, v in case.kw.items() if v is not None}
    got = remnant.mx4_sparse_decode_fwd(case.q.to(DEV), gpu(case.pool), wide[:, :3],
                                        gpu(case.indices), **kw)
    check(got, case.want())


def test_decode_ignores_what_is_not_selected():
    """NaN groups, NaN codes and any bytes in records that no list names, and in those
    named only by entries past the lists' ends."""
    banner("decode unselected records")
    case = Case(16, 100, seed=8, window=30)
    plain = [t.clone() for t in case.run()]
    used = set()
    for b in range(3):
        for k, r in enumerate(case.indices[b, 0]):
            if k < case.kw["topk_length"][b] and 0 <= r < case.kw["seqlens"][b]:
                used.add(int(case.table[b, r // 64]) * 64 + int(r) % 64)
    rec = case.pool.reshape(-1, 272)
    rec[[s for s in range(rec.shape[0]) if s not in used]] = 0xFF
    w = case.kw["swa_indices"][:, 0]
    named = {int(s) for b in range(3) for s in w[b, :case.kw["swa_lengths"][b]]}
    buf = case.kw["swa_pool"].buffer[0]
    for s in range(256):
        if s not in named:
            page, row = divmod(s, 64)
            buf[page, row * 576:(row + 1) * 576] = 0xFF
            buf[page, 64 * 576 + row * 8:64 * 576 + row * 8 + 8] = 0xFF
    for a, b in zip(case.run(), plain):
        assert torch.equal(a, b)


def test_decode_nan_group_poisons_its_token_alone():
    banner("decode NaN group")
    case = Case(16, 50, seed=9, full=True)
    case.kw["seqlens"][:] = 500
    case.indices[:] = case.indices % 64  # mapped for every request
    rec = case.pool.reshape(-1, 272)
    before = [t.clone() for t in case.run()]
    rec[int(case.table[1, 0]) * 64 + int(case.indices[1, 0, 49]), 256 + 15] = 255
    out, lse = case.run()
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    for b in (0, 2):
        assert torch.equal(out[b], before[0][b]) and torch.equal(lse[b], before[1][b])
    # a list of nothing but such records, with and without a sink, in one split and in many
    rec[:, 256] = 255
    for topk in (1, 50):
        case.indices = case.indices[..., :topk].copy()
        case.kw["topk_length"][:] = topk
        for sink in (case.kw["sink"], None):
            out, lse = case.run(sink=None if sink is None else gpu(sink))
            assert torch.isnan(out).all() and torch.isnan(lse).all()
    long = Case(16, 4000, seed=9, full=True, batch=1)
    long.pool.reshape(-1, 272)[:, 256] = 255
    for sink in (None, gpu(long.kw["sink"])):
        out, lse = long.run(sink=sink)
        assert torch.isnan(out).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("q", [1e-3, 8.0, 300.0])
def test_decode_flat_and_peaked_scores(q):
    """Scores from nearly equal to a spread of thousands, climbing along the list."""
    banner(f"decode q {q}")
    case = Case(16, 1500, seed=11, q=q, context=1500, full=True, batch=2)
    check(case.run(), case.want())
    # ascending scores of head 0, so that the maximum moves all the way along the list
    rows = ref.decode_rows(case.pool.reshape(-1, 272)[
        (case.table[0].repeat(64)[:1500].astype(np.int64) * 64 + np.arange(1500) % 64)])
    case.indices[0, 0] = np.argsort(rows @ case.q[0, 0, 0].double().numpy())
    check(case.run(), case.want())
    case.indices[0, 0] = case.indices[0, 0, ::-1]
    check(case.run(), case.want())
    check(case.run(softmax_scale=-0.125), case.want(scale=-0.125))
    check(case.run(softmax_scale=0.0), case.want(scale=0.0))


@pytest.mark.parametrize("sigma", [2.0 ** -13, 2.0 ** 20, 2.0 ** 31])
def test_decode_small_and_large_latents(sigma):
    banner(f"decode sigma {sigma}")
    case = Case(16, 200, seed=12, sigma=sigma, q=min(1.0, 1 / sigma))
    check(case.run(), case.want())


def test_decode_mixed_scales_between_records():
    """Records 2^25 apart in one list: the small ones' coordinates still count where a
    group of the large ones is zero."""
    banner("decode mixed scales")
    rng = np.random.default_rng(13)
    case = Case(16, 96, seed=13, full=True, batch=1, context=128, q=2.0 ** -12)
    x = rng.standard_normal((128, 512)) * np.where(np.arange(128) % 2, 2.0 ** 12, 2.0 ** -12)[:, None]
    x[1::2, 64:128] = 0
    pool = case.pool.reshape(-1, 272)
    slot = case.table[0].repeat(64)[:128].astype(np.int64) * 64 + np.arange(128) % 64
    pool[slot] = ref.encode(ref.bf16(x))
    case.kw["topk_length"] = None
    check(case.run(), case.want())


def test_decode_is_the_same_every_time():
    banner("decode repeats")
    for case in (Case(16, 2000, batch=4, context=2000, seed=14), Case(64, 300, seed=15, window=64)):
        first = [t.clone() for t in case.run()]
        for _ in range(5):
            for a, b in zip(case.run(), first):
                assert torch.equal(a, b)


def test_decode_of_one_token_does_not_depend_on_the_batch_behind_it():
    """Token 0 alone and in a batch: equal to rounding (the split plan may differ)."""
    banner("decode batch of one")
    case = Case(16, 500, batch=20, context=800, seed=16)
    out, lse = case.run()
    kw = {k: gpu(v[:1] if k != "sink" else v) for k, v in case.kw.items()}
    one = remnant.mx4_sparse_decode_fwd(case.q[:1].to(DEV), gpu(case.pool), gpu(case.table[:1]),
                                        gpu(case.indices[:1]), **kw)
    want = case.want()
    first = tuple(w[:1] for w in want)
    check(one, first)
    check((out[:1], lse[:1]), first)


def test_decode_outputs_in_place_and_workspace():
    banner("decode out/lse/workspace")
    case = Case(16, 3000, batch=2, context=3000, seed=17, window=33)
    splits, need = remnant.get_mx4_decode_metadata(2, 16, 3000, 33)
    assert splits >= 1 and (need > 0) == (splits > 1)
    out = torch.full((4, 1, 16, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((4, 1, 16), 7.0, device=DEV)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    got = case.run(out=out[1:3], lse=lse[1:3], workspace=ws[:need])
    check(got, case.want())
    assert got[0].data_ptr() == out[1:].data_ptr()
    assert (out[0] == 7).all() and (out[3] == 7).all() and (lse[0] == 7).all() and (lse[3] == 7).all()
    assert (ws[need:] == 0xFF).all()
    for a, b in zip(case.run(workspace=torch.empty(8, dtype=torch.uint8, device=DEV)), got):
        assert torch.equal(a, b)


def test_tensors_of_two_devices_are_refused():
    banner("two devices")
    pool = remnant.LatentPool(2, fmt="mx4", device=DEV)
    x, w, n = torch.zeros(4, 512), torch.ones(512), torch.zeros(4, dtype=I32)
    with pytest.raises(ValueError, match="same GPU"):
        remnant.mx4_store_rows(x.to(DEV), w, 1e-6, n.to(DEV), None, None, pool)
    with pytest.raises(ValueError, match="same GPU"):
        remnant.mx4_gather_bf16(pool, n[None], None)
    with pytest.raises(ValueError, match="same GPU"):
        remnant.window_slots(n[None].to(DEV), n[:1], 1, 4)
    with pytest.raises(ValueError, match="same GPU"):
        remnant.append_slots(n[None].to(DEV), n[:1].to(DEV), n[:1].to(DEV), n, rows=2)
    case = Case(16, 20, batch=1, seed=1)
    with pytest.raises(ValueError, match="same GPU"):
        case.run(sink=torch.zeros(16))
    with pytest.raises(ValueError, match="same GPU"):
        case.run(workspace=torch.zeros(1 << 20, dtype=torch.uint8))


def test_configured_dispatch_reaches_the_4bit_decode():
    banner("dispatch")
    case = Case(16, 64, seed=18)
    try:
        remnant.configure_cache_format("mx4")
        kw = {k: gpu(v) for k, v in case.kw.items()}
        got = remnant.sparse_decode_fwd(case.q.to(DEV), gpu(case.pool), gpu(case.table),
                                        gpu(case.indices), freqs_cis=None, **kw)
    finally:
        remnant.configure_cache_format("native")
    for a, b in zip(got, case.run()):
        assert torch.equal(a, b)


def test_host_cache_round_trip():
    banner("host cache")
    pool = remnant.LatentPool(4, layers=3, fmt="mx4", device=DEV)
    pool.buffer.copy_(torch.randint(0, 256, pool.buffer.shape, dtype=torch.uint8))
    host = remnant.HostLatentPool.like(pool, pages=2)
    src = gpu([200, 3, 255, -1, 64, 0], I32)
    dst = gpu([5, 127, 0, 4, 128, 66], I32)
    host.backup_from_device_all_layer(pool, dst, src)
    torch.cuda.synchronize()
    for layer in range(3):
        rec = host.buffer[layer].view(-1, 272)
        for s, d in ((200, 5), (3, 127), (255, 0), (0, 66)):
            assert torch.equal(rec[d], pool.buffer[layer].view(-1, 272)[s].cpu())
        assert (rec[4] == 0).all()
    back = remnant.LatentPool(4, layers=3, fmt="mx4", device=DEV)
    host.load_to_device_per_layer(back, dst, src, 1)
    got, want = back.buffer[1].view(-1, 272), pool.buffer[1].view(-1, 272)
    keep = [200, 3, 255, 0]
    assert torch.equal(got[keep], want[keep]) and int((got != 0).any(1).sum()) <= 4
    assert (back.buffer[0] == 0).all()


# ---- together, graphs, streams ----

class Serving:
    """A few requests' pools, tables and lengths, stepped through the public calls: C4
    records (4-bit) and window tokens (Native) written and attended each step."""

    def __init__(self, batch=3, heads=16, topk=48, window=20, first=3):
        self.b, self.heads, self.topk, self.window, self.first = batch, heads, topk, window, first
        self.c4 = remnant.LatentPool(16, fmt="mx4", device=DEV)
        self.swa = remnant.LatentPool(32, fmt="native", device=DEV)
        self.c4_table = torch.full((batch, 4), -1, dtype=I32, device=DEV)
        self.swa_table = torch.full((batch, 12), -1, dtype=I32, device=DEV)
        self.c4_free = torch.randperm(16, generator=torch.Generator().manual_seed(2)).to(I32).to(DEV)
        self.swa_free = torch.randperm(32, generator=torch.Generator().manual_seed(3)).to(I32).to(DEV)
        self.len = torch.zeros(batch, dtype=I32, device=DEV)
        self.weight = torch.linspace(0.5, 1.5, 512, device=DEV)
        self.freqs = syn.rope_freqs(4 * 256).to(DEV)
        self.sink = torch.linspace(-1, 1, heads, device=DEV)
        self.c4_taken = self.swa_taken = 0

    def step(self, new_len, x4, xw, q, indices):
        """x4 / xw: compressor and window rows (rows past the step's are padding)."""
        c4 = remnant.append_slots(self.c4_table, self.len, new_len, self.c4_free, ratio=4,
                                  rows=x4.shape[0])
        swa = remnant.append_slots(self.swa_table, self.len, new_len, self.swa_free,
                                   rows=xw.shape[0])
        remnant.mx4_store_rows(x4, self.weight, 1e-6, c4.loc, c4.positions, self.freqs, self.c4)
        remnant.native_store_rows(xw, self.weight, 1e-6, swa.loc, None, None, self.swa)
        slots, counts = remnant.window_slots(self.swa_table, new_len, 1, self.window,
                                             first=self.first)
        out, lse = remnant.mx4_sparse_decode_fwd(
            q, self.c4, self.c4_table, indices, seqlens=c4.seqlens, sink=self.sink,
            swa_pool=self.swa, swa_indices=slots, swa_lengths=counts)
        return c4, swa, slots, counts, out, lse


def test_serving_steps_together():
    """A prefill and several decode steps: every step's outputs against float64 attention
    over rows re-derived from the raw inputs."""
    banner("serving steps")
    s = Serving()
    g = torch.Generator().manual_seed(7)
    rows4, rowsw = [[] for _ in range(3)], [[] for _ in range(3)]
    length = np.zeros(3, np.int64)
    for step, grow in enumerate(([37, 258, 0], [1, 1, 5], [3, 0, 1], [7, 60, 130])):
        after = length + np.array(grow)
        n4 = (after // 4 - length // 4).tolist()
        x4 = syn.latents(sum(n4) + 3, seed=step)
        xw = syn.latents(sum(grow) + 2, seed=100 + step)
        q = (torch.randn(3, 1, 16, 512, generator=g) * 0.5).bfloat16()
        idx = np.full((3, 1, 48), -1, np.int32)
        for b in range(3):
            held = int(after[b] // 4)
            pick = np.random.default_rng(step * 9 + b).permutation(held)[:48]
            idx[b, 0, :len(pick)] = pick
        got = s.step(gpu(after, I32), x4.to(DEV), xw.to(DEV), q.to(DEV), gpu(idx))
        c4, swa, slots, counts, out, lse = got
        a4 = aw = 0
        for b in range(3):
            rows4[b].append(x4[a4:a4 + n4[b]])
            rowsw[b].append(xw[aw:aw + grow[b]])
            a4 += n4[b]
            aw += grow[b]
        assert (c4.loc[a4:] == -1).all() and (swa.loc[aw:] == -1).all()
        assert c4.seqlens.tolist() == (after // 4).tolist()
        # the same attention from the raw rows alone, in pools of the test's own
        pool4 = np.zeros((3 * 4 * 64, 272), np.uint8)
        poolw = remnant.LatentPool(3 * 8, fmt="native", device=DEV)
        widx = np.full((3, 1, 23), -1, np.int32)
        for b in range(3):
            x = torch.cat(rows4[b])
            pool4[b * 256:b * 256 + len(x)] = ref.store_rows(x, s.weight.cpu().numpy(), 1e-6,
                                                             np.arange(len(x)), s.freqs.cpu())
            x = torch.cat(rowsw[b])
            at = torch.arange(len(x), dtype=I32, device=DEV) + b * 512
            remnant.native_store_rows(x.to(DEV), s.weight, 1e-6, at, None, None, poolw)
            t = np.arange(after[b])
            seen = t[(t < 3) | (t > after[b] - 1 - 20)]
            assert counts[b] == len(seen)
            widx[b, 0, :len(seen)] = seen + b * 512
        table = np.arange(12).reshape(3, 4)
        check((out, lse), ref.decode(q, pool4.reshape(12, -1), table, idx, after // 4, None,
                                     s.sink.cpu().numpy(), None, poolw.layer().cpu().numpy(), widx))
        s.c4_free = s.c4_free[int(c4.pages_taken):].contiguous()
        s.swa_free = s.swa_free[int(swa.pages_taken):].contiguous()
        s.len.copy_(gpu(after, I32))
        length = after


def test_serving_step_in_a_graph_replays_with_new_inputs():
    """One captured step replayed with other lengths, rows, queries and lists, eager steps
    of a second instance and synchronizations between; two graphs that were captured one
    after the other and run alternately."""
    banner("serving graph")
    shape = dict(x4=(6, 512), xw=(24, 512), q=(3, 1, 16, 512))

    def static():
        s = Serving()
        s.start = torch.tensor([200, 5, 63], dtype=I32)  # tokens held before a step
        for t in ("c4", "swa"):
            ratio, taken = (4, 0) if t == "c4" else (1, 0)
            rows = 512
            remnant.append_slots(getattr(s, t + "_table"), torch.zeros(3, dtype=I32, device=DEV),
                                 s.start.to(DEV), getattr(s, t + "_free"), ratio=ratio, rows=rows)
        s.c4_free, s.swa_free = s.c4_free[3:].contiguous(), s.swa_free[6:].contiguous()
        s.c4.buffer.copy_(gpu(random_pool(16, 21)))
        s.swa.buffer.copy_(native_pool(32, 22).buffer)
        s.len.copy_(s.start)
        s.ins = dict(new=torch.zeros(3, dtype=I32, device=DEV),
                     idx=torch.zeros(3, 1, 48, dtype=I32, device=DEV),
                     **{k: torch.zeros(v, device=DEV, dtype=torch.bfloat16)
                        for k, v in shape.items()})
        return s

    def feed(s, seed):
        g = torch.Generator().manual_seed(seed)
        s.ins["new"].copy_(s.start + torch.randint(0, 8, (3,), generator=g))
        s.ins["idx"].copy_(torch.randint(-1, 55, (3, 1, 48), generator=g))
        for k, v in shape.items():
            s.ins[k].copy_(torch.randn(v, generator=g))

    def go(s):
        return s.step(s.ins["new"], s.ins["x4"], s.ins["xw"], s.ins["q"], s.ins["idx"])

    eager, graphs = static(), []
    for _ in range(2):
        s = static()
        feed(s, 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = go(s)
        graphs.append((s, graph, outs))
    for seed in range(1, 7):
        feed(eager, seed)
        want = go(eager)
        flat = lambda r: [*r[0], *r[1], *r[2:]]  # noqa: E731
        for s, graph, outs in graphs:
            feed(s, seed)
            graph.replay()
            if seed % 2:
                torch.cuda.synchronize()
            for a, b in zip(flat(outs), flat(want)):
                assert torch.equal(a, b)
            assert torch.equal(s.c4_table, eager.c4_table)
            assert torch.equal(s.swa_table, eager.swa_table)


def test_two_streams_at_once():
    banner("two streams")
    cases = [Case(16, 2000, batch=4, context=2000, seed=30), Case(64, 600, seed=31, window=64)]
    wants = [[t.clone() for t in c.run()] for c in cases]
    ins = []
    for c in cases:
        kw = {k: gpu(v) if isinstance(v, np.ndarray) else v for k, v in c.kw.items()}
        ins.append(((c.q.to(DEV), gpu(c.pool), gpu(c.table), gpu(c.indices)), kw))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(remnant.mx4_sparse_decode_fwd(*ins[i][0], **ins[i][1]))
    torch.cuda.synchronize()
    for want, outs in zip(wants, got):
        for o in outs:
            for a, b in zip(o, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("byte", [0, 1, 111, 112, 159])
def test_decode_reads_scale_bytes_up_to_the_reference(byte):
    """Bytes the store does not write, below its own: exact, as the reader gives them."""
    banner(f"decode scale byte {byte}")
    case = Case(16, 300, seed=17, full=True, q=2.0 ** -33 if byte == 159 else 0.5)
    rec = case.pool.reshape(-1, 272)
    rng = np.random.default_rng(byte)
    rec[::3, 256 + rng.integers(0, 16, len(rec[::3]))] = byte
    check(case.run(), case.want())


@pytest.mark.parametrize("byte", [160, 191, 223, 254, 255])
def test_decode_of_scales_past_the_reference_is_nan(byte):
    """In any group, in either half of a chunk, by itself or among others: the token is
    NaN, the others are as before."""
    banner(f"decode scale byte {byte}")
    case = Case(16, 64, seed=18, full=True)
    case.kw["seqlens"][:] = 500
    case.indices[:] = np.random.default_rng(18).permutation(64)  # mapped for every request
    rec = case.pool.reshape(-1, 272)
    before = [t.clone() for t in case.run()]
    plain = rec.copy()
    for group in range(16):
        rec[:] = plain
        rec[int(case.table[1, 0]) * 64 + int(case.indices[1, 0, (37 * group) % 64]), 256 + group] = byte
        out, lse = case.run()
        assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all(), group
        for b in (0, 2):
            assert torch.equal(out[b], before[0][b]) and torch.equal(lse[b], before[1][b])
    # in many splits, whatever the codes are (also zero), with and without a sink
    long = Case(16, 4000, seed=19, full=True, batch=1)
    at = long.pool.reshape(-1, 272)[int(long.table[0, 0]) * 64 + 5]
    long.indices[0, 0, 1234] = 5
    at[:256], at[256 + 7] = 0, byte
    for sink in (None, gpu(long.kw["sink"])):
        out, lse = long.run(sink=sink)
        assert torch.isnan(out).all() and torch.isnan(lse).all()
