"""GPU tests of the index operators: store bit-exact, reader exact, scores within derived
tolerances and selections equal to the plain definitions (index_reference.py); the steps of
a serving loop that score, select and attend; graphs and streams."""

import numpy as np
import pytest
import torch

import index_reference as ref
import mx4_reference
import remnant
from remnant import synthetic as syn

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = torch.int32
KEY = 128


def banner(msg):
    print(f"[gpu-index] {msg}", flush=True)


def gpu(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype).to(DEV)


def keys(rows, seed, dtype=torch.float32):
    return syn.latents(rows, seed=seed)[:, :KEY].float().contiguous().to(dtype)


def random_pool(pages, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((pages * 64, KEY)) * np.exp(rng.uniform(-2, 2, KEY))
    return ref.make_pool(*ref.codes_of(ref.bf16(x / np.sqrt((x * x).mean(1, keepdims=True)))))


# ---- store ----

def store(x, slots, pages, weight=None, eps=1e-6, positions=None, freqs=None, ratio=4, fill=0x5A):
    pool = remnant.LatentPool(pages, fmt="index", device=DEV)
    pool.buffer.fill_(fill)
    w = torch.ones(KEY) if weight is None else weight
    remnant.index_store_rows(x.to(DEV), w.float().to(DEV), eps, gpu(slots, I32),
                             None if positions is None else gpu(positions, I32),
                             None if freqs is None else freqs.to(DEV), pool, ratio=ratio)
    torch.cuda.synchronize()
    return pool.layer().cpu().numpy()


def expect(x, slots, pages, weight=None, eps=1e-6, positions=None, freqs=None, ratio=4, fill=0x5A):
    pool = np.full((pages, 8448), fill, np.uint8)
    slots = np.asarray(slots, np.int64)
    ok = (slots >= 0) & (slots < pages * 64)
    if freqs is not None:
        row = np.asarray(positions, np.int64) * ratio
        ok &= (row >= 0) & (row < freqs.shape[0])
        positions = np.asarray(positions)[ok]
    w = np.ones(KEY, np.float32) if weight is None else weight.float().numpy()
    codes, scales = ref.store_rows(x[torch.from_numpy(ok)], w, eps, positions, freqs, ratio)
    page, row = slots[ok] // 64, slots[ok] % 64
    pool[:, :8192].reshape(pages, 64, KEY)[page, row] = codes
    scale_bytes = np.ascontiguousarray(scales).view(np.uint8).reshape(-1, 4)
    # (numpy's NaN and the kernel's are the same bits)
    pool[:, 8192:].reshape(pages, 64, 4)[page, row] = scale_bytes
    return pool


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 5, 64, 1000, 70001])
def test_store_is_bit_exact(rows, dtype):
    banner(f"store {rows} {dtype}")
    rng = np.random.default_rng(rows)
    x = keys(rows, rows) * torch.pow(2.0, torch.randint(-20, 20, (rows, 1)).float())
    x = x.to(dtype)
    pages = rows // 64 + 2
    slots = rng.permutation(pages * 64)[:rows].astype(np.int32)
    slots[2::17] = -1
    slots[5::31] = pages * 64 + 3
    weight = torch.linspace(0.5, 1.5, KEY)
    freqs = syn.rope_freqs(4 * 500)
    for ratio in (4, 1):
        args = dict(weight=weight, positions=rng.integers(-1, 2000 // ratio + 1, rows), freqs=freqs,
                    ratio=ratio)
        assert np.array_equal(store(x, slots, pages, **args), expect(x, slots, pages, **args))
    assert np.array_equal(store(x, slots, pages, weight), expect(x, slots, pages, weight))


def test_store_special_rows():
    """Zeros, ties of every code, the largest and smallest magnitudes, infinities and NaN,
    which stay in their own rows; strided rows."""
    banner("store special rows")
    rows = torch.zeros(16, KEY)
    rows[1] = 1.0
    rows[2] = torch.arange(KEY) * 0.125 + 16
    rows[3] = -rows[2] / 64
    rows[4] = 3e38
    rows[5] = 1e-38
    rows[6, 7] = float("inf")
    rows[7, 70] = float("nan")
    rows[8] = torch.where(torch.arange(KEY) == 3, 1e30, 1e-30)
    rows[9] = torch.where(torch.arange(KEY) % 32 == 0, 448.0, 0.25)
    rows[10] = -0.0
    rows[11:] = torch.randn(5, KEY, generator=torch.Generator().manual_seed(3))
    wide = torch.zeros(16, 1024)
    wide[:, 512:512 + KEY] = rows
    big = torch.ones(KEY)
    big[32:64] = 1e12
    big[96] = float("inf")
    for x in (rows, rows.bfloat16(), wide[:, 512:512 + KEY]):
        for weight in (None, big):
            for eps in (1e-6, 0.0, 1e-30):
                got = store(x, np.arange(16), 1, weight, eps)
                want = expect(x, np.arange(16), 1, weight, eps)
                assert np.array_equal(got[:, :8192], want[:, :8192]), eps
                a, b = (np.ascontiguousarray(t[:, 8192:]).view(np.float32) for t in (got, want))
                assert np.array_equal(a, b, equal_nan=True), eps


def test_store_of_one_row_of_any_stride():
    """The distance to a next row is nobody's business where there is none."""
    banner("store one row")
    x = keys(1, 12)
    wide = torch.zeros(3, 129, device=DEV)
    wide[0, :KEY] = x[0].to(DEV)
    want = expect(x, [5], 1)
    for one in (x.to(DEV).t().contiguous().t(), wide[:1, :KEY], x.to(DEV).expand(4, KEY)[1:2]):
        assert one.shape == (1, KEY)
        assert np.array_equal(store(one, [5], 1), want), one.stride()
        assert np.array_equal(store(one.bfloat16().as_strided((1, KEY), (1, 1)), [5], 1),
                              expect(x.bfloat16(), [5], 1))


def test_store_and_reader_past_4_gib():
    banner("store far slots")
    pages = 520000  # 4.4 GB
    pool = remnant.LatentPool(pages, fmt="index", device=DEV)
    x = keys(40, 5)
    slots = np.concatenate([np.arange(20), pages * 64 - 1 - np.arange(20)])
    remnant.index_store_rows(x.to(DEV), torch.ones(KEY, device=DEV), 1e-6, gpu(slots, I32), None,
                             None, pool)
    codes, scales = ref.store_rows(x, np.ones(KEY), 1e-6)
    want = ref.levels()[codes] * scales[:, None]
    out = remnant.index_gather_bf16(pool, gpu(slots, I32)[None], None)
    assert np.array_equal(out.double().cpu().numpy(), want)
    # and scores through a block table that names the last page
    q = torch.randn(1, 1, 16, KEY, generator=torch.Generator().manual_seed(1)).bfloat16()
    w = torch.linspace(-1, 1, 16).reshape(1, 1, 16)
    table = np.array([[pages - 1, 0]], np.int32)
    got = remnant.index_scores(q.to(DEV), w.to(DEV), pool, gpu(table), gpu([84], I32))
    small = np.zeros((2, 8448), np.uint8)
    for page, at in ((0, 20), (1, 0)):
        small[page] = pool.layer()[pages - 1 if page == 0 else 0].cpu().numpy()
    check_scores(got, ref.scores(q, w.numpy(), small, np.array([[0, 1]]), [84], 128))


def test_store_of_more_rows_than_a_launch():
    """2^28 rows, 16 a workgroup of 256 threads, likewise; most have no slot."""
    banner("store 2^28 + 21 rows")
    rows = (1 << 28) + 21
    x = torch.empty(rows, KEY, dtype=torch.bfloat16, device=DEV)  # 69 GB
    slots = torch.full((rows,), -1, dtype=I32, device=DEV)
    at = [0, 1, (1 << 27) - 1, 1 << 27, (1 << 28) - 1, 1 << 28, rows - 1]
    some = keys(len(at), 8, torch.bfloat16)
    for i, row in enumerate(at):
        x[row] = some[i].to(DEV)
        slots[row] = 3 * i
    pool = remnant.LatentPool(1, fmt="index", device=DEV)
    pool.buffer.fill_(0x5A)
    remnant.index_store_rows(x, torch.ones(KEY, device=DEV), 1e-6, slots, None, None, pool)
    got = pool.layer().cpu().numpy()
    del x, slots
    torch.cuda.empty_cache()
    assert np.array_equal(got, expect(some, np.arange(len(at)) * 3, 1))


# ---- reader ----

@pytest.mark.parametrize("queries,k", [(1, 1), (1, 700), (3, 37), (5, 5), (2, 20000), (70000, 1)])
def test_gather_is_code_times_scale(queries, k):
    banner(f"gather {queries} x {k}")
    rng = np.random.default_rng(k)
    pages = 7
    pool = rng.integers(0, 256, (pages, 8448)).astype(np.uint8)  # every code, NaN among them
    scales = (2.0 ** rng.uniform(-40, 40, pages * 64)).astype(np.float32)
    scales[::7] = np.nan
    scales[3::11] *= -1
    pool[:, 8192:] = scales.reshape(pages, 64).view(np.uint8)
    slots = rng.integers(-2, pages * 64 + 2, (queries, k)).astype(np.int32)
    lengths = rng.integers(-1, k + 2, queries).astype(np.int32)
    wide = torch.zeros(queries, 2 * k, dtype=I32)
    wide[:, ::2] = torch.from_numpy(slots)
    out = torch.full((queries * k + 2, KEY), -91.0, dtype=torch.bfloat16, device=DEV)
    two = torch.zeros(queries, 2, dtype=I32, device=DEV)
    two[:, 1] = gpu(lengths)
    remnant.index_gather_bf16(gpu(pool), wide.to(DEV)[:, ::2], two[:, 1], out)
    codes, scales = ref.page_rows(pool)
    values = ref.levels()[codes].astype(np.float32) * scales[:, None]  # rounded to float32, then
    values = ref.bf16(values)
    ok = (np.arange(k) < lengths[:, None]) & (slots >= 0) & (slots < pages * 64)
    want = np.where(ok[..., None], values[slots.clip(0, pages * 64 - 1)], 0).reshape(-1, KEY)
    assert np.array_equal(out[:-2].float().cpu().numpy(), want, equal_nan=True)
    assert (out[-2:] == -91).all()  # rows behind the last query
    plain = remnant.index_gather_bf16(gpu(pool), gpu(slots), None)
    ok = (slots >= 0) & (slots < pages * 64)
    want = np.where(ok[..., None], values[slots.clip(0, pages * 64 - 1)], 0).reshape(-1, KEY)
    assert np.array_equal(plain.float().cpu().numpy(), want, equal_nan=True)


# ---- scores ----

def check_scores(got, want, where=""):
    got, (out, tol) = got.double().cpu().numpy(), want
    fine = np.isfinite(out)
    assert np.array_equal(got[~fine], out[~fine], equal_nan=True), where
    off = np.abs(got[fine] - out[fine])
    assert np.isfinite(off).all(), where
    if off.size:
        print(f"  {np.max(off / np.maximum(tol[fine], 1e-30)):.3f} of its tolerance", flush=True)
    assert (off <= tol[fine]).all(), where


class Scored:
    def __init__(self, heads, context, *, batch=2, q_len=1, seed=0, holes=True):
        rng = np.random.default_rng(seed * 7 + heads * 31 + context)
        contexts = [context] + [int(c) for c in rng.integers(0, context + 1, batch - 1)]
        self.table, pages = syn.paged_requests([max(c, 1) for c in contexts], seed, None)
        self.pool = random_pool(pages + 1, seed)
        self.q = (torch.randn(batch, q_len, heads, KEY, generator=torch.Generator()
                              .manual_seed(seed)) * 2).bfloat16()
        self.weights = rng.standard_normal((batch, q_len, heads)).astype(np.float32)
        self.lengths = np.repeat(contexts, q_len) - rng.integers(0, 4, batch * q_len)
        self.lengths[0] = context
        if holes and self.table.shape[1] > 1:
            self.table[0, self.table.shape[1] // 2] = rng.choice([-1, pages + 1, 1 << 30])
        self.width = self.table.shape[1] * 64

    def run(self, out=None):
        return remnant.index_scores(self.q.to(DEV), gpu(self.weights), gpu(self.pool),
                                    gpu(self.table), gpu(self.lengths, I32), out=out)

    def want(self, width=None):
        return ref.scores(self.q, self.weights, self.pool, self.table, self.lengths,
                          self.width if width is None else width)


@pytest.mark.parametrize("heads", [1, 8, 16, 17, 24, 32, 40, 64, 65, 128])
@pytest.mark.parametrize("q_len", [1, 2, 5])
def test_scores_heads(heads, q_len):
    banner(f"scores {heads} heads, {q_len} queries")
    case = Scored(heads, 333, q_len=q_len, seed=heads)
    check_scores(case.run(), case.want())


@pytest.mark.parametrize("q_len", [1, 2, 3, 7, 31, 32, 33, 64, 65, 130])
def test_scores_queries(q_len):
    banner(f"scores {q_len} queries")
    case = Scored(64, 200, batch=3, q_len=q_len, seed=q_len)
    check_scores(case.run(), case.want())


@pytest.mark.parametrize("context", [1, 2, 63, 64, 65, 129, 4097, 20000])
def test_scores_lengths(context):
    banner(f"scores {context} records")
    for heads, q_len, batch in ((64, 1, 1), (8, 33, 2), (16, 2, 5)):
        case = Scored(heads, context, batch=batch, q_len=q_len, seed=context)
        check_scores(case.run(), case.want())


def test_scores_of_many_requests():
    banner("scores 700 requests")
    case = Scored(16, 100, batch=700, seed=5)
    check_scores(case.run(), case.want())


@pytest.mark.parametrize("heads, q_len, batch", [(64, 1, 45), (20, 3, 21), (100, 2, 13)])
def test_scores_of_ragged_requests(heads, q_len, batch):
    """Long and short requests in one call, where a wave takes several pages at least and
    most waves of the short ones have none."""
    banner(f"scores ragged {heads} heads, {q_len} queries")
    case = Scored(heads, 21000, batch=batch, q_len=q_len, seed=batch)
    case.lengths[q_len:] = np.minimum(case.lengths[q_len:],
                                      np.arange(case.lengths.size - q_len) * 97 % 1500 - 3)
    check_scores(case.run(), case.want())


def test_scores_of_more_tokens_than_a_grid_dimension():
    """33,000 requests of 3 tokens are 66,000 rows of workgroups."""
    banner("scores 33,000 requests")
    batch, q_len = 33000, 3
    rng = np.random.default_rng(4)
    pool = random_pool(3, 4)
    q = (torch.randn(batch, q_len, 1, KEY, generator=torch.Generator().manual_seed(4)) * 2).bfloat16()
    weights = rng.standard_normal((batch, q_len, 1)).astype(np.float32)
    table = rng.integers(0, 3, (batch, 1))
    lengths = rng.integers(0, 6, batch * q_len)
    got = remnant.index_scores(q.to(DEV), gpu(weights), gpu(pool), gpu(table, I32),
                               gpu(lengths, I32), out=torch.empty(batch, q_len, 5, device=DEV))
    some = np.concatenate([np.arange(40), rng.integers(40, batch, 200), np.arange(batch - 40, batch)])
    want = ref.scores(q[some], weights[some], pool, table[some],
                      lengths.reshape(batch, q_len)[some].reshape(-1), 5)
    check_scores(got[torch.from_numpy(some).to(DEV)], want)


@pytest.mark.parametrize("heads, q_len, batch, context", [
    (128, 33, 2, 700), (65, 130, 1, 900),                             # eight tiles, tokens apart
    (32, 5, 11, 20000), (24, 31, 2, 20000),                           # two tiles, four tokens a wave
    (32, 67, 1, 20000), (17, 130, 1, 9000),                           # the same, apart
    (1, 9, 6, 20000), (16, 31, 2, 20000), (16, 8, 7, 19999),          # one tile, eight tokens
    (3, 35, 1, 31000), (64, 34, 1, 700), (40, 7, 3, 900)])
def test_scores_of_many_tokens(heads, q_len, batch, context):
    """Tokens that are no multiple of what a wave or workgroup takes, at sizes where those
    take as many as they can; lengths that differ widely between the tokens of a wave, and
    pages that are not mapped."""
    banner(f"scores {heads} heads, {q_len} tokens of {batch} x {context}")
    case = Scored(heads, context, batch=batch, q_len=q_len, seed=heads + q_len)
    rng = np.random.default_rng(q_len)
    case.lengths = np.where(rng.random(case.lengths.size) < 0.3,
                            rng.integers(-2, context + 1, case.lengths.size), case.lengths)
    case.lengths[0] = context
    case.table[:, 1] = -1
    check_scores(case.run(), case.want())


@pytest.mark.parametrize("width", [1, 63, 65, 127, 200, 700])
def test_scores_width(width):
    """Columns fewer than the table's records, more, and no whole pages; what stands
    around the output stays."""
    banner(f"scores width {width}")
    case = Scored(16, 333, batch=2, q_len=3, seed=width)
    case.lengths[1], case.lengths[2], case.lengths[3] = 0, -5, 1 << 30
    whole = torch.full((2 * 3 * width + 64,), 7.0, device=DEV)
    out = whole[32:-32].view(2, 3, width)
    assert case.run(out=out) is out
    check_scores(out, case.want(width))
    assert (whole[:32] == 7).all() and (whole[-32:] == 7).all()


def test_scores_without_heads_records_or_pages():
    banner("scores of nothing")
    case = Scored(16, 70, holes=False)
    case.q, case.weights = case.q[:, :, :0], case.weights[:, :, :0]
    got = case.run().cpu()
    live = torch.arange(case.width) < torch.from_numpy(case.lengths)[:, None]
    assert (got[:, 0][live] == 0).all() and (got[:, 0][~live] == -torch.inf).all()
    case = Scored(16, 70)
    case.pool = case.pool[:0]
    assert (case.run() == -torch.inf).all()
    case.table = case.table[:, :0]
    out = torch.zeros(2, 1, 40, device=DEV)
    assert (case.run(out=out) == -torch.inf).all()


def test_scores_keep_nan_to_themselves():
    """A NaN code, scale, weight or query coordinate gives NaN where it takes part and
    nowhere else; what lies past the lengths does not take part."""
    banner("scores NaN")
    for heads, q_len in ((16, 3), (64, 40)):
        case = Scored(heads, 200, batch=2, q_len=q_len, seed=3, holes=False)
        case.lengths[:] = 190
        case.pool[int(case.table[0, 0]), 5 * KEY + 17] = 0x7F
        case.pool[int(case.table[0, 1]), 9 * KEY + 100] = 0xFF
        slot = int(case.table[1, 0])
        case.pool[slot, 8192 + 4 * 7:8192 + 4 * 8] = np.float32([np.nan]).view(np.uint8)
        case.pool[int(case.table[0, 2]), 62 * KEY:64 * KEY] = 0x7F  # records 190 and 191: past
        case.q[0, 1, 3, 40] = float("inf")
        case.q[1, 2, 0, 3] = float("nan")
        case.weights[1, 0, 2] = np.nan
        want = case.want()
        # (a query's infinity or NaN is NaN for all of its row's scores that there are)
        for b, j in ((0, 1), (1, 2), (1, 0)):
            line = want[0][b, j]
            line[line != -np.inf] = np.nan
        got = case.run().cpu().numpy()
        assert np.isnan(want[0]).any() and not np.isnan(want[0]).all()
        check_scores(torch.from_numpy(got), want)


def test_scores_with_records_written_elsewhere():
    """Any finite scale, negative ones too; queries of every magnitude."""
    banner("scores any scale")
    case = Scored(32, 300, batch=2, q_len=2, seed=8)
    rng = np.random.default_rng(1)
    scale = (2.0 ** rng.uniform(-30, 30, len(case.pool) * 64)).astype(np.float32)
    scale[::5] *= -1
    case.pool[:, 8192:] = scale.reshape(-1, 64).view(np.uint8)
    case.q = (case.q.float() * torch.pow(2.0, torch.randint(-30, 30, (2, 2, 32, 1)).float())).bfloat16()
    case.q[0, 0, 5] = 0
    check_scores(case.run(), case.want())


# ---- selection ----

def check_topk(x, lengths, k, **kw):
    idx, counts = remnant.index_topk(x, None if lengths is None else gpu(lengths, I32), k, **kw)
    want, n = ref.topk(x.reshape(-1, x.shape[-1]).cpu().numpy(), lengths, k)
    assert np.array_equal(counts.cpu().numpy(), n)
    assert np.array_equal(idx.cpu().numpy().reshape(want.shape), want)


WIDTHS = [1, 2, 63, 257, 1000, 2047, 2048, 2049, 8191, 8193, 20000, 32768, 32769, 100003]


@pytest.mark.parametrize("width", WIDTHS)
def test_topk_sizes(width):
    banner(f"topk width {width}")
    rng = np.random.default_rng(width)
    x = gpu(rng.standard_normal((7, width)).astype(np.float32))
    lengths = np.array([width, 0, -3, width + 5, width // 2, max(width - 1, 0), 1])
    for k in sorted({0, 1, 2, 37, width // 2, width - 1, width, width + 3}):
        check_topk(x, lengths, k)
    check_topk(x, None, min(64, width))


@pytest.mark.parametrize("width", [4095, 4096, 4097, 8192, 16384, 16385, 65536, 65537])
def test_topk_around_the_threads_and_turns(width):
    """Both sides of the widths and of the k that other numbers of threads, turns and places
    for the keys begin at."""
    banner(f"topk around {width}")
    rng = np.random.default_rng(width)
    x = gpu(rng.standard_normal((3, width)).astype(np.float32))
    lengths = np.array([width, width - 1, width // 3])
    for k in (1, 512, 1024, 1025, 2048, 2049):
        check_topk(x, lengths, k)


@pytest.mark.parametrize("rows", [1023, 1024])
def test_topk_of_a_full_chip(rows):
    banner(f"topk of {rows} rows of 5,000")
    rng = np.random.default_rng(rows)
    x = gpu(rng.standard_normal((rows, 5000)).astype(np.float32))
    check_topk(x, rng.integers(0, 5001, rows), 300)


def shapes(rng, n):
    """Rows that a histogram of equal bins finds hard."""
    x = np.zeros((20, n), np.float32)
    x[0] = 1.5                                             # all equal
    x[1] = rng.integers(0, 2, n)                           # two values
    x[2] = rng.integers(-3, 4, n)                          # few values
    x[3] = np.where(np.arange(n) % 2, 0.0, -0.0)           # equal, by the sign of zero apart
    x[4] = rng.standard_normal(n)
    x[4, rng.integers(n)] = 3e38                           # one far out
    x[5] = 1 + rng.random(n) * 1e-5                        # close together
    x[6] = rng.standard_normal(n) * 1e-40                  # subnormal
    x[7] = np.exp(rng.uniform(-80, 80, n)) * rng.choice([-1, 1], n)
    x[8] = np.where(rng.random(n) < 0.5, -np.inf, rng.standard_normal(n))
    x[9] = -np.inf
    x[10] = np.inf
    x[11] = np.where(rng.random(n) < 0.3, np.nan, rng.standard_normal(n))
    x[12] = np.nan
    x[13] = np.finfo(np.float32).min                       # the lowest finite value ...
    x[13, ::3] = -np.inf                                   # ... and below it
    x[14] = np.arange(n)                                   # sorted
    x[15] = -np.arange(n)
    x[16] = np.sort(rng.standard_normal(n))[::-1]
    x[17] = np.frombuffer((np.arange(n) + 0x3F800000).astype(np.int32).tobytes(), np.float32)
    x[18] = np.where(np.arange(n) == n - 1, 2.0, 1.0)      # the last one
    x[19] = np.where(rng.random(n) < 0.01, np.inf, np.where(rng.random(n) < 0.5, np.nan, 0))
    return x


@pytest.mark.parametrize("width", [50, 2000, 8000, 30000, 50000])
def test_topk_distributions(width):
    banner(f"topk distributions {width}")
    rng = np.random.default_rng(width)
    x = gpu(shapes(rng, width))
    lengths = np.where(np.arange(20) % 3 == 2, width - 7, width)
    for k in (1, 33, width // 4, width - 9):
        check_topk(x, lengths, k)


def test_topk_does_not_read_past_the_lengths():
    banner("topk dead scores")
    rng = np.random.default_rng(4)
    for width in (1500, 5000, 40000):
        x = rng.standard_normal((3, width)).astype(np.float32)
        lengths = np.array([width // 3, width // 2 + 1, 600])
        for fill in (np.inf, np.nan, 3e38):
            for i, n in enumerate(lengths):
                x[i, n:] = fill
            check_topk(gpu(x), lengths, 512)


def test_topk_of_strided_rows():
    """Rows of a wider array, their start at any multiple of four bytes; batches."""
    banner("topk strides")
    rng = np.random.default_rng(5)
    whole = gpu(rng.standard_normal((4, 3, 6001)).astype(np.float32))
    for lo, hi in ((0, 6001), (0, 6000), (1, 5000), (2, 2002), (3, 4), (4, 4000)):
        view = whole[..., lo:hi]
        check_topk(view, rng.integers(0, hi - lo + 1, 12), 300)
        check_topk(view[0], rng.integers(0, hi - lo + 1, 3), 300)
        check_topk(view[1:2], None, 77)
    check_topk(whole[:, :1, 5:900], None, 50)
    check_topk(gpu(rng.standard_normal((2, 4000)).astype(np.float32))[:, 3:2051], None, 9)


def test_topk_outputs_in_place():
    banner("topk out")
    x = torch.randn(2, 3, 900, device=DEV)
    whole = torch.full((2 * 3 * 40 + 64,), 77, dtype=I32, device=DEV)
    counts = torch.full((10,), 77, dtype=I32, device=DEV)
    out = (whole[32:-32].view(2, 3, 40), counts[2:8])
    check_topk(x, np.array([900, 5, 0, 39, 40, 41]), 40, out=out)
    assert (whole[:32] == 77).all() and (whole[-32:] == 77).all()
    assert (counts[:2] == 77).all() and (counts[8:] == 77).all()


def test_topk_of_many_rows_and_no_rows():
    banner("topk rows")
    x = torch.randn(70000, 9, device=DEV)
    check_topk(x, None, 4)
    idx, counts = remnant.index_topk(x[:, :0], None, 4)
    assert (idx == -1).all() and (counts == 0).all()


def test_topk_of_more_rows_than_a_launch():
    """2^24 rows of 256 threads are as many threads as a launch cannot have."""
    banner("topk 2^24 + 5 rows")
    rows = (1 << 24) + 5
    x = torch.randn(rows, 2, device=DEV, generator=torch.Generator(DEV).manual_seed(6))
    idx, counts = remnant.index_topk(x, None, 1)
    assert torch.equal(idx[:, 0], (x[:, 1] > x[:, 0]).to(I32)) and (counts == 1).all()


# ---- host cache ----

def test_host_cache_round_trip():
    banner("host cache")
    pool = remnant.LatentPool(4, layers=3, fmt="index", device=DEV)
    pool.buffer.copy_(torch.randint(0, 256, pool.buffer.shape, dtype=torch.uint8))
    host = remnant.HostLatentPool.like(pool, pages=2)
    src, dst = gpu([200, 3, 255, -1, 64, 0], I32), gpu([5, 127, 0, 4, 128, 66], I32)
    host.backup_from_device_all_layer(pool, dst, src)
    torch.cuda.synchronize()
    shape = remnant.LatentPool(2, layers=3, fmt="index", device="cpu")
    shape.buffer.copy_(host.buffer)
    pairs = ((200, 5), (3, 127), (255, 0), (0, 66))
    for layer in range(3):
        got = shape.records(torch.tensor([d for _, d in pairs]), layer)
        want = pool.records(gpu([s for s, _ in pairs]), layer).cpu()
        assert torch.equal(got, want)
        rest = torch.tensor(sorted(set(range(128)) - {d for _, d in pairs}))
        assert (shape.records(rest, layer) == 0).all()
    back = remnant.LatentPool(4, layers=3, fmt="index", device=DEV)
    host.load_to_device_per_layer(back, dst, src, 1)
    keep = gpu([200, 3, 255, 0])
    assert torch.equal(back.records(keep, 1), pool.records(keep, 1))
    assert int((back.buffer[1] != 0).sum()) <= 4 * 132 and (back.buffer[0] == 0).all()


# ---- together, graphs, streams ----

class Loop:
    """Requests whose records are stored, scored, selected and attended each step: index
    keys and 4-bit latents in one block table."""

    def __init__(self, batch=3, heads=16, index_heads=64, topk=24, q_len=2):
        self.batch, self.topk, self.q_len = batch, topk, q_len
        self.keys = remnant.LatentPool(16, fmt="index", device=DEV)
        self.latents = remnant.LatentPool(16, fmt="mx4", device=DEV)
        self.table = torch.full((batch, 5), -1, dtype=I32, device=DEV)
        self.free = torch.randperm(16, generator=torch.Generator().manual_seed(2)).to(I32).to(DEV)
        self.len = torch.zeros(batch, dtype=I32, device=DEV)
        self.taken = torch.zeros(1, dtype=I32, device=DEV)
        self.key_weight = torch.linspace(0.5, 1.5, KEY, device=DEV)
        self.weight = torch.linspace(0.5, 1.5, 512, device=DEV)
        self.freqs = syn.rope_freqs(4 * 320).to(DEV)
        self.sink = torch.linspace(-1, 1, heads, device=DEV)
        self.back = torch.arange(q_len - 1, -1, -1, dtype=I32, device=DEV)

    def step(self, new_len, key_rows, latent_rows, iq, iw, q):
        slots = remnant.append_slots(self.table, self.len, new_len, self.free, ratio=4,
                                     rows=key_rows.shape[0], taken=self.taken)
        remnant.index_store_rows(key_rows, self.key_weight, 1e-6, slots.loc, slots.positions,
                                 self.freqs, self.keys)
        remnant.mx4_store_rows(latent_rows, self.weight, 1e-6, slots.loc, slots.positions,
                               self.freqs, self.latents)
        # records complete before each query token: (position + 1) / 4
        seen = ((new_len[:, None] - self.back).clamp_min(0) // 4).to(I32).reshape(-1)
        scores = remnant.index_scores(iq, iw, self.keys, self.table, seen)
        indices, counts = remnant.index_topk(scores, seen, self.topk)
        out, lse = remnant.mx4_sparse_decode_fwd(q, self.latents, self.table, indices,
                                                 seqlens=slots.seqlens, topk_length=counts,
                                                 sink=self.sink)
        self.taken.copy_(slots.pages_taken)
        self.len.copy_(new_len)
        return seen, scores, indices, counts, out, lse


def inputs(batch, q_len, rows, seed, index_heads=64, heads=16):
    g = torch.Generator().manual_seed(seed)
    return (keys(rows, seed), syn.latents(rows, seed=seed + 50),
            (torch.randn(batch, q_len, index_heads, KEY, generator=g) * 2).bfloat16(),
            torch.randn(batch, q_len, index_heads, generator=g) * 0.1,
            (torch.randn(batch, q_len, heads, 512, generator=g) * 0.5).bfloat16())


def test_serving_steps_together():
    """A prefill and several steps: scores against the raw rows' definition, selections of
    those scores, attention over the selected records."""
    banner("serving steps")
    loop = Loop()
    rows = [[] for _ in range(3)], [[] for _ in range(3)]
    length = np.zeros(3, np.int64)
    for step, grow in enumerate(([700, 258, 0], [2, 1, 5], [3, 0, 1], [70, 260, 130])):
        after = length + np.array(grow)
        n = (after // 4 - length // 4).tolist()
        kx, lx, iq, iw, q = inputs(3, 2, sum(n) + 3, step)
        seen, scores, indices, counts, out, lse = loop.step(
            gpu(after, I32), *(t.to(DEV) for t in (kx, lx, iq, iw, q)))
        at = 0
        codes, scales = np.zeros((16 * 64, KEY), np.uint8), np.zeros(16 * 64, np.float32)
        latent = np.zeros((16 * 64, 272), np.uint8)
        table = np.arange(15).reshape(3, 5)
        for b in range(3):
            rows[0][b].append(kx[at:at + n[b]])
            rows[1][b].append(lx[at:at + n[b]])
            at += n[b]
            k, x = torch.cat(rows[0][b]), torch.cat(rows[1][b])
            here = slice(b * 320, b * 320 + len(k))
            p = np.arange(len(k))
            codes[here], scales[here] = ref.store_rows(k, loop.key_weight.cpu().numpy(), 1e-6, p,
                                                       loop.freqs.cpu())
            latent[here] = mx4_reference.store_rows(x, loop.weight.cpu().numpy(), 1e-6, p,
                                                    loop.freqs.cpu())
        want_seen = np.maximum((after[:, None] - np.array([1, 0])) // 4, 0).reshape(-1)
        assert np.array_equal(seen.cpu().numpy(), want_seen)
        check_scores(scores, ref.scores(iq, iw.numpy(), ref.make_pool(codes, scales), table,
                                        want_seen, 320))
        check_topk(scores, want_seen, 24)
        want = mx4_reference.decode(q, latent.reshape(16, -1), table, indices.cpu().numpy(),
                                    after // 4, counts.cpu().numpy(), loop.sink.cpu().numpy())
        for got, w, tol in ((out, want[0], want[2]), (lse, want[1], want[3])):
            assert (np.abs(got.double().cpu().numpy() - w) <= tol + 1e-30).all()
        length = after


def test_serving_step_in_a_graph_is_a_step_a_replay():
    """A captured step replayed with other rows and queries, as one step after another,
    beside the same steps run eagerly; two graphs in turn."""
    banner("serving graph")
    start, grow, rows = [700, 5, 63], [1, 2, 5], 16

    def begin():
        loop = Loop()
        kx, lx, iq, iw, q = (t.to(DEV) for t in inputs(3, 2, 256, 9))
        loop.step(gpu(start, I32), kx, lx, iq, iw, q)
        return loop

    pairs = []
    for _ in range(2):
        eager, loop = begin(), begin()
        static = [t.to(DEV) for t in inputs(3, 2, rows, 0)]
        new = torch.zeros(3, dtype=I32, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # (a step of its own, and the state before it again)
            held = [t.clone() for t in (loop.len, loop.taken, loop.table, loop.keys.buffer,
                                        loop.latents.buffer)]
            new.copy_(loop.len + 1)
            loop.step(new, *static)
            for t, was in zip((loop.len, loop.taken, loop.table, loop.keys.buffer,
                               loop.latents.buffer), held):
                t.copy_(was)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = loop.step(new, *static)
        pairs.append((eager, loop, graph, static, new, outs))
    for turn in range(1, 6):
        for eager, loop, graph, static, new, outs in pairs:
            fresh = [t.to(DEV) for t in inputs(3, 2, rows, turn)]
            after = gpu(np.array(start) + turn * np.array(grow), I32)
            want = eager.step(after, *fresh)
            for s, f in zip(static, fresh):
                s.copy_(f)
            new.copy_(after)
            graph.replay()
            if turn % 2:
                torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b), turn
            assert torch.equal(loop.table, eager.table)


def test_two_streams_at_once():
    banner("two streams")
    cases = [Scored(64, 3000, batch=4, seed=30, holes=False), Scored(32, 900, q_len=40, seed=31)]
    ins = [(c.q.to(DEV), gpu(c.weights), gpu(c.pool), gpu(c.table), gpu(c.lengths, I32)) for c in cases]
    wants = []
    for i in ins:
        s = remnant.index_scores(*i)
        wants.append((s, *remnant.index_topk(s, i[4], 400)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                s = remnant.index_scores(*ins[i])
                got[i].append((s, *remnant.index_topk(s, ins[i][4], 400)))
    torch.cuda.synchronize()
    for want, outs in zip(wants, got):
        for o in outs:
            for a, b in zip(o, want):
                assert torch.equal(a, b)


def test_tensors_of_two_devices_are_refused():
    banner("two devices")
    case = Scored(16, 20, batch=1)
    with pytest.raises(ValueError, match="same GPU"):
        remnant.index_scores(case.q.to(DEV), torch.from_numpy(case.weights), gpu(case.pool),
                             gpu(case.table), gpu(case.lengths, I32))
    with pytest.raises(ValueError, match="same GPU"):
        remnant.index_topk(torch.zeros(2, 4, device=DEV), torch.zeros(2, dtype=I32), 2)
    with pytest.raises(ValueError, match="same GPU"):
        remnant.index_gather_bf16(gpu(case.pool), torch.zeros(1, 1, dtype=I32), None)
