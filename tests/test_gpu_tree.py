"""GPU tests of the attention of drafted trees, within derived tolerances of the plain
definition (index_reference.py): shapes, windows, histories, masks that leave nothing,
infinities and NaN in rows that some nodes do not see, far pages, graphs and streams; a
verification step that stores the drafted rows and attends them."""

import numpy as np
import pytest
import torch

import index_reference as ref
import remnant
from remnant import synthetic as syn

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = torch.int32


def banner(msg):
    print(f"[gpu-tree] {msg}", flush=True)


def gpu(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype).to(DEV)


def check(got, want, where=""):
    out, lse = (t.double().cpu().numpy() for t in got)
    ref_out, ref_lse, tol, ltol = want
    odd = ~np.isfinite(ref_lse)
    assert np.array_equal(lse[odd], ref_lse[odd], equal_nan=True), where
    nan = np.isnan(ref_out)
    assert np.array_equal(np.isnan(out), nan), where
    with np.errstate(invalid="ignore"):
        off = np.where(nan, 0, np.abs(out - ref_out) / np.maximum(tol, 1e-30))
        loff = np.where(odd, 0, np.abs(lse - ref_lse) / np.maximum(ltol, 1e-30))
    print(f"  out {off.max():.3f} of its tolerance, lse {loff.max():.3f}", flush=True)
    assert off.max() <= 1 and loff.max() <= 1, where


def random_parents(rng, batch, nodes):
    return np.array([[int(rng.integers(-1, j)) if j else -1 for j in range(nodes)]
                     for _ in range(batch)], np.int64).reshape(batch, nodes)


class Tree:
    def __init__(self, nodes, heads, *, batch=2, context=200, window=None, past=0, seed=0, sink=True,
                 q=0.5, parents=None):
        rng = np.random.default_rng(seed * 7 + heads * 31 + nodes + context)
        self.lengths = np.array([context] + [int(c) for c in rng.integers(0, context + 1, batch - 1)])
        self.table, pages = syn.paged_requests([int(n) + nodes for n in self.lengths], seed, None)
        self.pool = ref.random_native(pages + 1, seed)
        self.parents = random_parents(rng, batch, nodes) if parents is None else np.asarray(parents)
        self.window = window
        self.q = (torch.randn(batch, nodes, heads, 512, generator=torch.Generator()
                              .manual_seed(seed)) * q).bfloat16()
        self.sink = rng.standard_normal(heads).astype(np.float32) if sink else None
        self.past = None
        if past:
            n = np.array([past] + [int(c) for c in rng.integers(0, past + 1, batch - 1)])
            table, pages = syn.paged_requests([max(int(c), 1) for c in n], seed + 1, None)
            self.past = [ref.random_native(pages + 1, seed + 5), table, n]

    def args(self):
        kw = dict(window=self.window, sink=None if self.sink is None else gpu(self.sink))
        if self.past:
            kw |= dict(history_pool=gpu(self.past[0]), history_table=gpu(self.past[1], I32),
                       history_lengths=gpu(self.past[2], I32))
        return (self.q.to(DEV), gpu(self.pool), gpu(self.table, I32), gpu(self.lengths, I32),
                gpu(self.parents, I32)), kw

    def run(self, **more):
        a, kw = self.args()
        return remnant.tree_decode_fwd(*a, **(kw | more))

    def want(self, **kw):
        return ref.tree(self.q, self.pool, self.table, self.lengths, self.parents, self.window,
                        *(self.past or (None, None, None)), sink=self.sink, **kw)


@pytest.mark.parametrize("heads", [1, 3, 8, 16, 17, 24, 64, 128])
@pytest.mark.parametrize("nodes", [1, 2, 7])
def test_heads(nodes, heads):
    banner(f"{nodes} nodes, {heads} heads")
    case = Tree(nodes, heads, seed=heads)
    check(case.run(), case.want())


@pytest.mark.parametrize("nodes", [1, 4, 15, 16, 17, 33, 63, 64])
@pytest.mark.parametrize("window", [None, 20, 128])
def test_nodes(nodes, window):
    banner(f"{nodes} nodes, window {window}")
    case = Tree(nodes, 8, batch=3, window=window, seed=nodes)
    check(case.run(), case.want())


@pytest.mark.parametrize("context", [0, 1, 2, 15, 16, 17, 63, 64, 127, 128, 129, 700, 5000])
def test_lengths(context):
    banner(f"{context} committed")
    for window, past in ((None, 0), (64, 0), (None, 37), (128, context // 3)):
        case = Tree(5, 16, context=context, window=window, past=past, seed=context)
        check(case.run(), case.want())


@pytest.mark.parametrize("window", [1, 2, 3, 15, 16, 17, 31, 32, 64, 100, 1 << 20, (1 << 31) - 1])
def test_windows(window):
    """Chains and trees deeper than the window, whose nodes lose their ancestors too."""
    banner(f"window {window}")
    chain = np.arange(40)[None].repeat(2, 0) - 1
    for parents in (chain, None):
        case = Tree(40, 4, context=300, window=window, parents=parents, seed=window % 1000)
        check(case.run(), case.want())


@pytest.mark.parametrize("past", [1, 15, 16, 17, 64, 300, 2000])
def test_histories(past):
    banner(f"history {past}")
    for window in (None, 128):
        case = Tree(6, 16, batch=3, context=150, window=window, past=past, seed=past)
        case.past[2][1] = 0
        check(case.run(), case.want())


@pytest.mark.parametrize("batch", [1, 40, 300])
def test_batches(batch):
    banner(f"batch {batch}")
    case = Tree(4, 16, batch=batch, context=90, window=32, past=40, seed=batch)
    check(case.run(), case.want())


class Ragged(Tree):
    """A tree with given committed lengths, and histories."""

    def __init__(self, lengths, *, nodes=2, heads=4, window=None, past=None, seed=0):
        super().__init__(nodes, heads, batch=len(lengths), context=1, window=window, seed=seed)
        self.lengths = np.asarray(lengths)
        self.table, pages = syn.paged_requests([int(n) + nodes for n in lengths], seed, None)
        self.pool = ref.random_native(pages + 1, seed)
        if past is not None:
            table, pages = syn.paged_requests([max(int(c), 1) for c in past], seed + 1, None)
            self.past = [ref.random_native(pages + 1, seed + 5), table, np.asarray(past)]


@pytest.mark.parametrize("batch", [2, 5, 63, 64, 65, 129, 255, 256, 257, 300])
def test_ragged_batches(batch):
    """Rounds of all requests are dealt out to the workgroups: shares that begin and end
    anywhere in a request, several requests a share, and more requests than are dealt."""
    banner(f"{batch} ragged requests")
    rng = np.random.default_rng(batch)
    most = 30000 // batch
    case = Ragged(rng.integers(0, most, batch), seed=batch)
    check(case.run(), case.want())
    case = Ragged(rng.integers(0, most, batch), window=100, past=rng.integers(0, most, batch),
                  nodes=3, heads=3, seed=batch + 1)
    check(case.run(), case.want())


@pytest.mark.parametrize("batch", [2, 7, 30])
@pytest.mark.parametrize("at", [0, -1])
def test_a_long_request_among_short_ones(batch, at):
    """More shares than the workspace has places for a request's partials."""
    banner(f"one long of {batch}, at {at}")
    lengths = np.arange(batch) % 4
    lengths[at] = 20000
    case = Ragged(lengths, seed=batch)
    check(case.run(), case.want())
    window = Ragged(lengths[:, None].repeat(2, 1).reshape(-1)[:batch], window=64,
                    past=lengths[::-1], seed=batch)
    check(window.run(), window.want())


@pytest.mark.parametrize("nodes, heads", [(1, 1024), (20, 100), (64, 33), (64, 128)])
def test_many_tiles(nodes, heads):
    """More tiles of query rows than fill one turn of the chip: fewer shares, down to one."""
    banner(f"{nodes} x {heads}")
    case = Ragged([0, 333, 100], nodes=nodes, heads=heads, window=90, past=[70, 3, 0], seed=heads)
    check(case.run(), case.want())


@pytest.mark.parametrize("nodes, heads, batch", [(16, 16, 3), (63, 32, 3), (64, 32, 4), (40, 52, 3),
                                                 (64, 128, 3), (60, 160, 2), (64, 300, 1)])
def test_many_tiles_share_rounds(nodes, heads, batch):
    """8, 63, 64, 65, 256, 300 and 600 tiles of query rows whose requests' rounds are dealt
    out, to as many shares as there are for that many tiles (the last: one)."""
    banner(f"{nodes} x {heads} x {batch}, rounds dealt out")
    lengths = [1500, 0, 700, 90][:batch]
    for case in (Ragged(lengths, nodes=nodes, heads=heads, seed=heads),
                 Ragged(lengths, nodes=nodes, heads=heads, window=90, past=[900, 70, 0, 1200][:batch],
                        seed=heads + 1)):
        splits, need = remnant.get_tree_decode_metadata(
            batch, nodes, heads, case.table.shape[1], window=case.window,
            history_blocks=case.past[1].shape[1] if case.past else 0)
        assert (splits > 1 and need > 0) or nodes * heads > 512 * 32
        got = case.run()
        check(got, case.want())
        for a, b in zip(case.run(), got):
            assert torch.equal(a, b)


def test_padding_and_roots():
    """Padding by any number that is no parent, its descendants, trees of roots alone; a
    request without a live node."""
    banner("padding")
    parents = np.array([[-1, 0, -2, 2, 3, 1, 7, 6, -1], [-1] * 9, [-5, 1, 2, 3, 1 << 30, -1 << 31, 9, 8, 7],
                        [0, 0, -1, 2, 3, 4, 5, 6, 8]])
    for sink in (True, False):
        case = Tree(9, 16, batch=4, context=100, past=20, parents=parents, sink=sink, seed=2)
        got = case.run()
        check(got, case.want())
        dead = np.array([[p is None for p in ref.paths(row.tolist())] for row in parents])
        assert dead[2].all() and dead.any(1).tolist() == [True, False, True, True]
        assert (got[0].cpu()[torch.from_numpy(dead)] == 0).all()


def test_rows_that_see_nothing():
    """No page is mapped where the node looks: zeros, and lse of the sink or -inf."""
    banner("nothing seen")
    for sink in (True, False):
        case = Tree(3, 16, context=100, sink=sink, seed=4)
        case.table[:] = -1
        out, lse = case.run()
        assert (out == 0).all()
        want = torch.from_numpy(case.sink).expand(2, 3, 16) if sink else torch.full((2, 3, 16), -torch.inf)
        assert torch.allclose(lse.cpu(), want, atol=1e-5)
        case = Tree(3, 16, context=100, sink=sink, seed=4)
        case.pool = case.pool[:0]
        assert (case.run()[0] == 0).all()
        case.table = case.table[:, :0]
        assert (case.run()[0] == 0).all()


def test_unmapped_and_foreign_pages_are_not_seen():
    banner("holes")
    case = Tree(4, 16, batch=2, context=400, past=300, seed=6)
    case.table[0, 1], case.table[0, 3] = -1, len(case.pool)
    case.past[1][0, 2], case.past[1][1, 0] = 1 << 30, -7
    check(case.run(), case.want())
    # the drafted rows' own page
    case.table[1, int(case.lengths[1]) // 64:] = -1
    check(case.run(), case.want())
    # lengths past the tables, and negative ones
    case.lengths[0], case.past[2][0] = 10 ** 9, 10 ** 9
    check(case.run(), clipped(case))
    case.lengths[0], case.past[2][0] = -5, -5
    check(case.run(), case.want())


def clipped(case):
    """The same with lengths cut to the tables: what lies past them is not mapped."""
    rows = []
    for b in range(len(case.lengths)):
        n = min(int(case.lengths[b]), case.table.shape[1] * 64)
        past = min(int(case.past[2][b]), case.past[1].shape[1] * 64)
        rows.append(ref.tree(case.q[b:b + 1], case.pool, case.table[b:b + 1], [n],
                             case.parents[b:b + 1], case.window, case.past[0],
                             case.past[1][b:b + 1], [past], sink=case.sink))
    return [np.concatenate([r[i] for r in rows]) for i in range(4)]


def spoil(pool, table, b, position, how, rng):
    page, row = int(table[b, position // 64]), position % 64
    if how == "code":
        pool[page, row * 576 + int(rng.integers(448))] = rng.choice([0x7F, 0xFF])
    elif how == "tail":
        at = row * 576 + 448 + 2 * int(rng.integers(64))
        pool[page, at:at + 2] = np.array([rng.choice([0x7F80, 0xFF80, 0x7FC1])], np.uint16).view(np.uint8)
    else:
        pool[page, 64 * 576 + row * 8 + int(rng.integers(7))] = 255


@pytest.mark.parametrize("how", ["code", "tail", "scale"])
def test_infinities_and_nan_reach_only_those_who_see_them(how):
    """In a drafted row: its descendants; in a committed row at the window's edge: the
    shallow nodes; in rows behind the last drafted one, before the window, of the history
    past its length: nobody."""
    banner(f"special rows: {how}")
    rng = np.random.default_rng(len(how))
    parents = np.array([[-1, 0, 0, 1, 3, 2, -1, 6], [-1, 0, 1, 2, 3, 4, 5, 6]])
    for spot in ("drafted", "edge", "behind", "before", "past"):
        case = Tree(8, 16, context=200, window=50, past=100, parents=parents, seed=3)
        case.lengths[:] = 200
        case.table = np.arange(8).reshape(2, 4)[:, ::-1].copy()
        case.pool = ref.random_native(8, 3)
        clean = case.want()
        hit = np.zeros((2, 8), bool)
        if spot == "drafted":
            spoil(case.pool, case.table, 0, 203, how, rng)  # node 3: seen by 3 and 4
            hit[0, [3, 4]] = True
        elif spot == "edge":
            spoil(case.pool, case.table, 1, 153, how, rng)  # depth d sees 151 + d and up
            hit[1, :3] = True
        elif spot == "behind":
            for p in range(208, 216):
                spoil(case.pool, case.table, 0, p, how, rng)
        elif spot == "before":
            for p in range(128, 151):
                spoil(case.pool, case.table, 1, p, how, rng)
        else:
            case.past[2][0] = 90
            clean = case.want()
            for p in range(90, 100):
                spoil(case.past[0], case.past[1], 0, p, how, rng)
        got = case.run()
        want = [x.copy() for x in clean]
        for x in want[:2]:
            x[hit] = np.nan
        check(got, want, spot)


def test_whole_units_pass_nan_on():
    """A NaN in a committed row that every node sees: all of the request, and no other."""
    banner("NaN seen by all")
    case = Tree(3, 16, context=300, seed=9)
    case.lengths[:] = 300
    case.table = np.arange(10).reshape(2, 5)
    case.pool = ref.random_native(10, 9)
    want = case.want()
    for how, p in (("code", 70), ("tail", 100), ("scale", 33)):
        pool = case.pool.copy()
        if how == "tail":
            page = int(case.table[0, p // 64])
            pool[page, (p % 64) * 576 + 448:(p % 64) * 576 + 450] = np.array([0x7FC0], np.uint16).view(np.uint8)
        else:
            spoil(pool, case.table, 0, p, how, np.random.default_rng(1))
        a, kw = case.args()
        out, lse = remnant.tree_decode_fwd(a[0], gpu(pool), *a[2:], **kw)
        assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all(), how
        check((out[1:], lse[1:]), [x[1:] for x in want], how)


@pytest.mark.parametrize("context, window, past, split", [
    (300, None, 0, False), (300, None, 150, True), (300, 128, 150, False), (1300, None, 150, True)])
def test_infinities_in_whole_units(context, window, past, split):
    """An infinity that every node of a request sees, at rows of every unit: NaN for all of
    the request's outputs and sums, whatever its sign and the query rows' (half of the
    scores are -inf) and wherever the row lies in a unit; padding nodes stay zero, also
    with NaN queries; the other requests stay as they are."""
    banner(f"infinities seen by all, {context} committed, window {window}, history {past}")
    parents = np.array([[-1, 0, 0, -2, 1]] * 3)
    columns = (context + 5) // 64 + 1
    case = Tree(5, 16, batch=3, context=context, window=window, past=past, parents=parents, seed=21)
    case.lengths[:] = context
    case.table = np.arange(3 * columns).reshape(3, columns)
    case.pool = ref.random_native(3 * columns, 21)
    if past:
        case.past = [ref.random_native(9, 22), np.arange(9).reshape(3, 3), np.array([past] * 3)]
    splits = remnant.get_tree_decode_metadata(3, 5, 16, columns, window=window,
                                              history_blocks=3 if past else 0)[0]
    assert (splits > 1) == split
    spots = [(case.pool, case.table, p) for p in (0, 70, 143, 160, 180, 255, 285, 287, 295, 299, 640,
                                                  1023, 1290)
             if (context - 120 if window else 0) <= p < context]
    if past:
        spots += [(case.past[0], case.past[1], p) for p in (0, 17, 100, 149)]
    live = [0, 1, 2, 4]
    for filler in (1.0, torch.nan):
        case.q[:, 3] = filler
        want = case.want()
        check(case.run(), want)
        for pool, table, p in spots:
            for bits in (0x7F80, 0xFF80):
                page, at = int(table[1, p // 64]), (p % 64) * 576 + 448 + 2 * (p % 64)
                held = pool[page, at:at + 2].copy()
                pool[page, at:at + 2] = np.array([bits], np.uint16).view(np.uint8)
                out, lse = case.run()
                where = (filler, p, hex(bits))
                assert torch.isnan(out[1, live]).all() and torch.isnan(lse[1, live]).all(), where
                assert (out[1, 3] == 0).all() and torch.isfinite(lse[1, 3]).all(), where
                check((out[::2], lse[::2]), [x[::2] for x in want], where)
                pool[page, at:at + 2] = held


@pytest.mark.parametrize("sigma", [2.0 ** -12, 2.0 ** 20, 2.0 ** 60])
def test_small_and_large_rows(sigma):
    """Scales far from one: exponents of the weights, not values, carry them."""
    banner(f"sigma {sigma}")
    case = Tree(4, 16, context=150, past=40, seed=12, q=min(1.0, 1 / sigma))
    rng = np.random.default_rng(1)
    x = rng.standard_normal((len(case.pool) * 64, 512)) * sigma
    case.pool = ref.native_pages(ref.bf16(x.astype(np.float32)))
    if sigma > 1e10:  # (q in proportion: the other rows score next to nothing)
        case.past = None
    check(case.run(), case.want())


def test_every_scale_byte():
    """Records written elsewhere: one group's byte anything up to 254, the codes there zero
    or one in a row of its own."""
    banner("scale bytes")
    case = Tree(2, 16, batch=1, context=254, seed=13)
    case.table = np.arange(5)[None]
    pool = ref.random_native(5, 13)
    for p in range(254):
        page, row = p // 64, p % 64
        g = p % 7
        pool[page, 64 * 576 + row * 8 + g] = p
        codes = pool[page, row * 576 + 64 * g:row * 576 + 64 * g + 64]
        codes[:] = 0 if p > 140 else 0x38  # (a one times more than 2^13 outweighs the rest)
    case.pool = pool
    check(case.run(), case.want())


def test_scores_that_climb():
    """The largest score in the last rows, far above the others: the reference moves and
    what was summed is lowered; and a negative scale."""
    banner("climbing scores")
    case = Tree(3, 16, batch=1, context=1500, seed=14)
    case.table = np.arange(24)[None]
    x = ref.bf16(np.random.default_rng(2).standard_normal((24 * 64, 512)).astype(np.float32))
    x *= 2.0 ** (np.arange(24 * 64) // 100)[:, None]
    case.pool = ref.native_pages(x.astype(np.float32))
    case.q = (case.q.float() * 2.0 ** -9).bfloat16()
    check(case.run(), case.want())
    check(case.run(softmax_scale=-0.03), case.want(scale=-0.03))
    check(case.run(softmax_scale=0.0), case.want(scale=0.0))


def test_pool_past_4_gib():
    banner("far pages")
    pages = 120000  # 4.5 GB
    pool = torch.zeros(pages, 37376, dtype=torch.uint8, device=DEV)
    case = Tree(5, 16, batch=1, context=150, past=70, seed=15)
    far = np.array([[pages - 1, 3, pages - 2]])
    small = ref.random_native(3, 4)
    for i, page in enumerate(far[0]):
        pool[int(page)] = gpu(small[i])
    case.pool, case.table = small, np.arange(3)[None]
    a, kw = case.args()
    got = remnant.tree_decode_fwd(a[0], pool, gpu(far, I32), a[3], a[4], **kw)
    check(got, case.want())
    kw["history_pool"], kw["history_table"] = pool, gpu(far[:, :2], I32)
    case.past[0], case.past[1] = small, np.array([[0, 1]])
    check(remnant.tree_decode_fwd(a[0], pool, gpu(far, I32), a[3], a[4], **kw), case.want())


def test_layers_of_pools():
    banner("layers")
    case = Tree(4, 16, context=100, past=30, seed=16)
    pool = remnant.LatentPool(len(case.pool), layers=3, fmt="native", device=DEV)
    past = remnant.LatentPool(len(case.past[0]), layers=2, fmt="native", device=DEV)
    pool.buffer[2].copy_(gpu(case.pool))
    past.buffer[1].copy_(gpu(case.past[0]))
    a, kw = case.args()
    kw["history_pool"] = past
    got = remnant.tree_decode_fwd(a[0], pool, *a[2:], layer_id=2, history_layer_id=1, **kw)
    for x, y in zip(got, case.run()):
        assert torch.equal(x, y)


def test_outputs_in_place_and_workspace():
    banner("out/lse/workspace")
    case = Tree(8, 16, batch=1, context=3000, seed=17)
    splits, need = remnant.get_tree_decode_metadata(1, 8, 16, case.table.shape[1])
    assert splits > 1 and need > 0
    out = torch.full((3, 8, 16, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((3, 8, 16), 7.0, device=DEV)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    got = case.run(out=out[1:2], lse=lse[1:2], workspace=ws[:need])
    check(got, case.want())
    assert got[0].data_ptr() == out[1:].data_ptr()
    for t in (out, lse):
        assert (t[0] == 7).all() and (t[2] == 7).all()
    assert (ws[need:] == 0xFF).all()
    for a, b in zip(case.run(workspace=torch.empty(8, dtype=torch.uint8, device=DEV)), got):
        assert torch.equal(a, b)


def test_broadcast_tables_and_repeats():
    banner("one table row, repeats")
    case = Tree(8, 16, batch=1, context=900, past=200, seed=18)
    first = [t.clone() for t in case.run()]
    a, kw = case.args()
    wide = torch.full((3, 40), 5, dtype=I32, device=DEV)
    wide[1, :case.table.shape[1]] = gpu(case.table[0])
    got = remnant.tree_decode_fwd(*a[:2], wide[1:2, :case.table.shape[1]], *a[3:], **kw)
    for x, y in zip(got, first):
        assert torch.equal(x, y)
    for _ in range(5):
        for x, y in zip(case.run(), first):
            assert torch.equal(x, y)


def test_a_chain_is_the_native_decode():
    """One node after another with a window: the sparse decode over window_slots' lists."""
    banner("chain against the decode")
    batch, nodes, window = 3, 4, 100
    case = Tree(nodes, 16, batch=batch, context=300, window=window, seed=19,
                parents=np.arange(nodes)[None].repeat(batch, 0) - 1)
    a, kw = case.args()
    got = remnant.tree_decode_fwd(*a, **kw)
    slots, counts = remnant.window_slots(gpu(case.table, I32), gpu(case.lengths + nodes, I32), nodes, window)
    none = torch.zeros(batch, nodes, 0, dtype=I32, device=DEV)
    out, lse = remnant.native_sparse_decode_fwd(a[0], a[1], gpu(case.table), none, sink=kw["sink"],
                                                swa_pool=a[1], swa_indices=slots, swa_lengths=counts)
    want = case.want()
    check(got, want)
    assert (np.abs((out.float() - got[0].float()).cpu().numpy()) <= 0.02 + 0.02 * np.abs(want[0])).all()
    assert np.abs((lse - got[1]).cpu().numpy()).max() <= 0.02


class Verify:
    """A verification step: the drafted rows' slots, their store, and their attention."""

    def __init__(self, batch=3, nodes=6, heads=16, window=40):
        self.batch, self.nodes, self.window = batch, nodes, window
        self.pool = remnant.LatentPool(20, fmt="native", device=DEV)
        self.table = torch.full((batch, 6), -1, dtype=I32, device=DEV)
        self.free = torch.randperm(20, generator=torch.Generator().manual_seed(2)).to(I32).to(DEV)
        self.taken = torch.zeros(1, dtype=I32, device=DEV)
        self.len = torch.zeros(batch, dtype=I32, device=DEV)
        self.weight = torch.linspace(0.5, 1.5, 512, device=DEV)
        self.freqs = syn.rope_freqs(512).to(DEV)
        self.sink = torch.linspace(-1, 1, heads, device=DEV)

    def commit(self, new_len, rows):
        slots = remnant.append_slots(self.table, self.len, new_len, self.free, rows=rows.shape[0],
                                     taken=self.taken)
        remnant.native_store_rows(rows, self.weight, 1e-6, slots.loc, slots.positions, self.freqs,
                                  self.pool, ratio=1)
        self.taken.copy_(slots.pages_taken)
        self.len.copy_(new_len)

    def draft(self, rows, depths, q, parents):
        slots = remnant.append_slots(self.table, self.len, self.len + self.nodes, self.free,
                                     rows=rows.shape[0], taken=self.taken)
        at = (self.len.repeat_interleave(self.nodes) + depths.reshape(-1)).to(I32)
        remnant.native_store_rows(rows, self.weight, 1e-6, slots.loc, at, self.freqs, self.pool,
                                  ratio=1)
        return remnant.tree_decode_fwd(q, self.pool, self.table, self.len, parents,
                                       window=self.window, sink=self.sink)


def test_verification_steps_together():
    """Committed and drafted rows written by the store at their positions in the text; the
    attention against float64 over the stored pages."""
    banner("verification steps")
    v = Verify()
    length = np.zeros(3, np.int64)
    rng = np.random.default_rng(1)
    for step, grow in enumerate(([130, 7, 60], [2, 3, 1], [4, 60, 6])):
        length = length + np.array(grow)
        v.commit(gpu(length, I32), syn.latents(sum(grow), seed=step).to(DEV))
        parents = random_parents(rng, 3, 6)
        depths = np.array([[len(p) - 1 for p in ref.paths(row.tolist())] for row in parents])
        q = (torch.randn(3, 6, 16, 512, generator=torch.Generator().manual_seed(step)) * 0.5).bfloat16()
        got = v.draft(syn.latents(18, seed=50 + step).to(DEV), gpu(depths), q.to(DEV),
                      gpu(parents, I32))
        want = ref.tree(q, v.pool.layer().cpu().numpy(), v.table.cpu().numpy(), length, parents, 40,
                        sink=v.sink.cpu().numpy())
        check(got, want)


def test_graphs_replay_with_new_inputs():
    """Two captured verification steps run in turn, with other lengths, trees and rows each
    time, beside eager ones; the second graph's workspace is its own."""
    banner("graphs")
    def begin(seed):
        v = Verify(nodes=6)
        v.commit(gpu([130, 7, 60], I32), syn.latents(197, seed=seed).to(DEV))
        return v

    def feed(seed, base):
        rng = np.random.default_rng(seed)
        parents = random_parents(rng, 3, 6)
        depths = np.array([[len(p) - 1 for p in ref.paths(row.tolist())] for row in parents])
        return (syn.latents(18, seed=seed).to(DEV), gpu(depths),
                (torch.randn(3, 6, 16, 512, generator=torch.Generator().manual_seed(seed)) * 0.5)
                .bfloat16().to(DEV), gpu(parents, I32))

    pairs = []
    for g in range(2):
        eager, v = begin(g), begin(g)
        static = list(feed(99, g))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            v.draft(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = v.draft(*static)
        pairs.append((eager, v, graph, static, outs))
    for turn in range(6):
        for eager, v, graph, static, outs in pairs:
            fresh = feed(turn, 0)
            for s, f in zip(static, fresh):
                s.copy_(f)
            want = eager.draft(*fresh)
            graph.replay()
            if turn % 2:
                torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b), turn


def test_graphs_deal_by_the_lengths_of_the_replay():
    """Two captured calls, each with a workspace of its own that holds anything before a
    replay: lengths from none to the tables' capacity, so that a request is now finished by
    one workgroup, now split over many."""
    banner("graphs with other lengths")
    batch, nodes, heads, columns = 3, 4, 16, 20
    splits, need = remnant.get_tree_decode_metadata(batch, nodes, heads, columns, history_blocks=4)
    assert splits > 1 and need > 0
    rng = np.random.default_rng(7)
    full = columns * 64 - nodes
    turns = [([0, 0, 0], [0, 0, 0]), ([full, 1, 64], [0, 256, 3]), ([5, full, 700], [256] * 3),
             ([full] * 3, [256, 0, 9]), ([64, 0, 3], [0] * 3), ([full + nodes, 900, 17], [1, 2, 3]),
             ([0, 130, full], [0] * 3)]

    def feed(seed, turn):
        g = torch.Generator().manual_seed(100 * seed + turn)
        lengths, past = turns[turn]
        return [(torch.randn(batch, nodes, heads, 512, generator=g) * 0.5).bfloat16().to(DEV),
                gpu(lengths, I32), gpu(random_parents(rng, batch, nodes), I32), gpu(past, I32)]

    sides = []
    for seed in range(2):
        pool, old = ref.random_native(batch * columns, seed), ref.random_native(12, seed + 9)
        table = rng.permutation(batch * columns).reshape(batch, columns)
        past_table = rng.permutation(12).reshape(batch, 4)
        sink = rng.standard_normal(heads).astype(np.float32)
        on = [gpu(pool), gpu(table, I32), gpu(old), gpu(past_table, I32), gpu(sink)]

        def call(q, lengths, parents, past, on=on, workspace=None):
            return remnant.tree_decode_fwd(q, on[0], on[1], lengths, parents, history_pool=on[2],
                                           history_table=on[3], history_lengths=past, sink=on[4],
                                           workspace=workspace)

        static, ws = feed(seed, 1), torch.empty(need, dtype=torch.uint8, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(*static, workspace=ws)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call(*static, workspace=ws)
        sides.append((seed, (pool, table, old, past_table, sink), call, static, ws, graph, outs))
    for turn in range(len(turns)):
        for seed, (pool, table, old, past_table, sink), call, static, ws, graph, outs in sides:
            fresh = feed(seed, turn)
            for s, f in zip(static, fresh):
                s.copy_(f)
            ws.fill_(0xFF)
            graph.replay()
            if turn % 2:
                torch.cuda.synchronize()
            eager = call(*fresh)
            for a, b in zip(outs, eager):
                assert torch.equal(a, b), turn
            lengths, past = turns[turn]
            check(outs, ref.tree(fresh[0].cpu(), pool, table, lengths, fresh[2].cpu().numpy(), None,
                                 old, past_table, past, sink=sink), (turn, seed))


def test_two_streams_at_once():
    banner("two streams")
    cases = [Tree(8, 16, batch=2, context=3000, seed=30), Tree(16, 8, context=300, past=500, seed=31)]
    wants = [[t.clone() for t in c.run()] for c in cases]
    ins = [c.args() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(remnant.tree_decode_fwd(*ins[i][0], **ins[i][1]))
    torch.cuda.synchronize()
    for want, outs in zip(wants, got):
        for o in outs:
            for a, b in zip(o, want):
                assert torch.equal(a, b)


def test_tensors_of_two_devices_are_refused():
    banner("two devices")
    case = Tree(2, 16, context=20)
    with pytest.raises(ValueError, match="same GPU"):
        case.run(sink=torch.zeros(16))
    a, kw = case.args()
    with pytest.raises(ValueError, match="same GPU"):
        remnant.tree_decode_fwd(*a[:4], torch.from_numpy(case.parents).to(I32), **kw)
