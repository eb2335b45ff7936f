"""GPU tests of the frequency rows of the full-row stores: the row of a position is
position * ratio, for token positions (ratio 1, the window pool) as for record numbers."""

import numpy as np
import pytest
import torch

import mx4_reference as ref
import oracle
import remnant
from remnant import synthetic as syn
from test_gpu_mx4 import check, gpu

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = torch.int32


def inputs(rows, dtype, ratio):
    """Rows at positions on both sides of the table's two ends; slots left out among them."""
    rng = np.random.default_rng(rows * 8 + ratio)
    x = syn.latents(rows, seed=rows).to(dtype)
    freqs = syn.rope_freqs(301)
    positions = rng.integers(-1, 300 // ratio + 3, rows)
    positions[: min(rows, 2)] = (300 // ratio, 2 ** 31 - 1)[: min(rows, 2)]
    pages = rows // 64 + 1
    slots = rng.permutation(pages * 64)[:rows]
    slots[3::19] = -1
    ok = (slots >= 0) & (positions >= 0) & (positions * ratio < 301)
    return x, freqs, positions, slots, pages, ok


# rows: of each way the stores share them out (one a wave, four a wave, streamed)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("ratio", [1, 3, 2 ** 31 - 1])
@pytest.mark.parametrize("rows", [1, 700, 4100, 65600])
def test_4bit_store_rotates_by_position_times_ratio(rows, ratio, dtype):
    print(f"[gpu-ratio] 4-bit store {rows} / {ratio} {dtype}", flush=True)
    x, freqs, positions, slots, pages, ok = inputs(rows, dtype, ratio)
    weight = torch.linspace(0.5, 1.5, 512)
    pool = remnant.LatentPool(pages, fmt="mx4", device=DEV)
    pool.buffer.fill_(0x5A)
    remnant.mx4_store_rows(x.to(DEV), weight.to(DEV), 1e-6, gpu(slots, I32), gpu(positions, I32),
                           freqs.to(DEV), pool, ratio=ratio)
    # the definition takes row 4 p of its table: give it one row in four
    table = freqs[np.where(ok, positions * ratio, 0)].repeat_interleave(4, 0)
    want = np.full((pages * 64, 272), 0x5A, np.uint8)
    want[slots[ok]] = ref.store_rows(x, weight.numpy(), 1e-6, np.arange(rows), table)[ok]
    assert np.array_equal(pool.layer().cpu().numpy().reshape(-1, 272), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("ratio", [1, 3, 2 ** 31 - 1])
@pytest.mark.parametrize("rows", [1, 20000, 140000])
def test_native_store_rotates_by_position_times_ratio(rows, ratio, dtype):
    print(f"[gpu-ratio] Native store {rows} / {ratio} {dtype}", flush=True)
    x, freqs, positions, slots, pages, ok = inputs(rows, dtype, ratio)
    pool = remnant.LatentPool(pages, fmt="native", device=DEV)
    pool.buffer.fill_(0x5A)
    remnant.native_store_rows(x.to(DEV), torch.ones(512, device=DEV), 1e-6, gpu(slots, I32),
                              gpu(positions, I32), freqs.to(DEV), pool, ratio=ratio)
    got = pool.layer().cpu().numpy()
    untouched = np.ones(pages * 64, bool)
    untouched[slots[ok]] = False
    data = got[:, :64 * 576].reshape(-1, 576)
    scales = got[:, 64 * 576:].reshape(-1, 8)
    assert (data[untouched] == 0x5A).all() and (scales[untouched] == 0x5A).all()
    f = torch.view_as_real(freqs).numpy()
    for i in np.flatnonzero(ok)[:: max(rows // 1000, 1)]:
        d, s = oracle.native_pack_row(x[i].float().numpy(), np.ones(512, np.float32), 1e-6,
                                      f[positions[i] * ratio])
        assert np.array_equal(data[slots[i]], d) and np.array_equal(scales[slots[i]], s), i


def test_window_rows_of_a_step_are_rotated_by_their_tokens():
    """append_slots at ratios 4 and 1, both stores with its positions, window_slots and the
    decode: against attention over rows rotated by the tokens' own frequency rows."""
    print("[gpu-ratio] step", flush=True)
    old, new = np.array([0, 30, 101]), np.array([5, 95, 230])
    freqs, ones = syn.rope_freqs(256), torch.ones(512)
    tables, pools, raw, maps = [], [], [], []
    for fmt, ratio, pages in (("mx4", 4, 8), ("native", 1, 16)):
        table = torch.full((3, 4), -1, dtype=I32, device=DEV)
        free = torch.randperm(pages, generator=torch.Generator().manual_seed(ratio)).to(I32).to(DEV)
        pool = remnant.LatentPool(pages, fmt=fmt, device=DEV)
        rows = [syn.latents(int(n) // ratio, seed=10 * b + ratio) for b, n in enumerate(new)]
        store = remnant.mx4_store_rows if fmt == "mx4" else remnant.native_store_rows
        taken = 0
        for lo, hi in ((np.zeros(3, int), old), (old, new)):
            m = remnant.append_slots(table, gpu(lo, I32), gpu(hi, I32), free[taken:].contiguous(),
                                     ratio=ratio, rows=300)
            x = torch.cat([r[a // ratio:b // ratio] for r, a, b in zip(rows, lo, hi)])
            x = torch.cat([x, torch.ones(300 - len(x), 512, dtype=x.dtype)])
            store(x.to(DEV), ones.to(DEV), 1e-6, m.loc, m.positions, freqs.to(DEV), pool,
                  ratio=ratio)
            taken += int(m.pages_taken)
        tables.append(table), pools.append(pool), raw.append(rows), maps.append(m)
    slots, counts = remnant.window_slots(tables[1], gpu(new, I32), 1, 20, first=3)
    rng = np.random.default_rng(1)
    idx = np.stack([rng.integers(0, max(int(n) // 4, 1), (1, 40)) for n in new]).astype(np.int32)
    q = (torch.randn(3, 1, 16, 512, generator=torch.Generator().manual_seed(4)) * 0.5).bfloat16()
    got = remnant.mx4_sparse_decode_fwd(q.to(DEV), pools[0], tables[0], gpu(idx),
                                        seqlens=maps[0].seqlens, swa_pool=pools[1],
                                        swa_indices=slots, swa_lengths=counts)
    # the same from the raw rows: request b's records from 256 b on, in pools built here
    rec = np.zeros((3 * 256, 272), np.uint8)
    win = np.zeros((3 * 4, 37376), np.uint8)
    widx = np.full((3, 1, 23), -1, np.int32)
    f = torch.view_as_real(freqs).numpy()
    for b, n in enumerate(new):
        k = int(n) // 4
        rec[256 * b:256 * b + k] = ref.store_rows(raw[0][b], ones.numpy(), 1e-6, np.arange(k), freqs)
        for t in range(int(n)):
            page, row = divmod(256 * b + t, 64)
            d, s = oracle.native_pack_row(raw[1][b][t].float().numpy(), ones.numpy(), 1e-6, f[t])
            win[page, row * 576:row * 576 + 576] = d
            win[page, 64 * 576 + row * 8:64 * 576 + row * 8 + 8] = s
        t = np.arange(n)
        seen = t[(t < 3) | (t > n - 1 - 20)]
        assert counts[b] == len(seen)
        widx[b, 0, :len(seen)] = 256 * b + seen
    check(got, ref.decode(q, rec.reshape(12, -1), np.arange(12).reshape(3, 4), idx, new // 4,
                          swa_pool=win, swa_indices=widx))


def test_captured_steps_carry_on():
    """One captured serving step -- both appends behind the pages taken, both stores with
    their rotation, window lists, decode -- replayed as one step after another, beside the
    same steps run eagerly: all outputs, tables and pools equal after every replay."""
    print("[gpu-ratio] captured steps", flush=True)
    freqs, ones = syn.rope_freqs(400).to(DEV), torch.ones(512, device=DEV)
    sink = torch.linspace(-1, 1, 16, device=DEV)
    grow = gpu([1, 4, 7], I32)

    class State:
        def __init__(self):
            self.pools = [remnant.LatentPool(9, fmt="mx4", device=DEV),
                          remnant.LatentPool(9, fmt="native", device=DEV)]
            self.tables = [torch.full((3, 3), -1, dtype=I32, device=DEV) for _ in range(2)]
            self.free = [gpu(np.random.default_rng(i).permutation(9), I32) for i in range(2)]
            self.taken = [torch.zeros(1, dtype=I32, device=DEV) for _ in range(2)]
            self.old, self.new = (torch.zeros(3, dtype=I32, device=DEV) for _ in range(2))
            self.x = [torch.zeros(n, 512, dtype=torch.bfloat16, device=DEV) for n in (6, 12)]
            self.q = torch.zeros(3, 1, 16, 512, dtype=torch.bfloat16, device=DEV)
            self.idx = torch.zeros(3, 1, 40, dtype=I32, device=DEV)

        def feed(self, seed):
            g = torch.Generator().manual_seed(seed)
            for t in (*self.x, self.q):
                t.copy_(torch.randn(t.shape, generator=g))
            self.idx.copy_(torch.randint(-1, 40, self.idx.shape, generator=g))

        def step(self):
            torch.add(self.old, grow, out=self.new)
            maps = []
            for i, (ratio, store) in enumerate(((4, remnant.mx4_store_rows),
                                                (1, remnant.native_store_rows))):
                m = remnant.append_slots(self.tables[i], self.old, self.new, self.free[i],
                                         ratio=ratio, rows=self.x[i].shape[0], taken=self.taken[i])
                store(self.x[i], ones, 1e-6, m.loc, m.positions, freqs, self.pools[i], ratio=ratio)
                self.taken[i].copy_(m.pages_taken)
                maps.append(m)
            slots, counts = remnant.window_slots(self.tables[1], self.new, 1, 16, first=2)
            out, lse = remnant.mx4_sparse_decode_fwd(
                self.q, self.pools[0], self.tables[0], self.idx, seqlens=maps[0].seqlens, sink=sink,
                swa_pool=self.pools[1], swa_indices=slots, swa_lengths=counts)
            self.old.copy_(self.new)
            return [*maps[0], *maps[1], slots, counts, out, lse]

        def held(self):
            return [*self.tables, *self.taken, self.old] + [p.buffer for p in self.pools]

    side, warm = torch.cuda.Stream(), State()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.step()
    torch.cuda.current_stream().wait_stream(side)
    graphed, eager, graph = State(), State(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = graphed.step()
    for seed in range(25):
        graphed.feed(seed)
        eager.feed(seed)
        graph.replay()
        if seed % 2:
            torch.cuda.synchronize()
        want = eager.step()
        for i, (a, b) in enumerate(zip(got + graphed.held(), want + eager.held())):
            assert torch.equal(a, b), (seed, i)
    assert graphed.old.tolist() == [25, 100, 175]
    assert [t.tolist() for t in graphed.taken] == [[3], [6]]
    for t in graphed.tables:
        pages = [p for p in t.flatten().tolist() if p >= 0]
        assert len(set(pages)) == len(pages)
