"""GPU tests of the slot maps: equal to plain loops over the requests."""

import numpy as np
import pytest
import torch

import mx4_reference as ref
import remnant

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = torch.int32


def gpu(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=I32).to(DEV)


def run_append(table, old, new, free, ratio, rows, pad=0):
    """The call on a table embedded in a wider one; the rest must stay as it was."""
    wide = torch.full((table.shape[0], table.shape[1] + pad), 77, dtype=I32, device=DEV)
    view = wide[:, :table.shape[1]]
    view.copy_(gpu(table))
    got = remnant.append_slots(view, gpu(old), gpu(new), gpu(free), ratio=ratio, rows=rows)
    want = ref.append(table, old, new, free, ratio, rows)
    for name, a, b in zip(got._fields, got, want):
        assert np.array_equal(a.cpu().numpy(), b), name
    assert np.array_equal(view.cpu().numpy(), want[5])
    assert (wide[:, table.shape[1]:] == 77).all()


@pytest.mark.parametrize("batch", [0, 1, 2, 63, 64, 255, 256, 257, 1000])
@pytest.mark.parametrize("ratio", [1, 4])
def test_append_equals_loops(batch, ratio):
    print(f"[gpu-slots] append {batch} / {ratio}", flush=True)
    rng = np.random.default_rng(batch * 10 + ratio)
    for grow in (1, 3, 130):
        old = rng.integers(0, 700, batch)
        new = old + rng.integers(0, grow + 1, batch)
        old[rng.random(batch) < 0.1] = 0
        new[rng.random(batch) < 0.05] -= 5  # shorter than before: nothing added
        held = -(-(old // ratio) // 64)
        after = -(-(np.maximum(new, old) // ratio) // 64)
        width = int(after.max(initial=1)) + 2
        pages = rng.permutation(int(held.sum()) + int((after - held).sum()) + 5)
        table = np.full((batch, width), -1)
        at = 0
        for b in range(batch):
            table[b, :held[b]] = pages[at:at + held[b]]
            at += held[b]
        free, total = pages[at:], int((np.maximum(new, old) // ratio - old // ratio).sum())
        for rows in (total, total + 70, max(total - 3, 0)):
            run_append(table, old, new, free, ratio, rows)
        run_append(table, old, new, free[:len(free) // 3], ratio, total, pad=3)  # short of pages
        run_append(table[:, :max(width - 3, 1)], old, new, free, ratio, total, pad=1)  # columns


def test_append_largest_batch_and_long_prompts():
    print("[gpu-slots] append 8192, long prompts", flush=True)
    rng = np.random.default_rng(5)
    old = rng.integers(0, 300, 8192)
    new = old + rng.integers(0, 2, 8192)
    table = np.arange(8192 * 6).reshape(8192, 6)
    run_append(table, old, new, np.arange(50000, 58000), 1, 8192)
    old, new = np.array([0, 63, 64, 100000]), np.array([131072, 64, 65, 300001])
    table = np.full((4, 4800), -1)
    table[1, 0], table[2, 0] = 9000, 9001
    table[3, :1563] = np.arange(20000, 21563)
    run_append(table, old, new, rng.permutation(8000), 1, 400000)


def test_append_extreme_values():
    """Lengths at the ends of int32, free and mapped pages no slot can name."""
    print("[gpu-slots] append extremes", flush=True)
    big = 2 ** 31 - 1
    old, new = np.array([-5, big - 1, -big - 1, big]), np.array([3, big, -1, 0])
    table = np.array([[5, 6], [7, 8], [1, 2], [3, 4]])
    run_append(table, old, new, np.array([1 << 25, -4, 9]), 1, 10)
    run_append(table, old, new, np.array([(1 << 25) - 1, 9]), 1, 10)
    run_append(table, old, new, np.zeros(0, np.int64), 1, 10)
    run_append(np.zeros((4, 0), np.int64), old, new, np.array([4, 9]), 1, 10)
    # sums that pass int32 saturate; the first rows stay right
    n = 64
    got = remnant.append_slots(gpu(np.full((n, 3), -1)), gpu(np.zeros(n)), gpu(np.full(n, big)),
                               gpu(np.arange(4)), ratio=1, rows=300)
    starts = got.row_starts.cpu().numpy()
    assert starts[0] == 0 and (starts[1:] == big).all()
    assert got.pages_taken.item() == big  # 64 x 2^25 pages
    assert got.loc.tolist() == list(range(192)) + [-1] * 108
    assert got.positions.tolist() == list(range(300))


@pytest.mark.parametrize("ratio", [2, 3, 7, 641, 65537, 2 ** 30 - 1, 2 ** 30 + 1, 2 ** 31 - 1])
def test_append_divides_exactly(ratio):
    """old // ratio at the multiples of the ratio, beside them and at the ends of int32."""
    print(f"[gpu-slots] append ratio {ratio}", flush=True)
    rng = np.random.default_rng(ratio)
    big = 2 ** 31 - 1
    near = rng.integers(0, big // ratio + 1, 300) * ratio
    new = np.concatenate([near, near - 1, near + 1, [big, big - 1, 0, 1, -1], rng.integers(0, big, 300)])
    new = np.clip(new, -1, big)
    got = remnant.append_slots(gpu(np.zeros((len(new), 0))), gpu(new), gpu(new), gpu([]),
                               ratio=ratio, rows=3)
    assert np.array_equal(got.seqlens.cpu().numpy(), np.maximum(new, 0) // ratio)
    assert got.row_starts.max().item() == 0 and got.pages_taken.item() == 0
    assert got.loc.tolist() == [-1] * 3


def test_append_writes_caller_buffers():
    print("[gpu-slots] append out", flush=True)
    out = [torch.full((n,), 55, dtype=I32, device=DEV) for n in (20, 20, 3, 2, 1)]
    table = gpu([[3, -1], [-1, -1]])
    got = remnant.append_slots(table, gpu([60, 0]), gpu([70, 5]), gpu([8, 9, 10]), out=out)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(got, out))
    assert table.tolist() == [[3, 8], [9, -1]]
    assert got.loc.tolist() == [252, 253, 254, 255] + list(range(512, 518)) + list(range(576, 581)) \
        + [-1] * 5
    assert got.positions.tolist() == list(range(60, 70)) + list(range(5)) + [0] * 5
    assert got.row_starts.tolist() == [0, 10, 15] and got.seqlens.tolist() == [70, 5]
    assert got.pages_taken.tolist() == [2]


@pytest.mark.parametrize("q_len,window,first", [(1, 1, 0), (1, 128, 0), (2, 128, 4), (3, 7, 33),
                                                (1, 0, 5), (4, 500, 0), (2, 64, 64), (1, 0, 0),
                                                (1, 2000, 3)])
def test_window_equals_loops(q_len, window, first):
    print(f"[gpu-slots] window {q_len} {window} {first}", flush=True)
    rng = np.random.default_rng(window)
    lengths = np.concatenate([[0, 1, 2, 63, 64, 65, 127, 128, 129, 700],
                              rng.integers(0, 1500, 12)])
    table = rng.permutation(22 * 23).reshape(22, 23)
    table[3, 0] = -1
    table[9, 9] = 1 << 25
    for width in (23, 10):
        wide = torch.full((22, width + 2), -9, dtype=I32, device=DEV)
        wide[:, :width] = gpu(table[:, :width])
        slots, counts = remnant.window_slots(wide[:, :width], gpu(lengths), q_len, window,
                                             first=first)
        want, n = ref.window(table[:, :width], lengths, q_len, window, first)
        assert np.array_equal(slots.cpu().numpy(), want)
        assert np.array_equal(counts.cpu().numpy(), n)


@pytest.mark.parametrize("window,first,shift", [(32768, 0, 0), (32764, 4, 0), (32766, 5, 0),
                                                (32768, 0, 1), (39999, 1, 0)])
def test_window_long_lists(window, first, shift):
    """Lists long enough for the form of four entries a thread, rows that do not divide
    by it and a buffer that is not 16-byte aligned."""
    print(f"[gpu-slots] window long {window} {first} {shift}", flush=True)
    rng = np.random.default_rng(window + first)
    lengths = np.array([0, 1, 63, 20000, 32767, 32770, 39999, 40000, 33000])
    table = rng.permutation(9 * 626).reshape(9, 626)
    table[4, 100] = -1
    n = 9 * (first + window)
    flat = torch.full((n + shift + 8,), -7, dtype=I32, device=DEV)
    out = flat[shift:shift + n].view(9, 1, first + window), torch.empty(9, dtype=I32, device=DEV)
    remnant.window_slots(gpu(table), gpu(lengths), 1, window, first=first, out=out)
    want, count = ref.window(table, lengths, 1, window, first)
    assert np.array_equal(out[0].cpu().numpy(), want)
    assert np.array_equal(out[1].cpu().numpy(), count)
    assert (flat[:shift] == -7).all() and (flat[shift + n:] == -7).all()


def test_window_more_than_32_bits_of_entries():
    print("[gpu-slots] window 4.3e9 entries", flush=True)
    tokens, window = 33000, 131073
    table = torch.arange(tokens, dtype=I32, device=DEV)[:, None] + torch.arange(2, dtype=I32,
                                                                                device=DEV)
    table = table.contiguous()
    lengths = torch.arange(tokens, dtype=I32, device=DEV) % 140 + 1
    slots, counts = remnant.window_slots(table, lengths, 1, window)
    assert torch.equal(counts, lengths)
    some = [0, 1, 139, 20000, 32767, 32768, 32999]
    want, _ = ref.window(table[some].cpu().numpy(), lengths[some].cpu().numpy(), 1, window, 0)
    assert np.array_equal(slots[some].cpu().numpy(), want)


def test_window_many_tokens_and_extreme_lengths():
    print("[gpu-slots] window many", flush=True)
    lengths = torch.full((70000,), 3, dtype=I32, device=DEV)
    table = torch.arange(70000, dtype=I32, device=DEV)[:, None].contiguous()
    slots, counts = remnant.window_slots(table, lengths, 1, 2)
    assert torch.equal(slots[:, 0], table * 64 + torch.tensor([1, 2], device=DEV, dtype=I32))
    assert (counts == 2).all()
    big = 2 ** 31 - 1
    lengths = gpu([big, -big - 1, -1])
    table = gpu([[5], [6], [7]])
    slots, counts = remnant.window_slots(table, lengths, 2, 3, first=2)
    assert slots[0, 1].tolist() == [320, 321, -1, -1, -1]
    assert counts.tolist() == [5, 5, 0, 0, 0, 0] and (slots[1:] == -1).all()


def test_window_lists_feed_the_readers():
    """A window as long as the history lists a request's slots in order, for the 4-bit
    and the Packed reader."""
    print("[gpu-slots] window lists", flush=True)
    table = gpu([[2, 0, 1], [3, -1, -1]])
    slots, counts = remnant.window_slots(table, gpu([150, 20]), 1, 192)
    pool = remnant.LatentPool(4, fmt="mx4", device=DEV)
    x = torch.randn(170, 512, generator=torch.Generator().manual_seed(1))
    loc = torch.cat([slots[0, 0, :150], slots[1, 0, :20]]).contiguous()
    remnant.mx4_store_rows(x.to(DEV), torch.ones(512, device=DEV), 1e-6, loc, None, None, pool)
    out = remnant.mx4_gather_bf16(pool, slots[:, 0], counts).view(2, 192, 512)
    want = ref.decode_rows(ref.store_rows(x, np.ones(512), 1e-6))
    assert np.array_equal(out[0, :150].double().cpu().numpy(), want[:150])
    assert np.array_equal(out[1, :20].double().cpu().numpy(), want[150:])
    assert (out[0, 150:] == 0).all() and (out[1, 20:] == 0).all()
    packed = remnant.LatentPool(4, device=DEV)
    remnant.pack_rows_fused(x.to(DEV), torch.ones(512, device=DEV), 1e-6, loc, packed)
    rows = torch.empty(384, 512, dtype=torch.bfloat16, device=DEV)
    remnant.unpack_gather_bf16(packed, slots[:, 0], None, counts, None, rows)
    assert torch.equal(rows.view(2, 192, 512)[0, :150], remnant.unpack_rows(packed, loc[:150]))


@pytest.mark.parametrize("batch", [0, 5, 300])
@pytest.mark.parametrize("gone", [-7, 0, 1, 40, 100000, 2 ** 31 - 1])
def test_append_takes_pages_behind_those_taken(gone, batch):
    """The list starts behind `taken`, the count goes on from it (and saturates)."""
    print(f"[gpu-slots] append {batch} after {gone}", flush=True)
    rng = np.random.default_rng(batch)
    old = rng.integers(0, 300, batch)
    new = old + rng.integers(0, 200, batch)
    table = rng.integers(0, 1000, (batch, 9))
    free = rng.permutation(5000)
    for n_free in (5000, 60, 40, 0):
        dev, taken = gpu(table), gpu([gone])
        got = remnant.append_slots(dev, gpu(old), gpu(new), gpu(free[:n_free]), rows=500, taken=taken)
        want = ref.append(table, old, new, free[:n_free][max(gone, 0):], 1, 500)
        pages = min(int(want[4][0]) + max(gone, 0), 2 ** 31 - 1)
        assert got.pages_taken.tolist() == [pages] and taken.tolist() == [gone]
        for name, a, b in zip(got._fields[:4], got, want):
            assert np.array_equal(a.cpu().numpy(), b), name
        assert np.array_equal(dev.cpu().numpy(), want[5])


def test_captured_steps_take_pages_of_their_own():
    """One captured step replayed again and again: lengths and the count of pages are
    carried on in the graph. Every replay against loops on the host, until the list is
    short; eager work of the same tensors' values between the replays."""
    print("[gpu-slots] captured steps", flush=True)
    rng = np.random.default_rng(3)
    table, free = np.full((6, 8), -1), rng.permutation(30)
    grow = gpu([1, 64, 0, 33, 3, 70])
    dev = dict(table=gpu(table), old=gpu(np.zeros(6)), new=gpu(np.zeros(6)), free=gpu(free),
               taken=gpu([0]))

    def step(d):
        torch.add(d["old"], grow, out=d["new"])
        m = remnant.append_slots(d["table"], d["old"], d["new"], d["free"], rows=200,
                                 taken=d["taken"])
        d["taken"].copy_(m.pages_taken)
        d["old"].copy_(d["new"])
        return m

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step({k: t.clone() for k, t in dev.items()})
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(dev)
    eager = {k: t.clone() for k, t in dev.items()}
    old, taken = np.zeros(6, np.int64), 0
    for i in range(13):
        new = old + grow.cpu().numpy()
        want = ref.append(table, old, new, free[taken:], 1, 200)
        taken, table, old = taken + int(want[4][0]), want[5], new
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        same = step(eager)
        for name, a, b, c in zip(got._fields[:4], got, want, same):
            assert np.array_equal(a.cpu().numpy(), b) and torch.equal(a, c), (i, name)
        assert got.pages_taken.tolist() == [taken] == dev["taken"].tolist()
        assert np.array_equal(dev["table"].cpu().numpy(), table)
        mapped = table[table >= 0]
        assert len(np.unique(mapped)) == len(mapped)
    assert taken > 30
