"""Cases of the 4-bit latent cache and of the slot maps that address it.

Five kinds of case, each one public operator of ``remnant``:

``append``  ``append_slots``: block tables extended and the slots of a step's new
            records, from the requests' lengths,
``window``  ``window_slots``: per query token the slots it may see (a sliding window
            and the first tokens of the request),
``store``   ``mx4_store_rows``: compressor rows normalised, rotated and written as
            4-bit records; the pass reads them back (``mx4_gather_bf16``), as the
            attention of a prefill chunk does, so that it returns the stored values,
``gather``  ``mx4_gather_bf16``: 4-bit records -> dense BF16 rows,
``decode``  ``mx4_sparse_decode_fwd``: attention over the 4-bit cache, with sink and,
            where ``window`` > 0, sliding-window rows of a Native (8-bit) pool.

A 4-bit record holds 512 coordinates in 272 bytes: 256 bytes of E2M1 codes (coordinate
2i in the low half of byte i) and 16 UE8M0 scale bytes, one for 32 coordinates. 64
records make a page; slot s is record s % 64 of page s / 64. A Native record is 448
E4M3 codes, 64 BF16 and 7 UE8M0 scales (one for 64 coordinates).
"""

import math
import os
import sys

import torch

own = False

DIM, NOPE, PAIRS, PAGE, REC = 512, 448, 32, 64, 272
NATIVE_DATA = 576
BANK = 4096  # distinct records a pool is filled with
SCALE = 1.0 / math.sqrt(DIM)
I32 = torch.int32
DEV = "cuda" if torch.cuda.is_available() else "cpu"


def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "flash-optimizations_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import remnant
    return remnant


# ---- cases ----

def _append(name, batch, held, new, *, ratio, rows, spare=1.0):
    """held / new: largest tokens of a request before the step and added by it
    (log-uniform from a 32nd of them); spare: free pages over those needed."""
    return dict(name=name, kind="append", batch=batch, held=held, new=new, ratio=ratio, rows=rows,
                spare=spare)


def _window(name, batch, q_len, window, first, length):
    return dict(name=name, kind="window", batch=batch, q_len=q_len, window=window, first=first,
                length=length)


def _store(name, rows, dtype, *, valid=1.0, rope=True):
    return dict(name=name, kind="store", rows=rows, dtype=dtype, valid=valid, rope=rope)


def _gather(name, queries, k, *, valid=1.0):
    return dict(name=name, kind="gather", queries=queries, k=k, valid=valid)


def _decode(name, batch, heads, topk, *, context, shortest=None, valid=None, q_len=1, window=0):
    """context / shortest: largest and smallest records of a request (log-uniform
    between); valid: entries of a list in use where the context has as many."""
    return dict(name=name, kind="decode", batch=batch, heads=heads, topk=topk, context=context,
                shortest=shortest or context, valid=valid or topk, q_len=q_len, window=window)


def listed():
    return [
        # one decode step of a serving batch, contexts up to 128k tokens: a request in four
        # completes a record of four tokens, one in 256 takes a page
        _append("slots-step-b256", 256, 131072, 1, ratio=4, rows=256),
        # a prefill batch's tokens, one slot each (the window pool's), prompts of up to 128k
        _append("slots-prefill-b16", 16, 4096, 131072, ratio=1, rows=1 << 20),
        # the window lists of a decode step with one draft token, four first tokens kept
        _window("window-step-b256x2", 256, 2, 128, 4, 131072),
        # whole histories as slot lists, what a prefill chunk reads
        _window("window-history-b8", 8, 1, 131072, 0, 131072),
        # decode phase: the records that 24 sequences complete in one step
        _store("store-step-r24", 24, "float32"),
        # bulk conversion of a cache: BF16 latents into randomly placed slots
        _store("store-bulk-1m", 1 << 20, "bfloat16"),
        # a prefill chunk's selections as dense rows
        _gather("gather-q16-k512", 16, 512, valid=0.8),
        # the history of a 143,360-token prompt (one record for 4 tokens)
        _gather("gather-history-35840", 1, 35840),
        # a single long conversation: the smallest decode step, latency
        _decode("decode-b1", 1, 16, 2048, context=8192),
        # an ordinary serving batch, contexts of 4k to 128k tokens
        _decode("decode-b64", 64, 16, 2048, context=32768, shortest=1024),
        # all 64 heads on one GPU, ragged short lists and window rows
        _decode("decode-h64-b16-k317", 16, 64, 512, context=4096, valid=317, window=64),
        # the largest: a full batch with draft tokens at 128k tokens
        _decode("decode-b128x2", 128, 16, 2048, context=32768, q_len=2),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "window", "store", "gather", "decode", "decode"))
    if kind == "append":
        batch = _log_uniform(rng, 1, 4096)
        new = _log_uniform(rng, 1, max(1, min(131072, (1 << 20) // batch)))
        c = _append("", batch, _log_uniform(rng, 64, 131072 if batch <= 512 else 8192), new,
                    ratio=rng.choice((1, 4)), rows=max(1, batch * new - rng.randrange(3)),
                    spare=rng.choice((1.0, 1.5, 0.6)))
    elif kind == "window":
        batch, q_len = _log_uniform(rng, 1, 1024), rng.choice((1, 1, 2, 4))
        most = max(1, (1 << 20) // (batch * q_len))
        window = _log_uniform(rng, 1, min(131072, most))
        c = _window("", batch, q_len, window, rng.choice((0, 0, 1, 4, 33)),
                    _log_uniform(rng, 1, 131072 if batch <= 512 else 16384))
    elif kind == "store":
        dtype = rng.choice(("float32", "bfloat16"))
        rows = _log_uniform(rng, 1, (1 << 20) if dtype == "bfloat16" else (1 << 19))
        c = _store("", rows, dtype, valid=rng.choice((1.0, 0.75)), rope=rng.random() < 0.75)
    elif kind == "gather":
        rows, queries = _log_uniform(rng, 1, 1 << 20), rng.choice((1, 1, 3, 16))
        c = _gather("", queries, max(1, rows // queries), valid=rng.choice((1.0, 0.8)))
    else:
        batch, q_len = _log_uniform(rng, 1, 128), rng.choice((1, 1, 2))
        heads = rng.choice((16, 16, 16, 1, 8, 24, 32, 64, 128))
        while batch * q_len * heads > 4096:
            batch = (batch + 1) // 2
        topk = _log_uniform(rng, 1, 2048)
        context = _log_uniform(rng, 64, 32768)
        c = _decode("", batch, heads, topk, context=context,
                    shortest=max(1, context // rng.choice((1, 4, 64))),
                    valid=rng.choice((topk, max(1, (topk * 5) // 8))), q_len=q_len,
                    window=rng.choice((0, 0, 17, 64, 128)))
    del c["name"]
    return c


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 6007 + 29)


def _lengths(lo, hi, n, g):
    """n whole numbers, log-uniform on [lo, hi]."""
    a, b = math.log(lo), math.log(hi)
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    return torch.exp(a + u * (b - a)).round().to(torch.int64)


def _latents(n, g, dtype):
    lo, hi = math.log(0.1), math.log(10.0)
    sigma = torch.exp(torch.rand(DIM, device=DEV, generator=g) * (hi - lo) + lo)
    return (torch.randn(n, DIM, device=DEV, generator=g) * sigma).to(dtype)


def _rope_table(rows):
    """complex64 [rows, 32]: polar(1, position * 10000^(-j / 32)), angles in 64 bits."""
    theta = 10000.0 ** (-torch.arange(PAIRS, dtype=torch.float64, device=DEV) / PAIRS)
    angle = torch.outer(torch.arange(rows, dtype=torch.float64, device=DEV), theta)
    return torch.complex(angle.cos().float(), angle.sin().float())


def _blocks(records):
    return (records + PAGE - 1) // PAGE


def _random_pages(blocks, g):
    """A block table of random distinct pages, -1 behind each request's."""
    width, pages = max(1, int(blocks.max())), max(1, int(blocks.sum()))
    order = torch.randperm(pages, device=DEV, generator=g).to(I32)
    at = torch.arange(width, device=DEV) + (torch.cumsum(blocks, 0) - blocks)[:, None]
    table = order[at.clamp_max(pages - 1)]
    table[torch.arange(width, device=DEV) >= blocks[:, None]] = -1
    return table.contiguous(), pages


def _append_inputs(c, seed):
    g = _generator(seed)
    old = _lengths(max(1, c["held"] // 32), c["held"], c["batch"], g)
    # (a request in 16 is new, and an eighth of them have nothing this step)
    old[torch.rand(c["batch"], device=DEV, generator=g) < 1 / 16] = 0
    new = _lengths(max(1, c["new"] // 32), c["new"], c["batch"], g)
    new[torch.rand(c["batch"], device=DEV, generator=g) < 1 / 8] = 0
    held, after = _blocks(old // c["ratio"]), _blocks((old + new) // c["ratio"])
    table, pages = _random_pages(held, g)
    width = max(1, _blocks((c["held"] + c["new"]) // c["ratio"]))
    table = torch.nn.functional.pad(table, (0, max(0, width - table.shape[1])), value=-1)
    need = int((after - held).sum())
    count = max(1, int(need * c["spare"]))
    free = (torch.randperm(count, device=DEV, generator=g) + pages).to(I32)
    out = [torch.empty(n, dtype=I32, device=DEV)
           for n in (c["rows"], c["rows"], c["batch"] + 1, c["batch"], 1)]
    return dict(table=table.contiguous(), old=old.to(I32), new=(old + new).to(I32), free=free,
                out=out)


def _window_inputs(c, seed):
    g = _generator(seed)
    length = _lengths(max(1, c["length"] // 32), c["length"], c["batch"], g)
    table, _ = _random_pages(_blocks(length), g)
    tokens = c["batch"] * c["q_len"]
    out = [torch.empty(c["batch"], c["q_len"], c["first"] + c["window"], dtype=I32, device=DEV),
           torch.empty(tokens, dtype=I32, device=DEV)]
    return dict(table=table, length=length.to(I32), out=out)


def _store_inputs(c, seed):
    g = _generator(seed)
    rows = c["rows"]
    pages = _blocks(max(rows, 1024))
    loc = torch.randperm(pages * PAGE, device=DEV, generator=g)[:rows].to(I32)
    loc[int(rows * c["valid"]):] = -1  # rows without a record this step
    return dict(x=_latents(rows, g, getattr(torch, c["dtype"])), loc=loc,
                weight=torch.rand(DIM, device=DEV, generator=g) + 0.5,
                positions=torch.randint(0, 32768, (rows,), device=DEV, generator=g, dtype=I32),
                freqs=_rope_table(4 * 32768) if c["rope"] else None,
                pool=torch.zeros(pages, PAGE * REC, dtype=torch.uint8, device=DEV),
                out=torch.empty(rows, DIM, dtype=torch.bfloat16, device=DEV))


def _mx4_pool(pages, g):
    """Random latents, normalised and coded, in random order."""
    x = _latents(BANK, g, torch.float32)
    bank = _encode((x * torch.rsqrt(x.square().mean(-1, keepdim=True))).to(torch.bfloat16).float())
    ids = torch.randint(BANK, (pages * PAGE,), device=DEV, generator=g)
    return bank[ids].reshape(pages, PAGE * REC)


def _native_pool(pages, g):
    x = _latents(pages * PAGE, g, torch.float32)
    n = (x * torch.rsqrt(x.square().mean(-1, keepdim=True))).to(torch.bfloat16)
    groups = n[:, :NOPE].float().reshape(-1, 7, 64)
    e = torch.ceil(torch.log2(groups.abs().amax(-1).clamp_min(1e-4) / 448.0))
    codes = (groups * torch.exp2(-e)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    data = torch.cat([codes.reshape(-1, NOPE), n[:, NOPE:].contiguous().view(torch.uint8)], 1)
    scales = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, 1))
    return torch.cat([data.reshape(pages, -1), scales.reshape(pages, -1)], 1).contiguous()


def _gather_inputs(c, seed):
    g = _generator(seed)
    rows = c["queries"] * c["k"]
    pages = _blocks(rows)
    slots = torch.randperm(pages * PAGE, device=DEV, generator=g)[:rows].to(I32)
    slots[torch.rand(rows, device=DEV, generator=g) < 0.02] = -1
    lengths = torch.full((c["queries"],), int(c["k"] * c["valid"]), dtype=I32, device=DEV)
    return dict(pool=_mx4_pool(pages, g), slots=slots.reshape(c["queries"], c["k"]),
                lengths=lengths, out=torch.empty(rows, DIM, dtype=torch.bfloat16, device=DEV))


def _decode_inputs(c, seed):
    g = _generator(seed)
    batch, q_len, heads, topk = c["batch"], c["q_len"], c["heads"], c["topk"]
    contexts = _lengths(c["shortest"], c["context"], batch, g)
    table, pages = _random_pages(_blocks(contexts), g)
    # top-k lists: the records of the highest scores, in score order
    score = torch.rand(batch, q_len, max(c["context"], topk), device=DEV, generator=g)
    at = torch.arange(score.shape[-1], device=DEV)
    score.masked_fill_((at >= contexts[:, None])[:, None], -1.0)
    top = score.topk(topk, dim=-1).indices
    count = contexts.clamp_max(c["valid"])
    live = torch.arange(topk, device=DEV) < count[:, None, None]
    q = torch.randn(batch, q_len, heads, DIM, device=DEV, generator=g) * 2.0
    s = dict(table=table, seqlens=contexts.to(I32), pool=_mx4_pool(pages, g),
             indices=torch.where(live, top, -1).to(I32).contiguous(),
             lengths=count.repeat_interleave(q_len).to(I32), q=q.to(torch.bfloat16),
             sink=torch.randn(heads, device=DEV, generator=g), swa_pool=None, swa_indices=None,
             out=torch.empty(batch, q_len, heads, DIM, dtype=torch.bfloat16, device=DEV),
             lse=torch.empty(batch, q_len, heads, device=DEV), workspace=None)
    if c["window"]:
        rows = batch * c["window"]
        s["swa_pool"] = _native_pool(_blocks(rows), g)
        w = torch.randperm(rows, device=DEV, generator=g).reshape(batch, 1, -1)
        s["swa_indices"] = w.expand(-1, q_len, -1).to(I32).contiguous()
    return s


INPUTS = {"append": _append_inputs, "window": _window_inputs, "store": _store_inputs,
          "gather": _gather_inputs, "decode": _decode_inputs}


def prepare(case, seed):
    return dict(INPUTS[case["kind"]](case, seed), case=case)


# ---- plain forms ----

def _slot(table, request, record):
    """Pool slots of (request, record), int64; -1 where the table maps no page."""
    block = record // PAGE
    page = table[request, block.clamp(0, table.shape[1] - 1)].long()
    ok = (block >= 0) & (block < table.shape[1]) & (page >= 0) & (page < 1 << 25)
    return torch.where(ok, page * PAGE + record % PAGE, -1)


def _append_plain(s):
    c, table, free = s["case"], s["table"], s["free"]
    o = s["old"].long().clamp_min(0) // c["ratio"]
    n = torch.maximum(s["new"].long().clamp_min(0) // c["ratio"], o)
    held, after = _blocks(o), _blocks(n)
    pages = torch.cumsum(after - held, 0)
    ends = torch.cumsum(n - o, 0)
    col = torch.arange(table.shape[1], device=DEV)
    take = (pages - (after - held) - held)[:, None] + col
    got = torch.where(take < free.numel(), free[take.clamp(0, free.numel() - 1)], -1)
    fresh = (col >= held[:, None]) & (col < after[:, None])
    table.copy_(torch.where(fresh, got, table))
    i = torch.arange(c["rows"], device=DEV)
    request = torch.searchsorted(ends, i, right=True).clamp_max(c["batch"] - 1)
    record = o[request] + i - (ends - (n - o))[request]
    live = i < ends[-1]
    loc = torch.where(live, _slot(table, request, record), -1).to(I32)
    positions = torch.where(live, record, 0).to(I32)
    starts = torch.nn.functional.pad(ends, (1, 0)).to(I32)
    return [loc, positions, starts, n.to(I32), pages[-1:].to(I32), table]


def _window_plain(s):
    c, table = s["case"], s["table"]
    batch, q_len, window, first = c["batch"], c["q_len"], c["window"], c["first"]
    p = s["length"].long()[:, None] - q_len + torch.arange(q_len, device=DEV)  # own position
    f = (p + 1).clamp(0, first)
    start = torch.maximum(f, p + 1 - window)
    count = torch.where(p < 0, 0, f + p + 1 - start)
    at = torch.arange(first + window, device=DEV)
    token = torch.where(at < f[..., None], at, start[..., None] + at - f[..., None])
    request = torch.arange(batch, device=DEV)[:, None, None].expand_as(token)
    slots = torch.where(at < count[..., None], _slot(table, request, token), -1)
    return [slots.to(I32), count.reshape(-1).to(I32)]


def _encode(n):
    """[rows, 512] BF16 values in float32 -> record bytes [rows, 272]."""
    groups = n.reshape(-1, 16, 32)
    # smallest e with max(amax, 1e-4) <= 6 * 2^e, at most 32: amax = m * 2^k with m in [1/2, 1)
    m, k = torch.frexp(groups.abs().amax(-1).clamp_min(1e-4))
    e = (k - 3 + (m > 0.75)).clamp_max(32)
    v = torch.ldexp(groups.abs(), -e[..., None])
    # E2M1: steps of 1/2 below 2, 1 below 4, 2 to 6; ties to even
    code = torch.where(v < 2, torch.round(v * 2), torch.where(v < 4, torch.round(v) + 2,
                                                              torch.round(v / 2) + 4)).clamp_max(7)
    code = code.to(torch.uint8) + 8 * torch.signbit(groups).to(torch.uint8)
    code = code.reshape(-1, DIM)
    return torch.cat([code[:, 0::2] + 16 * code[:, 1::2], (e + 127).to(torch.uint8)], 1)


def _decode_rows(record):
    """Record bytes [..., 272] -> float32 values [..., 512]."""
    level = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV)
    level = torch.cat([level, -level])
    byte = record[..., :256].to(I32)
    value = level[torch.stack([byte & 15, byte >> 4], -1)]
    e = record[..., 256:].to(I32) - 127
    shape = record.shape[:-1]
    return torch.ldexp(value.reshape(*shape, 16, 32), e[..., None]).reshape(*shape, DIM)


def _store_plain(s):
    x, eps = s["x"].float(), 1e-6
    # sum of squares in the codec's order: 8 neighbours in turn, then pairs of neighbours
    sq = (x * x).reshape(-1, 64, 8)
    p = sq[..., 0]
    p = p + sq[..., 1]
    p = p + sq[..., 2]
    p = p + sq[..., 3]
    p = p + sq[..., 4]
    p = p + sq[..., 5]
    p = p + sq[..., 6]
    p = p + sq[..., 7]
    p = p[:, 0::2] + p[:, 1::2]
    p = p[:, 0::2] + p[:, 1::2]
    p = p[:, 0::2] + p[:, 1::2]
    p = p[:, 0::2] + p[:, 1::2]
    p = p[:, 0::2] + p[:, 1::2]
    p = p[:, 0::2] + p[:, 1::2]
    # root and reciprocal each rounded once to float32
    r = (1.0 / (p * (1.0 / DIM) + eps).double().sqrt().float().double()).float()
    n = ((x * r) * s["weight"]).to(torch.bfloat16).float()
    ok = (s["loc"] >= 0) & (s["loc"] < s["pool"].shape[0] * PAGE)
    if s["freqs"] is not None:
        row = s["positions"].long() * 4
        ok = ok & (row >= 0) & (row < s["freqs"].shape[0])
        f = s["freqs"][row.clamp(0, s["freqs"].shape[0] - 1)]
        re, im = n[:, NOPE::2], n[:, NOPE + 1::2]
        a, b = re * f.real, im * f.imag
        d, e = re * f.imag, im * f.real
        tail = torch.stack([a - b, d + e], -1).reshape(-1, 2 * PAIRS)
        n = torch.cat([n[:, :NOPE], tail.to(torch.bfloat16).float()], 1)
    records = s["pool"].view(-1, REC)
    records[s["loc"][ok].long()] = _encode(n[ok])
    return _rows_plain(records, s["loc"], ok)


def _rows_plain(records, slots, ok):
    rows = _decode_rows(records[slots.long().clamp(0, records.shape[0] - 1)])
    return torch.where(ok[:, None], rows, 0.0).to(torch.bfloat16)


def _gather_plain(s):
    records = s["pool"].view(-1, REC)
    k = torch.arange(s["slots"].shape[1], device=DEV)
    ok = (k < s["lengths"][:, None]) & (s["slots"] >= 0) & (s["slots"] < records.shape[0])
    return _rows_plain(records, s["slots"].reshape(-1), ok.reshape(-1))


def _native_rows(pool, slots):
    """Native records -> float32 values [..., 512]."""
    data = pool[:, :PAGE * NATIVE_DATA].reshape(-1, NATIVE_DATA)[slots]
    scales = pool[:, PAGE * NATIVE_DATA:].reshape(-1, 8)[slots][..., :7].to(I32) - 127
    shape = data.shape[:-1]
    codes = data[..., :NOPE].contiguous().view(torch.float8_e4m3fn).float()
    head = torch.ldexp(codes.reshape(*shape, 7, 64), scales[..., None]).reshape(*shape, NOPE)
    return torch.cat([head, data[..., NOPE:].contiguous().view(torch.bfloat16).float()], -1)


def _entries(s):
    """Slots and validity of each token's list entries, [tokens, topk]."""
    c = s["case"]
    record = s["indices"].reshape(-1, c["topk"]).long()
    request = torch.arange(c["batch"], device=DEV).repeat_interleave(c["q_len"])[:, None]
    slot = _slot(s["table"], request.expand_as(record), record.clamp_min(0))
    ok = (torch.arange(c["topk"], device=DEV) < s["lengths"][:, None]) & (record >= 0) & (slot >= 0)
    ok = ok & (record < s["seqlens"][request])
    return slot.clamp_min(0), ok


def _decode_plain(s):
    c = s["case"]
    slot, ok = _entries(s)
    rows = _decode_rows(s["pool"].view(-1, REC)[slot])
    if c["window"]:
        w = s["swa_indices"].reshape(-1, c["window"]).long()
        rows = torch.cat([rows, _native_rows(s["swa_pool"], w.clamp_min(0))], 1)
        ok = torch.cat([ok, w >= 0], 1)
    q = s["q"].reshape(-1, c["heads"], DIM).float()
    logits = torch.bmm(q, rows.transpose(1, 2).contiguous()) * SCALE
    logits = torch.where(ok[:, None], logits, -math.inf)
    sink = s["sink"][:, None]
    top = torch.maximum(logits.amax(-1, keepdim=True), sink)
    weight = torch.exp(logits - top)
    z = weight.sum(-1, keepdim=True) + torch.exp(sink - top)
    out = torch.bmm(weight, rows) / z
    return [out.to(torch.bfloat16).reshape(s["q"].shape),
            (top + torch.log(z)).reshape(s["q"].shape[:3])]


PLAIN = {"append": _append_plain, "window": _window_plain, "store": _store_plain,
         "gather": _gather_plain, "decode": _decode_plain}


# ---- the framework's operators ----

def _append_own(s):
    c = s["case"]
    got = _package().append_slots(s["table"], s["old"], s["new"], s["free"], ratio=c["ratio"],
                                  rows=c["rows"], out=s["out"])
    return [*got, s["table"]]


def _window_own(s):
    c = s["case"]
    return list(_package().window_slots(s["table"], s["length"], c["q_len"], c["window"],
                                        first=c["first"], out=s["out"]))


def _store_own(s):
    remnant = _package()
    remnant.mx4_store_rows(s["x"], s["weight"], 1e-6, s["loc"], s["positions"], s["freqs"],
                           s["pool"])
    return remnant.mx4_gather_bf16(s["pool"], s["loc"][None], None, s["out"])


def _gather_own(s):
    return _package().mx4_gather_bf16(s["pool"], s["slots"], s["lengths"], s["out"])


def _decode_own(s):
    c, remnant = s["case"], _package()
    if s["workspace"] is None:  # kept, as a serving loop keeps it
        _, need = remnant.get_mx4_decode_metadata(c["batch"] * c["q_len"], c["heads"], c["topk"],
                                                  c["window"])
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    return list(remnant.mx4_sparse_decode_fwd(
        s["q"], s["pool"], s["table"], s["indices"], seqlens=s["seqlens"],
        topk_length=s["lengths"], sink=s["sink"], out=s["out"], lse=s["lse"],
        workspace=s["workspace"], swa_pool=s["swa_pool"], swa_indices=s["swa_indices"]))


OWN = {"append": _append_own, "window": _window_own, "store": _store_own, "gather": _gather_own,
       "decode": _decode_own}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----

def _mean_log_uniform(a, b, most):
    """Mean of min(x, most) for x log-uniform on [a, b]."""
    if most <= a or a == b:
        return min(b, most)
    if most >= b:
        return (b - a) / math.log(b / a)
    return ((most - a) + most * math.log(b / most)) / math.log(b / a)


def work(case):
    c = case
    if c["kind"] == "append":
        records = 7 / 8 * c["batch"] * _mean_log_uniform(max(1, c["new"] // 32), c["new"],
                                                         c["new"]) / c["ratio"]
        # lengths in; slots, positions, starts and record counts out; a page read and written
        return {"bytes": 16 * c["batch"] + 8 * c["rows"] + 8 * records / PAGE, "flops": 0}
    if c["kind"] == "window":
        tokens, width = c["batch"] * c["q_len"], c["first"] + c["window"]
        live = _mean_log_uniform(max(1, c["length"] // 32), c["length"], width)
        return {"bytes": tokens * (4 * width + 4) + c["batch"] * (4 + 4 * live / PAGE), "flops": 0}
    if c["kind"] == "store":
        valid = int(c["rows"] * c["valid"])
        per = DIM * (2 if c["dtype"] == "bfloat16" else 4) + REC + (260 if c["rope"] else 0)
        # (written, then read back as BF16 rows)
        return {"bytes": valid * (per + REC) + c["rows"] * (4 + 4 + 2 * DIM) + 4 * DIM,
                "flops": valid * DIM * 8}
    if c["kind"] == "gather":
        rows, valid = c["queries"] * c["k"], c["queries"] * int(c["k"] * c["valid"])
        return {"bytes": 0.98 * valid * REC + rows * (4 + 2 * DIM), "flops": valid * DIM}
    tokens = c["batch"] * c["q_len"]
    mean = _mean_log_uniform(c["shortest"], c["context"], min(c["valid"], c["topk"]))
    per = mean * (REC + 4) + c["window"] * (584 + 4) + c["heads"] * (2 * DIM * 2 + 4) + 8
    return {"bytes": tokens * per,
            "flops": tokens * c["heads"] * (mean + c["window"]) * DIM * 4}


# ---- expected values in 64 bits ----

def _exact_code(n):
    """[rows, 512] float64 -> the nearest E2M1 values times their groups' powers of two."""
    groups = n.reshape(-1, 16, 32)
    amax = groups.abs().amax(-1, keepdim=True).clamp_min(1e-4)
    scale = torch.exp2(torch.ceil(torch.log2(amax / 6.0)).clamp_max(32))
    v = groups.abs() / scale
    # between two neighbours the midpoint goes to the even code: 0, 1, 2 and 4
    out = torch.zeros_like(v)
    for level, above, tie in ((0.5, 0.25, False), (1.0, 0.75, True), (1.5, 1.25, False),
                              (2.0, 1.75, True), (3.0, 2.5, False), (4.0, 3.5, True),
                              (6.0, 5.0, False)):
        out = torch.where((v >= above) if tie else (v > above), level, out)
    return (out * scale * torch.sign(groups)).reshape(-1, DIM)


def _exact_store(s):
    x = s["x"].double()
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].double()
    n = n.to(torch.bfloat16).double()
    if s["freqs"] is not None:
        f = s["freqs"][s["positions"].long() * 4].to(torch.complex128)
        tail = torch.view_as_complex(n[:, NOPE:].reshape(-1, PAIRS, 2).contiguous()) * f
        tail = torch.view_as_real(tail).reshape(-1, 2 * PAIRS).to(torch.bfloat16).double()
        n = torch.cat([n[:, :NOPE], tail], 1)
    return _exact_code(n) * (s["loc"] >= 0)[:, None]


def _exact_mx4(record):
    """Record bytes -> float64 values: sign, two exponent bits, one mantissa bit."""
    byte = record[:, :256].long()
    code = torch.stack([byte % 16, byte // 16], -1).reshape(-1, DIM)
    exponent, half = code // 2 % 4, code % 2
    value = torch.where(exponent == 0, half * 0.5,
                        (1 + 0.5 * half) * torch.exp2(exponent.double() - 1))
    value = torch.where(code >= 8, -value, value).double()
    return value * torch.exp2(record[:, 256:].double() - 127).repeat_interleave(32, 1)


def _exact_gather(s):
    slots = s["slots"].clone()
    for query, length in enumerate(s["lengths"].tolist()):
        slots[query, length:] = -1
    slots = slots.reshape(-1).long()
    out = torch.zeros(slots.numel(), DIM, dtype=torch.float64, device=DEV)
    live = slots >= 0
    out[live] = _exact_mx4(s["pool"].view(-1, REC)[slots[live]])
    return out


def _exact_native(pool, slots):
    page, row = slots // PAGE, slots % PAGE
    rows = torch.empty(slots.numel(), DIM, dtype=torch.float64, device=DEV)
    at = row[:, None] * NATIVE_DATA + torch.arange(NATIVE_DATA, device=DEV)
    data = pool[page[:, None], at]
    scale = pool[page[:, None], PAGE * NATIVE_DATA + row[:, None] * 8 + torch.arange(7, device=DEV)]
    codes = data[:, :NOPE].contiguous().view(torch.float8_e4m3fn).double()
    rows[:, :NOPE] = codes * torch.exp2(scale.double() - 127).repeat_interleave(64, 1)
    rows[:, NOPE:] = data[:, NOPE:].contiguous().view(torch.bfloat16).double()
    return rows


def _exact_decode(s):
    c = s["case"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.empty(s["lse"].shape, dtype=torch.float64, device=DEV)
    sink = s["sink"].double()[:, None]
    records = s["pool"].view(-1, REC)
    for b in range(c["batch"]):
        for t in range(c["q_len"]):
            record = s["indices"][b, t, :int(s["lengths"][b * c["q_len"] + t])].long()
            slot = s["table"][b, record // PAGE].long() * PAGE + record % PAGE
            rows = _exact_mx4(records[slot])
            if c["window"]:
                w = s["swa_indices"][b, t].long()
                rows = torch.cat([rows, _exact_native(s["swa_pool"], w)])
            logits = torch.cat([s["q"][b, t].double() @ rows.t().contiguous() * SCALE, sink], 1)
            lse[b, t] = torch.logsumexp(logits, 1)
            out[b, t] = torch.softmax(logits, 1)[:, :-1].contiguous() @ rows
    return [out, lse]


def exact(case, seed):
    if case["kind"] in ("append", "window"):
        return None  # whole numbers
    s = prepare(case, seed)
    return {"store": _exact_store, "gather": _exact_gather,
            "decode": _exact_decode}[case["kind"]](s)
