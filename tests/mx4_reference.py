"""Plain definitions of the 4-bit record codec, of the decode over it and of the slot
maps, for the tests: numpy in float32 where the codec fixes each rounding, float64
otherwise. Nothing of the library is used."""

import numpy as np
import torch

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
PAGE, REC, DIM, NOPE = 64, 272, 512, 448


def bf16(x):
    """float32 array rounded to BF16 (nearest even), as float32."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).float().numpy()


def encode(n):
    """[rows, 512] BF16 values as float32 -> record bytes [rows, 272]."""
    g = n.reshape(-1, 16, 32)
    mag = np.abs(g)
    special = ~np.isfinite(g).all(-1)
    amax = np.where(special, 1.0, np.nan_to_num(mag, nan=0, posinf=0).max(-1)).astype(np.float64)
    # smallest e with max(amax, 1e-4) <= 6 * 2^e, at most 32 (m in [1/2, 1): 6 = 0.75 * 8)
    m, k = np.frexp(np.maximum(amax, np.float64(np.float32(1e-4))))
    e = np.minimum(k - 3 + (m > 0.75), 32)
    v = np.nan_to_num(mag, nan=0, posinf=0).astype(np.float64) * 2.0 ** -e[..., None]
    # nearest level, a midpoint to the even code
    mid = (LEVELS[1:] + LEVELS[:-1]) / 2
    code = np.zeros(v.shape, np.int64)
    for i, x in enumerate(mid):
        code[(v > x) | ((v == x) & (i % 2 == 1))] = i + 1
    code = code + 8 * np.signbit(g)
    code[special] = 0
    code = code.reshape(-1, DIM)
    scale = np.where(special, 255, e + 127)
    return np.concatenate([code[:, 0::2] | code[:, 1::2] << 4, scale], 1).astype(np.uint8)


def decode_rows(rec):
    """Record bytes [..., 272] -> float64 values [..., 512] (scale byte 255: NaN)."""
    rec = np.asarray(rec)
    lv = np.concatenate([LEVELS, -LEVELS])
    byte = rec[..., :256]
    v = lv[np.stack([byte & 15, byte >> 4], -1)].reshape(*rec.shape[:-1], 16, 32)
    s = rec[..., 256:].astype(np.int64)
    scale = np.where(s == 255, np.nan, 2.0 ** (s - 127.0))
    return (v * scale[..., None]).reshape(*rec.shape[:-1], DIM)


def store_rows(x, weight, eps, positions=None, freqs=None):
    """Rows (any of float32 / bfloat16 tensors) -> record bytes, every rounding the codec's."""
    x = x.float().numpy()
    w = np.asarray(weight, np.float32)
    one = np.float32
    with np.errstate(all="ignore"):
        sq = (x * x).reshape(-1, 64, 8)
        p = sq[..., 0]
        for i in range(1, 8):
            p = p + sq[..., i]
        while p.shape[1] > 1:
            p = p[:, 0::2] + p[:, 1::2]
        r = one(1) / np.sqrt(p * one(1 / 512) + one(eps))
        n = bf16((x * r) * w)
        if freqs is not None:
            f = freqs.numpy()[np.asarray(positions, np.int64) * 4]
            c, s = f.real.astype(np.float32), f.imag.astype(np.float32)
            re, im = n[:, NOPE::2].copy(), n[:, NOPE + 1::2].copy()
            n[:, NOPE::2] = bf16(re * c - im * s)
            n[:, NOPE + 1::2] = bf16(re * s + im * c)
    return encode(n)


def native_rows(pool, slots):
    """Native records of a uint8 [pages, 37376] array at slots -> float64 [n, 512]."""
    if len(slots) == 0:
        return np.zeros((0, DIM))
    page, row = slots // PAGE, slots % PAGE
    data = pool[page[:, None], row[:, None] * 576 + np.arange(576)]
    scale = pool[page[:, None], PAGE * 576 + row[:, None] * 8 + np.arange(7)].astype(np.float64)
    codes = torch.from_numpy(np.ascontiguousarray(data[:, :NOPE])).view(torch.float8_e4m3fn)
    head = codes.double().numpy() * np.repeat(2.0 ** (scale - 127), 64, axis=1)
    tail = torch.from_numpy(np.ascontiguousarray(data[:, NOPE:])).view(torch.bfloat16)
    return np.concatenate([head, tail.double().numpy()], 1)


def decode(q, pool, table, indices, seqlens=None, topk_length=None, sink=None, scale=None,
           swa_pool=None, swa_indices=None, swa_lengths=None):
    """Attention in float64: (out, lse, out's tolerance, lse's). Arrays are numpy, q a
    bfloat16 tensor [B, Sq, H, 512].

    The tolerances count roundings: every weight may be rounded to BF16 (half a step,
    2^-8 of it) and every output is (2^-8); a logit is a float32 sum of 512 exact
    products and moves by at most 520 * 2^-24 of the sum of their magnitudes (the sum,
    and the scaling, each rounded), which moves a weight by that factor and lse by that
    much; exp2, log2 and the float32 sums are held to 2^-18 altogether, relative to the
    sum of the terms' magnitudes. Weights are BF16 numbers in units of a record's scale
    over 2^32, the largest scale there is, and one below 2^-126 of the unit may become
    zero: at most 2^-126 * 2^32 * 6 < 2^-91 of a coordinate for each record, over a sum of
    weights of at least 1/2 (the largest weight is in (1/2, 1])."""
    b, sq, h, _ = q.shape
    scale = 512 ** -0.5 if scale is None else scale
    qd = q.double().numpy()
    out, lse = np.zeros((b, sq, h, DIM)), np.full((b, sq, h), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros_like(lse)
    records = pool.reshape(-1, REC)
    for i in range(b):
        for j in range(sq):
            t = i * sq + j
            r = indices[i, j].astype(np.int64)
            if topk_length is not None:
                r = r[:max(int(topk_length[t]), 0)]
            r = r[(r >= 0) & (r < (seqlens[i] if seqlens is not None else 1 << 40))]
            r = r[r // PAGE < table.shape[1]]
            page = table[i, r // PAGE].astype(np.int64)
            ok = (page >= 0) & (page < pool.shape[0])
            rows = decode_rows(records[(page * PAGE + r % PAGE)[ok]])
            if swa_indices is not None:
                w = swa_indices[i, j].astype(np.int64)
                if swa_lengths is not None:
                    w = w[:max(int(swa_lengths[t]), 0)]
                w = w[(w >= 0) & (w < swa_pool.shape[0] * PAGE)]
                rows = np.concatenate([rows, native_rows(swa_pool, w)])
            logits = qd[i, j] @ rows.T * scale
            full = logits if sink is None else np.concatenate([logits, sink[:, None]], 1)
            if full.shape[1] == 0:
                continue
            with np.errstate(invalid="ignore", divide="ignore"):
                top = full.max(1, keepdims=True)
                weight = np.exp(full - np.where(np.isfinite(top), top, 0))
                z = weight.sum(1, keepdims=True)
                lse[i, j] = (np.where(np.isfinite(top), top, 0) + np.log(z))[:, 0]
                weight = np.where(z > 0, weight / z, 0)[:, :rows.shape[0]]
            out[i, j] = weight @ rows
            if rows.shape[0] == 0:
                ltol[i, j] = 2.0 ** -18 * (1 + np.abs(lse[i, j]))
                continue
            terms = (np.abs(qd[i, j]) @ np.abs(rows).T).max(1) * abs(scale)
            move = 520 * 2.0 ** -24 * terms
            spread = weight @ np.abs(rows)
            tol[i, j] = 2.0 ** -8 * (spread + np.abs(out[i, j])) \
                + (2 * move + 2.0 ** -18)[:, None] * spread * (1 + 2.0 ** -8) \
                + 2.0 ** -90 * rows.shape[0]
            ltol[i, j] = move + 2.0 ** -18 * (1 + np.abs(lse[i, j]))
    return out, lse, tol, ltol


def append(table, old, new, free, ratio, rows):
    """(loc, positions, row_starts, seqlens, pages_taken, table after), plain loops."""
    table, at, taken = table.copy(), 0, 0
    loc, pos = np.full(rows, -1, np.int64), np.zeros(rows, np.int64)
    starts, lens = [0], []
    for b, (lo, hi) in enumerate(zip(old.tolist(), new.tolist())):
        o = max(lo, 0) // ratio
        n = max(max(hi, 0) // ratio, o)
        first = -(-o // PAGE)
        for c in range(first, -(-n // PAGE)):
            page = int(free[taken]) if taken < len(free) else -1
            taken += 1
            if c < table.shape[1]:
                table[b, c] = page
        for r in range(o, n):
            if at < rows:
                page = int(table[b, r // PAGE]) if r // PAGE < table.shape[1] else -1
                loc[at] = page * PAGE + r % PAGE if 0 <= page < 1 << 25 else -1
                pos[at] = r
            at += 1
        starts.append(at)
        lens.append(n)
    return loc, pos, np.array(starts), np.array(lens), np.array([taken]), table


def window(table, lengths, q_len, win, first):
    batch = len(lengths)
    slots = np.full((batch, q_len, first + win), -1, np.int64)
    counts = np.zeros(batch * q_len, np.int64)
    for b in range(batch):
        for j in range(q_len):
            p = int(lengths[b]) - q_len + j
            seen = [t for t in range(max(p + 1, 0)) if t < first or t > p - win]
            counts[b * q_len + j] = len(seen)
            for i, t in enumerate(seen):
                page = int(table[b, t // PAGE]) if t // PAGE < table.shape[1] else -1
                if 0 <= page < 1 << 25:
                    slots[b, j, i] = page * PAGE + t % PAGE
    return slots, counts
