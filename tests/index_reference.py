"""Plain definitions of the index records, of what is computed from them, and of the tree
attention, for the tests: numpy in float32 where the codec fixes each rounding, float64
otherwise. Nothing of the library is used."""

import numpy as np
import torch

from mx4_reference import PAGE, bf16, native_rows

KEY, DIM, PAGE_BYTES = 128, 512, 8448
BF16 = 2.0 ** -8   # half a step of a BF16 value, relative to it
F32 = 2.0 ** -24


def codes_of(n):
    """[rows, 128] BF16 values as float32 -> E4M3 codes uint8 [rows, 128], scales float32
    [rows]."""
    special = ~np.isfinite(n).all(-1)
    safe = np.where(special[:, None], 1.0, n).astype(np.float64)
    amax = np.maximum(np.abs(safe).max(-1), np.float64(np.float32(1e-4)))
    # smallest e with amax <= 448 * 2^e (m in [1/2, 1): 448 = 0.875 * 2^9)
    m, k = np.frexp(amax)
    e = k - 9 + (m > 0.875)
    v = np.abs(safe) * 2.0 ** -e[:, None].astype(np.float64)
    # eight steps an octave from 2^-6 on, the same step below; ties to even
    octave = np.maximum(np.floor(np.log2(np.maximum(v, 1e-300))), -6)
    steps = np.rint(v / 2.0 ** (octave - 3))  # 8 .. 16 of a normal, 0 .. 8 of a subnormal
    code = np.where((octave == -6) & (steps < 8), steps, (octave + 7) * 8 + steps - 8)
    code = code.astype(np.int64) + 128 * np.signbit(np.where(special[:, None], 1.0, n))
    code[special] = 0
    scale = np.where(special, np.nan, 2.0 ** e.astype(np.float64))
    return code.astype(np.uint8), scale.astype(np.float32)


def levels():
    """float64 [256]: the value of each E4M3 code."""
    c = np.arange(256)
    e, m = c // 8 % 16, c % 8
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[(c % 128) == 127] = np.nan
    return np.where(c >= 128, -v, v)


def store_rows(x, weight, eps, positions=None, freqs=None, ratio=4):
    """Rows (float32 / bfloat16 tensor [n, 128]) -> (codes, scales), every rounding the
    codec's."""
    x = x.float().numpy()
    one = np.float32
    with np.errstate(all="ignore"):
        sq = (x * x).reshape(-1, 16, 8)
        p = sq[..., 0]
        for i in range(1, 8):
            p = p + sq[..., i]
        while p.shape[1] > 1:
            p = p[:, 0::2] + p[:, 1::2]
        r = one(1) / np.sqrt(p * one(1 / 128) + one(eps))
        n = bf16((x * r) * np.asarray(weight, np.float32))
        if freqs is not None:
            f = freqs.numpy()[np.asarray(positions, np.int64) * ratio]
            c, s = f.real.astype(np.float32), f.imag.astype(np.float32)
            re, im = n[:, 64::2].copy(), n[:, 65::2].copy()
            n[:, 64::2] = bf16(re * c - im * s)
            n[:, 65::2] = bf16(re * s + im * c)
    return codes_of(n)


def page_rows(pool):
    """Codes [slots, 128] and scales [slots] of uint8 [pages, 8448]."""
    pool = np.ascontiguousarray(pool)
    return (pool[:, :8192].reshape(-1, KEY),
            np.ascontiguousarray(pool[:, 8192:]).view(np.float32).reshape(-1))


def make_pool(codes, scales):
    pages = len(scales) // PAGE
    return np.concatenate([codes.reshape(pages, -1),
                           scales.astype(np.float32).reshape(pages, -1).view(np.uint8)], 1)


def scores(q, weights, pool, table, lengths, width):
    """(scores float64 [B, Sq, width], tolerance). A dot product is a float32 sum of 128
    exact products: at most 130 roundings, each 2^-24 of the sum of magnitudes; the sum over
    heads, its factors and the record's scale add at most heads + 10 more."""
    b, sq, h, _ = q.shape
    code, scale = page_rows(pool)
    lv = levels()
    qc, qs = codes_of(q.float().numpy().reshape(-1, KEY))
    qv = lv[qc].reshape(b, sq, h, KEY)
    a = weights.astype(np.float64) * qs.reshape(b, sq, h)
    out, tol = np.full((b, sq, width), -np.inf), np.zeros((b, sq, width))
    for i in range(b):
        r = np.arange(min(width, table.shape[1] * PAGE))
        page = table[i, r // PAGE].astype(np.int64)
        ok = (page >= 0) & (page < len(pool))
        r = r[ok]
        slot = page[ok] * PAGE + r % PAGE
        k, c = lv[code[slot]], scale[slot].astype(np.float64)
        for j in range(sq):
            live = r < lengths[i * sq + j]
            with np.errstate(invalid="ignore"):
                dots = qv[i, j] @ k[live].T
                # (a NaN code is NaN, also where another term is)
                s = (np.where(dots < 0, 0, dots) * a[i, j][:, None]).sum(0) * c[live]
                mag = np.abs(c[live]) * (np.abs(a[i, j])[:, None] * (np.abs(qv[i, j]) @ np.abs(k[live]).T)).sum(0)
            out[i, j, r[live]] = s
            tol[i, j, r[live]] = (130 + h + 10) * F32 * mag
    return out, tol


def topk(scores, lengths, k):
    """(indices [rows, k], counts [rows]) of scores [rows, width]."""
    rows, width = scores.shape
    idx, counts = np.full((rows, k), -1, np.int64), np.zeros(rows, np.int64)
    for i in range(rows):
        n = width if lengths is None else min(max(int(lengths[i]), 0), width)
        x = scores[i, :n].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x) + 0.0
        best = np.sort(np.lexsort((np.arange(n), -x))[:k])
        idx[i, :len(best)] = best
        counts[i] = len(best)
    return idx, counts


def paths(parents):
    """Nodes on each node's path, root first, or None for padding."""
    out = []
    for j in range(len(parents)):
        at, path = j, []
        while at >= 0 and -1 <= parents[at] < at:
            path.append(at)
            at = parents[at]
        out.append(path[::-1] if at == -1 else None)
    return out


def tree(q, pool, table, lengths, parents, window=None, past_pool=None, past_table=None,
         past_lengths=None, sink=None, scale=None):
    """Attention of drafted trees in float64: (out, lse, out's tolerance, lse's).

    The tolerances count roundings: each weight may be rounded to BF16 (2^-8 of it) above
    and below the fraction, and the output is (2^-8); a logit is a float32 sum of 512 exact
    products and moves by at most 520 * 2^-24 of the sum of their magnitudes; in units of
    log2 it, the reference and their difference are rounded, 3 * 2^-24 of its size and of
    the largest's; exp2, log2 and the float32 sums are held to 2^-18 altogether. A weight
    in the units of its row's scale that falls below 2^-126 becomes zero: at most 2^-126 *
    448 * 2^18 < 2^-99 of a coordinate for each row, the sum of weights being at least
    2^-18."""
    b, n, h, _ = q.shape
    scale = DIM ** -0.5 if scale is None else scale
    qd = q.double().numpy()
    out, lse = np.zeros((b, n, h, DIM)), np.full((b, n, h), -np.inf)
    tol, ltol = np.zeros_like(out), np.full((b, n, h), 1e-30)

    def rows_at(p, t, r):
        r = np.asarray(r, np.int64)
        r = r[(r >= 0) & (r // PAGE < t.shape[0])]
        page = t[r // PAGE].astype(np.int64)
        ok = (page >= 0) & (page < len(p))
        return native_rows(p, (page * PAGE + r % PAGE)[ok])

    for i in range(b):
        held = max(int(lengths[i]), 0)
        for j, path in enumerate(paths(parents[i].tolist())):
            if sink is not None:
                lse[i, j] = sink
                ltol[i, j] = 2.0 ** -18 * (1 + np.abs(lse[i, j]))
            if path is None:
                continue
            lowest = held + len(path) - window if window else 0
            see = list(range(max(lowest, 0), held))
            see += [held + x for d, x in enumerate(path) if held + d >= lowest]
            rows = rows_at(pool, table[i], see)
            if past_pool is not None:
                past = rows_at(past_pool, past_table[i], range(max(int(past_lengths[i]), 0)))
                rows = np.concatenate([past, rows])
            if len(rows) == 0:
                continue
            with np.errstate(invalid="ignore", divide="ignore"):
                logits = qd[i, j] @ rows.T * scale
                full = logits if sink is None else np.concatenate([logits, sink[:, None]], 1)
                top = full.max(1, keepdims=True)
                weight = np.exp(full - top)
                z = weight.sum(1, keepdims=True)
                lse[i, j] = (top + np.log(z))[:, 0]
                weight = (weight / z)[:, :len(rows)]
                out[i, j] = weight @ rows
                terms = (np.abs(qd[i, j]) @ np.abs(rows).T).max(1) * abs(scale)
                size = np.abs(logits).max(1) * 1.45 + 20
                move = 520 * F32 * terms + 3 * F32 * size
                spread = weight @ np.abs(rows)
                tol[i, j] = BF16 * (spread + 2 * np.abs(out[i, j])) * (1 + BF16) \
                    + (2 * move + 2.0 ** -18)[:, None] * spread + 2.0 ** -99 * len(rows)
                ltol[i, j] = move + 2.0 ** -18 * (1 + np.abs(lse[i, j]))
    return out, lse, tol, ltol


def random_native(pages, seed):
    """uint8 [pages, 37376] of coded unit-RMS rows with spread coordinates."""
    rng = np.random.default_rng(seed)
    scale = np.exp(rng.uniform(np.log(0.1), np.log(10), DIM))
    x = rng.standard_normal((pages * PAGE, DIM)) * scale
    x = bf16(x / np.sqrt((x * x).mean(1, keepdims=True)))
    return native_pages(x)


def native_pages(x):
    """BF16 rows as float32 [pages * 64, 512] -> Native pages."""
    pages = len(x) // PAGE
    g = x[:, :448].reshape(-1, 7, 64)
    m, k = np.frexp(np.maximum(np.abs(g).max(-1), np.float32(1e-4)).astype(np.float64))
    e = k - 9 + (m > 0.875)
    codes = torch.from_numpy((g / 2.0 ** e[..., None]).astype(np.float32)).to(torch.float8_e4m3fn)
    tail = torch.from_numpy(np.ascontiguousarray(x[:, 448:])).to(torch.bfloat16)
    data = np.concatenate([codes.view(torch.uint8).numpy().reshape(-1, 448),
                           tail.view(torch.uint8).numpy()], 1)
    scale = np.concatenate([e + 127, np.zeros((len(x), 1))], 1).astype(np.uint8)
    return np.concatenate([data.reshape(pages, -1), scale.reshape(pages, -1)], 1)
