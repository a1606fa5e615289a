"""The 8-bit cache and the page operators in 64 bits, one sequence, block and page at a time (NumPy, CPU)."""
from __future__ import annotations

import math

import numpy as np

GRAIN = 64
TOP = 448.0
MIN_EXPONENT, MAX_EXPONENT = -117, 119


def e4m3_table() -> np.ndarray:
    """The values of the 256 codes: sign, four exponent bits of bias 7, three of fraction; 0x7f and 0xff are NaN."""
    out = np.empty(256)
    for code in range(256):
        e, f = code >> 3 & 15, code & 7
        x = math.nan if code & 127 == 127 else (f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10))
        out[code] = -x if code >> 7 else x
    return out


TABLE = e4m3_table()


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """The e4m3 value nearest to x, ties to the even code, saturating; NaN stays NaN."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), TOP)
    _, e = np.frexp(np.maximum(np.where(np.isnan(a), 0.0, a), 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.copysign(np.minimum(np.rint(a / step) * step, TOP), x)


def scale_for(amax: float) -> float:
    """The smallest power of two s with amax <= 448 s, its exponent within its limits."""
    k = MIN_EXPONENT
    while k < MAX_EXPONENT and amax > TOP * 2.0 ** k:
        k += 1
    return 2.0 ** k


def store(rows, values, scales, slots):
    """rows [T, KVH, 128] -> copies of (values [slots, KVH, 128], scales [slots / 64, KVH]) with the rows stored."""
    values, scales = values.astype(np.float64).copy(), scales.astype(np.float64).copy()
    rows = np.asarray(rows, np.float64)
    last = {}  # slot -> token: of two rows for a slot the later one stays
    for t, s in enumerate(np.asarray(slots).tolist()):
        if 0 <= s < len(values):
            last[s] = t
    for block in sorted({s // GRAIN for s in last}):
        mine = {s: t for s, t in last.items() if s // GRAIN == block}
        lo = block * GRAIN
        for h in range(rows.shape[1]):
            x = np.stack([rows[t, h] for t in mine.values()])
            fine = np.where(np.isfinite(x), np.abs(x), 0.0)
            old = scales[block, h]
            if not old > 0 or lo in mine:
                old = 0.0
            new = max(old, scale_for(float(fine.max())))
            if old > 0 and new > old:
                for s in range(lo, lo + GRAIN):
                    if s not in mine:
                        values[s, h] = to_e4m3(values[s, h] * (old / new))
            for s, t in mine.items():
                values[s, h] = to_e4m3(np.where(np.isfinite(rows[t, h]), rows[t, h], np.nan) / new)
            scales[block, h] = new
    return values, scales


def dequantised(values, scales):
    """[NB, block, KVH, 128] values and [NB, block / 64, KVH] scales -> what they stand for."""
    return values.astype(np.float64) * np.repeat(scales.astype(np.float64), GRAIN, axis=1)[..., None]


def attention(q, k, v, tables, len_q, len_k, scale, block):
    """Causal attention of the last len_q[b] tokens of every sequence over its len_k[b] tokens in the pages.

    q [sum len_q, H, 128]; k, v [NB, block, KVH, 128].  Returns (out, weight, score, small), the last three for bounds of errors:
    weight = sum p |v|; score = the largest sum |q||k| scale of a row; small = sum min(p |v|, 2^-21 p16 |v| + 2^-31 max p max |v|)
    with p16 the largest p of a token's sixteen: what probabilities that underflow in fp16 may cost.  A sequence without keys gives
    zeros.
    """
    t, h, d = q.shape
    nb, kvh = k.shape[0], k.shape[2]
    g = h // kvh
    out, weight, small, score = np.zeros((t, h, d)), np.zeros((t, h, d)), np.zeros((t, h, d)), np.zeros((t, h, 1))
    row = 0
    for b in range(len(len_q)):
        n = int(len_k[b])
        pages = np.clip(np.asarray(tables[b][:-(-n // block)], np.int64), 0, nb - 1)
        kk, vv = (x[pages].reshape(-1, kvh, d)[:n].astype(np.float64) for x in (k, v))
        for i in range(int(len_q[b])):
            seen = n - int(len_q[b]) + i + 1
            if seen > 0:
                for head in range(h):
                    kh, vh = kk[:seen, head // g], vv[:seen, head // g]
                    qr = q[row, head].astype(np.float64)
                    s = kh @ qr * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[row, head] = p @ vh
                    av = np.abs(vh)
                    weight[row, head] = p @ av
                    p16 = np.repeat(np.pad(p, (0, -seen % 16)).reshape(-1, 16).max(1), 16)[:seen]
                    small[row, head] = np.minimum(p[:, None] * av, (2.0 ** -21 * p16)[:, None] * av + 2.0 ** -31 * p.max() * av.max()).sum(0)
                    score[row, head] = (np.abs(kh) @ np.abs(qr)).max() * abs(scale)
            row += 1
    return out, weight, score, small


def copy_pages(caches, src, dst, block, tokens=None, tables=None):
    """Copies of the caches and tables with the pairs carried out, and whether one was left out."""
    nb = caches[0].shape[0]
    tables = None if tables is None else np.asarray(tables, np.int32)
    pairs = [(int(s), int(d)) for s, d in zip(src, dst)]
    live = [0 <= s < nb and 0 <= d < nb for s, d in pairs]

    def clash(i):
        return any(live[j] and j != i and (pairs[j][0] == pairs[i][1] or (pairs[j][1] == pairs[i][1] and j > i)) for j in range(len(pairs)))

    good = [live[i] and not clash(i) for i in range(len(pairs))]
    out = [c.copy() for c in caches]
    for i, (s, d) in enumerate(pairs):
        if not good[i]:
            continue
        for c, o in zip(caches, out):
            rows = c.shape[1] if tokens is None else -(-min(max(int(tokens[i]), 0), block) * c.shape[1] // block)
            o[d, :rows] = c[s, :rows]
    if tables is not None:
        to = {}
        for i, (s, d) in enumerate(pairs):
            if good[i]:
                to.setdefault(s, d)
        tables = np.vectorize(lambda e: to.get(int(e), int(e)), otypes=[np.int32])(tables) if tables.size else tables
    return out, tables, any(live[i] and not good[i] and pairs[i][0] != pairs[i][1] for i in range(len(pairs)))
