"""Position rotation and cache append in 64 bits: the formulas, one token and one group at a time."""
from __future__ import annotations

import numpy as np

from . import formats

GROUP = 16
MIN_EXP = -100


def rotate(x: np.ndarray, positions: np.ndarray, table: np.ndarray | None, interleaved: bool) -> np.ndarray:
    """x [T, H, D] with the first R = table.shape[1] elements of each head rotated; NaN outside the table."""
    y = np.array(x, dtype=np.float64)
    if table is None:
        return y
    half = table.shape[1] // 2
    for t, p in enumerate(positions):
        inside = 0 <= p < table.shape[0]
        row = table[p].astype(np.float64) if inside else np.full(2 * half, np.nan)
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            y[t, :, a] = x[t, :, a] * row[i] - x[t, :, b] * row[half + i]
            y[t, :, b] = x[t, :, b] * row[i] + x[t, :, a] * row[half + i]
    return y


def needed_exp(rows: np.ndarray) -> int:
    """Smallest e >= MIN_EXP with 2^e * 448 >= every finite |row element|."""
    a = np.abs(rows[np.isfinite(rows)])
    top = float(a.max()) if a.size else 0.0
    e = MIN_EXP
    if top > 0:
        e = max(e, int(np.ceil(np.log2(top / 448.0))) - 1)
        while np.ldexp(448.0, e) < top:
            e += 1
    return e


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 number, ties to even, saturating; NaN stays."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        mag = np.where(np.isfinite(x), np.abs(x), 0.0)
        _, e = np.frexp(mag)
        step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
        y = np.clip(np.rint(np.where(np.isfinite(x), x, 0.0) / step) * step, -448.0, 448.0)
        y = np.where(np.isinf(x), np.sign(x) * 448.0, y)
    return np.where(np.isnan(x), np.nan, y)


def append_blk(key, value, k_codes, v_codes, scales, starts, seq_lens, table, pblk):
    """What a block-scaled append leaves: key / value [T, HKV, D] already rotated, codes uint8 [NB, PBLK, HKV, D],
    scales uint8 [NB, PBLK / 16, HKV, 2].  Returns float64 code values of K and V (as codes stand, before their
    scale) and the scale bytes."""
    dec = formats.e4m3fn_table()
    vals = [dec[k_codes].copy(), dec[v_codes].copy()]
    sc = scales.astype(np.int64).copy()
    for s, n in enumerate(np.diff(starts)):
        first, length = int(seq_lens[s]) - int(n), int(seq_lens[s])
        lo = max(first, 0)
        for g in range(lo // GROUP, (length + GROUP - 1) // GROUP if n > 0 else 0):
            t0 = g * GROUP
            if t0 // pblk >= table.shape[1]:
                continue
            blk, part = int(table[s, t0 // pblk]), t0 % pblk // GROUP
            if not 0 <= blk < k_codes.shape[0]:
                continue
            a, b = max(t0, lo), min(t0 + GROUP, length)
            old = slice(t0 % pblk, t0 % pblk + max(0, min(first - t0, GROUP)))
            new = slice(a % pblk, a % pblk + b - a)
            for x, src in enumerate((key, value)):
                rows = src[starts[s] + a - first:starts[s] + b - first]
                for h in range(rows.shape[1]):
                    e = needed_exp(rows[:, h])
                    if t0 < first:
                        before = int(sc[blk, part, h, x]) - 127
                        e = max(e, before)
                        if e > before:
                            vals[x][blk, old, h] = round_e4m3(vals[x][blk, old, h] * 2.0 ** (before - e))
                    sc[blk, part, h, x] = e + 127
                    vals[x][blk, new, h] = round_e4m3(rows[:, h] * 2.0 ** -e)
    return vals[0], vals[1], sc.astype(np.uint8)
