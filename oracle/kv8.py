"""Numpy restatement, in 64 bits, of the 8-bit paged KV cache: append, read-back and attention.

Test infrastructure only.  The cache is ``vals[2, NB, BS, Hkv, D]`` (the e4m3 numbers, not their bytes)
and ``exps[2, NB, Hkv]`` (scale exponents) of one layer.
"""

from __future__ import annotations

import numpy as np

MIN_EXP = -118


def e4m3_round(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value, ties to even: four significant bits, steps of at least 2^-9; non-finite values
    and what would round past 448 become NaN."""
    x = np.asarray(x, np.float64)
    out = np.full(x.shape, np.nan)
    ok = np.isfinite(x)
    a = np.abs(x[ok])
    step = np.exp2(np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    y = np.round(x[ok] / step) * step
    out[ok] = np.where(np.abs(y) <= 448, y, np.nan)
    return out


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 bytes."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * np.exp2(e.astype(np.float64) - 7))
    v[(b & 127) == 127] = np.nan
    return np.where(b & 128, -v, v)


def scale_exponent(rows: np.ndarray) -> np.ndarray:
    """Smallest e >= MIN_EXP with every finite |rows[:, h]| <= 448 2^e, per head."""
    a = np.where(np.isfinite(rows), np.abs(rows), 0).max(axis=(0, 2))
    e = np.full(a.shape, MIN_EXP)
    for h, x in enumerate(a):
        while x > 448 * 2.0 ** float(e[h]):
            e[h] += 1
    return e


def append(vals, exps, table, seq_len: int, k, v) -> None:
    """Rows k, v [n, Hkv, D] become positions seq_len - n .. seq_len - 1 of one sequence."""
    bs = vals.shape[2]
    n0 = seq_len - k.shape[0]
    start = max(n0, 0)
    for page in range(start // bs, -(-seq_len // bs) if seq_len > start else 0):
        blk = table[page] if page < len(table) else -1
        if not 0 <= blk < vals.shape[1]:
            continue
        a, e = max(start, page * bs), min(seq_len, (page + 1) * bs)
        for plane, x in ((0, k), (1, v)):
            rows = np.asarray(x[a - n0:e - n0], np.float64)
            ex = scale_exponent(rows)
            r0 = a - page * bs
            if r0 > 0:
                old = exps[plane, blk]
                ex = np.maximum(ex, old)
                kept = vals[plane, blk, :r0]
                vals[plane, blk, :r0] = np.where((ex > old)[None, :, None],
                                                 e4m3_round(kept * np.exp2((old - ex).astype(np.float64))[None, :, None]),
                                                 kept)
            vals[plane, blk, r0:r0 + e - a] = e4m3_round(rows * np.exp2(-ex.astype(np.float64))[None, :, None])
            exps[plane, blk] = ex


def rows_of(vals, exps, table, positions) -> tuple[np.ndarray, np.ndarray]:
    """K and V [n, Hkv, D] at the positions (zeros where there is none)."""
    bs = vals.shape[2]
    out = np.zeros((2, len(positions)) + vals.shape[3:])
    for i, p in enumerate(positions):
        if p < 0 or p // bs >= len(table) or not 0 <= table[p // bs] < vals.shape[1]:
            continue
        blk = table[p // bs]
        out[:, i] = vals[:, blk, p % bs] * np.exp2(exps[:, blk].astype(np.float64))[..., None]
    return out[0], out[1]


def attention(q, vals, exps, tables, seq_lens, q_lens, scale) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """out [B, T, Hq, D]; and, for error bounds, sum_j w_j |V_j| and the largest scale * sum |q| |k| a row meets."""
    q = np.asarray(q, np.float64)
    B, T, hq, D = q.shape
    hkv = vals.shape[3]
    G = hq // hkv
    out, mass, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros((B, T, hq, 1))
    for b in range(B):
        n = int(seq_lens[b])
        k, v = rows_of(vals, exps, tables[b], range(max(n, 0)))
        for t in range(int(q_lens[b])):
            see = n - int(q_lens[b]) + t + 1
            if see <= 0:
                continue
            for h in range(hq):
                kk, vv = k[:see, h // G], v[:see, h // G]
                s = scale * (kk @ q[b, t, h])
                with np.errstate(invalid="ignore"):
                    w = np.exp(s - s.max())
                w /= w.sum()
                out[b, t, h] = w @ vv
                mass[b, t, h] = w @ np.abs(vv)
                size[b, t, h] = (scale * (np.abs(kk) @ np.abs(q[b, t, h]))).max()
    return out, mass, size
