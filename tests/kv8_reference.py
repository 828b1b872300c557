"""What the 8-bit cache's attention has to give, in 64 bits, and how far the kernels may be off, with each term from
the arithmetic they state."""

from __future__ import annotations

import numpy as np

from oracle import kv8 as o

LOG2E = 1.4426950408889634


def attention(q, vals, exps, tables, lens, ql, scale, heads=None, skip=None) -> dict:
    """out [B, T, Hq, D] of the query heads `heads` (None: all); `mass` = sum_j w_j |V_j|; per row `size`, the largest
    scale * sum |q| |k|, and `top`, the largest w_j 2^c(j) (c: exponent of V's scale).  `skip`: a position left out of
    every row (a planted mistake)."""
    q = np.asarray(q, np.float64)
    B, T, hq, D = q.shape
    bs, hkv = vals.shape[2], vals.shape[3]
    heads = range(hq) if heads is None else heads
    r = {"out": np.zeros(q.shape), "mass": np.zeros(q.shape), "size": np.zeros((B, T, hq, 1)),
         "top": np.zeros((B, T, hq, 1)), "n": max(int(x) for x in lens)}
    for b in range(B):
        n, m = int(lens[b]), int(ql[b])
        k, v = o.rows_of(vals, exps, tables[b], range(max(n, 0)))
        blk = tables[b][np.arange(max(n, 0)) // bs]
        there = (blk >= 0) & (blk < vals.shape[1])
        if skip is not None:
            there[skip] = False
        c = np.where(there[:, None], exps[1][np.clip(blk, 0, vals.shape[1] - 1)], -10 ** 6)
        pos = n - m + np.arange(m)
        see = (np.arange(max(n, 0))[None] <= pos[:, None]) & there[None]
        ok = see.any(1)
        for h in heads:
            g = h // (hq // hkv)
            if not ok.any():
                continue
            s = np.where(see, scale * (q[b, :m, h] @ k[:, g].T), -np.inf)[ok]
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            at = np.flatnonzero(ok)
            r["out"][b, at, h] = w @ v[:, g]
            r["mass"][b, at, h] = w @ np.abs(v[:, g])
            r["size"][b, at, h, 0] = np.where(see[ok], scale * (np.abs(q[b, at, h]) @ np.abs(k[:, g]).T), 0).max(1)
            r["top"][b, at, h, 0] = (w * np.exp2(np.maximum(c[:, g], -1000).astype(np.float64))).max(1)
    return r


def bound(r: dict, exps, dtype: str) -> np.ndarray:
    """Largest error of an output, A = mass, S = size, n positions, D dims, E = 16 + the largest |exponent| of a scale:

    scores, in nats: D products summed with at most one unit in the last place lost a step, and eleven more steps
      for the factors, (D + 11) 2^-23 S; the exponential's argument, a sum of the score in powers of two, V's
      exponent and the reference (at most 15 + the two), rounded four times, 2^-22 (S log2 e + E); its result, 2^-22.
      A weight and the normaliser are off by that much each: 2.1 of it, of A;
    the reference's moves and the join: sixteen factors of 2^-22 A;
    16-bit queries hold bf16's bits (below 2^-28 of the row's largest not: 2^-39 of the largest product);
    16-bit weights: half a step, 2^-11 A, and below 2^-14 of the format 2^-25, which the reference (2^7 at least for
      the largest) makes 2^-32 of the largest w_j 2^c(j), times 448;
    n sums, a unit in the last place each: (n + 64) 2^-23 A;
    the output: half a step."""
    A, S, n, D = r["mass"], r["size"], r["n"], r["out"].shape[-1]
    E = 16 + np.abs(exps[exps < 120]).max()  # pages never written: exponent 120
    ds = (D + 11) * 2.0 ** -23 * S + 2.0 ** -22 * (S * LOG2E + E) + 2.0 ** -22
    tol = (2.1 * ds + 16 * 2.0 ** -22 + (n + 64) * 2.0 ** -23) * A
    if dtype == "bf16":
        tol = tol + 2.0 ** -11 * A + n * 2.0 ** -32 * 448 * r["top"] + D * 2.0 ** -39 * S * A
    return tol + {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}[dtype] * np.abs(r["out"])


def sparse_pool(rng, nb: int, bs: int, hkv: int, d: int) -> tuple[np.ndarray, np.ndarray]:
    """One layer, vals [2, nb, bs, hkv, d] and exps [2, nb, hkv]: normal K, and V rows with one positive element, its
    dimension spread evenly over the rows.  An output is then a sum over every d-th position or so, without
    cancellation: one that is lost or counted twice moves it by about d / n of itself."""
    vals = np.zeros((2, nb, bs, hkv, d))
    exps = rng.integers(-8, -4, (2, nb, hkv))
    vals[0] = o.e4m3_round(np.clip(rng.standard_normal((nb, bs, hkv, d)) * np.exp2(-exps[0].astype(float))[:, None, :, None],
                                   -448, 448))
    dim = rng.permuted(np.tile(np.arange(nb * bs) % d, (hkv, 1)), axis=1).T.reshape(nb, bs, hkv)
    mag = o.e4m3_round(rng.uniform(0.6, 1, dim.shape) * np.exp2(-exps[1].astype(float))[:, None])
    np.put_along_axis(vals[1], dim[..., None], mag[..., None], axis=-1)
    return vals, exps


def e4m3_bytes(vals: np.ndarray) -> np.ndarray:
    """The bytes of e4m3 numbers."""
    table = o.e4m3_values()[:127]
    b = np.searchsorted(table, np.abs(vals)).astype(np.uint8)
    return b | np.where(np.signbit(vals), 128, 0).astype(np.uint8)
