"""CPU: the 64-bit attention and its error bounds, which the kernels' tests go by."""

from __future__ import annotations

import numpy as np
import pytest

import kv8_reference as ref
from oracle import kv8 as o


def test_bytes_and_the_oracles_attention():
    rng = np.random.default_rng(0)
    vals, exps = ref.sparse_pool(rng, 9, 16, 2, 64)
    assert (o.e4m3_values()[ref.e4m3_bytes(vals)] == vals).all()
    tables = rng.permutation(9).astype(np.int32)[:8].reshape(2, 4)
    tables[1, 1] = -1
    q = rng.standard_normal((2, 3, 4, 64))
    lens, ql = [64, 37], [3, 2]
    r = ref.attention(q[:1], vals, exps, tables[:1], lens[:1], ql[:1], 0.125)
    out, mass, size = o.attention(q[:1], vals, exps, tables[:1], lens[:1], ql[:1], 0.125)
    for a, b in ((r["out"], out), (r["mass"], mass), (r["size"], size)):
        np.testing.assert_allclose(a, b, rtol=1e-12)
    # a page that is missing takes no part
    full = ref.attention(q, vals, exps, tables, lens, ql, 0.125)
    seen = np.r_[0:16, 32:36]
    k, v = o.rows_of(vals, exps, tables[1], seen)
    s = 0.125 * k[:, 1] @ q[1, 0, 3]
    w = np.exp(s - s.max())
    np.testing.assert_allclose(full["out"][1, 0, 3], w @ v[:, 1] / w.sum(), rtol=1e-12)
    assert (full["out"][1, 2] == 0).all()


@pytest.mark.parametrize("n,hq,hkv,d,t", [(4096, 2, 2, 64, 1), (8192, 8, 1, 256, 2), (1000, 4, 1, 128, 3)])
def test_a_lost_position_exceeds_the_bound(n, hq, hkv, d, t):
    rng = np.random.default_rng(n)
    vals, exps = ref.sparse_pool(rng, n // 16 + 1, 16, hkv, d)
    tables = rng.permutation(n // 16 + 1).astype(np.int32)[None]
    q = 0.25 * rng.standard_normal((1, t, hq, d))  # weights alike: each position counts
    r = ref.attention(q, vals, exps, tables, [n], [t], d ** -0.5)
    tol = ref.bound(r, exps, "bf16")
    for j in [0, 1, n - t, *rng.integers(0, n - t, 20)]:
        off = np.abs(ref.attention(q, vals, exps, tables, [n], [t], d ** -0.5, skip=int(j))["out"] - r["out"])
        assert (off > tol).any(), j
