"""GPU: the 8-bit paged KV cache against the oracle in 64 bits -- append, RoPE append, read-back, attention."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import kv8 as o

pytestmark = pytest.mark.gpu

EPS = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # half a step, relative


def _torch():
    import torch

    return torch, {"bf16": torch.bfloat16, "f32": torch.float32}


def _round(x, dtype):
    torch, dts = _torch()
    return torch.tensor(np.asarray(x, np.float32)).to(dts[dtype]).float().numpy().astype(np.float64)


class Pool:
    """A one-layer (layer 1 of 2) cache with tables, on both sides; dead bytes are NaN and dead scales garbage."""

    def __init__(self, rng, b, bs, hkv, d, cols):
        from ssd_b200.kernels.kv8_cache import KV8CacheState

        torch, _ = _torch()
        nb = b * cols + 3
        self.bs, self.hkv, self.d = bs, hkv, d
        self.cache = KV8CacheState.allocate(2, nb, bs, hkv, d)
        self.cache.pages.view(torch.uint8).fill_(0x7F)
        self.cache.scales.fill_(float("nan"))
        self.vals = np.full((2, nb, bs, hkv, d), np.nan)
        self.exps = np.full((2, nb, hkv), 120, np.int64)
        self.tables = np.full((b, cols), -1, np.int32)
        perm = rng.permutation(nb)
        for i in range(b):
            self.tables[i] = perm[i * cols:(i + 1) * cols]
        self.dev_tables = torch.tensor(self.tables, device="cuda")

    def append(self, seq_lens, k, v, q_lens, dtype):
        from ssd_b200.kernels.kv8_cache import append_kv8

        torch, dts = _torch()
        t = lambda a: torch.tensor(np.asarray(a, np.float32)).to(dts[dtype]).cuda()  # noqa: E731
        i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
        k, v = _round(k, dtype), _round(v, dtype)  # what the device is given, on both sides
        append_kv8(self.cache, 1, self.dev_tables, i(seq_lens), t(k), t(v), q_lens=i(q_lens))
        for r, (n, m) in enumerate(zip(seq_lens, q_lens)):
            m = min(max(int(m), 0), k.shape[1])
            o.append(self.vals, self.exps, self.tables[r], int(n), k[r, :m], v[r, :m])

    def check(self):
        """The whole layer, dead rows included, byte for byte; the other layer untouched."""
        torch, _ = _torch()
        got = self.cache.pages[:, 1].float().cpu().numpy().astype(np.float64)
        np.testing.assert_array_equal(got, self.vals)
        live = ~np.isnan(self.vals).all(axis=(2, 4))  # pages and heads that hold something
        sc = self.cache.scales[:, 1].cpu().numpy()
        np.testing.assert_array_equal(sc[live], np.exp2(self.exps[live].astype(np.float64)))
        assert (self.cache.pages[:, 0].view(torch.uint8) == 0x7F).all() and self.cache.scales[:, 0].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bs,hkv,d", [(16, 1, 256), (16, 4, 64), (4, 2, 128), (32, 3, 256), (1, 2, 64), (7, 2, 128),
                                      (100, 1, 256)])
def test_append_in_steps_of_every_size(cuda, dtype, bs, hkv, d):
    """Prompts, then single tokens and short runs whose magnitudes rise and fall; rows with nothing new; then a
    rollback: the sequence goes on from a shorter length."""
    rng = np.random.default_rng(bs * d + hkv)
    b = 4
    p = Pool(rng, b, bs, hkv, d, cols=3 + 60 // bs)
    lens = np.zeros(b, int)
    for step, (t, mag) in enumerate([(37, 1.0), (1, 0.01), (1, 900.0), (5, 1.0), (0, 1.0), (3, 2.0 ** -30), (2, 1e30),
                                     (1, 0.0), (4, 1.0)]):
        if step == 6:
            lens = np.maximum(lens - np.arange(b) * 3, 0)  # rolled back by 0, 3, 6, 9 tokens
        ql = np.array([t, max(t - 1, 0), 0 if step % 2 else t, t])
        lens = lens + ql
        k = _round(mag * rng.standard_normal((b, max(t, 1), hkv, d)), dtype)
        v = _round(rng.standard_normal((b, max(t, 1), hkv, d)) * np.exp2(rng.integers(-6, 6, (b, 1, hkv, 1))), dtype)
        p.append(lens, k, v, ql, dtype)
        p.check()


def test_append_skips_what_it_cannot_place(cuda):
    """Tables without a block, pages past the table, q_lens above T and above the length: no write there."""
    torch, _ = _torch()
    rng = np.random.default_rng(5)
    p = Pool(rng, 3, 16, 2, 64, cols=3)
    p.tables[0, 1], p.tables[1, 0] = -1, 10 ** 6
    p.dev_tables = torch.tensor(p.tables, device="cuda")
    k = _round(rng.standard_normal((3, 40, 2, 64)), "bf16")
    p.append([40, 60, 8], k, 2 * k, [40, 99, 40], "bf16")  # row 2: positions -32 .. 7
    p.check()


def test_append_of_non_finite_rows(cuda):
    """Infinities and NaN are stored as NaN and leave the scale to the finite values."""
    rng = np.random.default_rng(6)
    p = Pool(rng, 1, 16, 1, 64, cols=2)
    k = _round(rng.standard_normal((1, 20, 1, 64)), "bf16")
    k[0, 3, 0, 5], k[0, 3, 0, 6], k[0, 17, 0, 0] = np.inf, np.nan, -np.inf
    p.append([20], k, k[:, ::-1].copy(), [20], "bf16")
    p.check()


@pytest.mark.parametrize("bs,hkv,d,n", [(16, 1, 64, 5), (16, 16, 256, 33), (4, 3, 128, 1), (32, 2, 64, 70)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gather_returns_the_stored_values(cuda, dtype, bs, hkv, d, n):
    from ssd_b200.kernels.kv8_cache import gather_kv8

    torch, dts = _torch()
    rng = np.random.default_rng(n)
    p = Pool(rng, 2, bs, hkv, d, cols=80 // bs + 1)
    k = _round(rng.standard_normal((2, 75, hkv, d)), "bf16")
    p.append([75, 40], k, 3 * k, [75, 40], "bf16")
    pos = rng.integers(-2, 40, (2, n)).astype(np.int32)
    pos[0, 0] = 10 ** 6
    gk, gv = gather_kv8(p.cache, 1, p.dev_tables, torch.tensor(pos, device="cuda"), dtype=dts[dtype])
    for r in range(2):
        rk, rv = o.rows_of(p.vals, p.exps, p.tables[r], pos[r])
        np.testing.assert_array_equal(gk[r].float().cpu().numpy(), rk)
        np.testing.assert_array_equal(gv[r].float().cpu().numpy(), rv)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,bs,t", [(8, 1, 256, 16, 1), (16, 16, 256, 16, 5), (4, 2, 128, 4, 7), (4, 1, 64, 16, 3),
                                           (6, 2, 64, 32, 64)])
def test_rope_append(cuda, dtype, hq, hkv, d, bs, t):
    from ssd_b200.kernels.kv8_cache import gather_kv8, rope_append_kv8
    from ssd_b200.models.gemma import rope_tables

    torch, dts = _torch()
    rng = np.random.default_rng(hq * d + t)
    b = 3
    lens, ql = np.array([t + 9, t + 30, t]), np.array([t, t, max(t - 1, 0)])
    p = Pool(rng, b, bs, hkv, d, cols=-(-(t + 30) // bs))
    old = _round(rng.standard_normal((b, 30, hkv, d)), "bf16")
    p.append(lens - ql, old, old, np.minimum(lens - ql, 30), "bf16")
    cos, sin = rope_tables(t + 40, d)
    x = _round(rng.standard_normal((b, t, hq + 2 * hkv, d)), dtype)
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    q = rope_append_kv8(torch.tensor(x.reshape(b * t, -1)).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, i(lens), hq,
                        torch.tensor(cos, device="cuda"), torch.tensor(sin, device="cuda"), q_lens=i(ql))
    got = q.float().cpu().numpy()
    for r in range(b):
        n = int(ql[r])
        at = np.arange(lens[r] - n, lens[r])
        c, s = cos[at].astype(np.float64)[:, None], sin[at].astype(np.float64)[:, None]
        a, z = x[r, :n, :hq + hkv, :d // 2], x[r, :n, :hq + hkv, d // 2:]
        y = np.concatenate([a * c - z * s, z * c + a * s], -1)
        # two products and a sum in fp32, then the output's rounding
        tol = 3 * 2.0 ** -24 * (np.abs(np.concatenate([a, z], -1)) + np.abs(np.concatenate([z, a], -1)))
        assert (np.abs(got[r, :n] - y[:, :hq]) <= tol[:, :hq] + EPS[dtype] * np.abs(y[:, :hq])).all()
        assert (got[r, n:] == 0).all()
        o.append(p.vals, p.exps, p.tables[r], int(lens[r]), y[:, hq:], x[r, :n, hq + hkv:])
        pos = np.arange(lens[r])
        tab = p.dev_tables[r:r + 1].contiguous()
        gk, gv = (g[0].float().cpu().numpy() for g in gather_kv8(p.cache, 1, tab, i(pos[None]), dtype=torch.float32))
        rk, rv = o.rows_of(p.vals, p.exps, p.tables[r], pos)
        np.testing.assert_array_equal(gv, rv)
        # a K value whose fp32 rotation is off in its last bits may round to the next e4m3 value: one step, rarely
        off = np.abs(gk - rk)
        assert (off <= 2.0 ** -3 * np.abs(rk) + 2.0 ** -9 * 448 * np.exp2(p.exps[0, p.tables[r][pos // bs]])[..., None]).all()
        assert (off > 0).mean() <= 1e-3


CASES = [  # dtype, hq, hkv, d, bs, t, sequence lengths
    ("bf16", 8, 1, 256, 16, 1, [1, 2, 15, 16, 17, 33, 127, 128, 129, 300]),
    ("bf16", 16, 16, 256, 16, 5, [5, 6, 255, 256, 257, 1000]),
    ("bf16", 16, 16, 64, 16, 7, [7, 100, 511, 513]),
    ("bf16", 8, 2, 128, 16, 3, [3, 64, 65, 700]),
    ("bf16", 8, 8, 64, 16, 1, [1, 31, 90]),
    ("bf16", 8, 1, 256, 16, 2, [2, 40, 270]),        # 16 rows a KV head
    ("bf16", 8, 1, 256, 16, 3, [3, 47, 200]),        # 24 rows
    ("bf16", 8, 1, 256, 16, 40, [40, 41, 333]),      # prompt chunk: 320 rows
    ("bf16", 4, 4, 128, 16, 65, [65, 128, 600]),
    ("bf16", 16, 4, 64, 16, 150, [150, 407]),
    ("bf16", 4, 2, 128, 4, 5, [5, 9, 130]),          # pages smaller than a tile
    ("bf16", 4, 2, 64, 1, 4, [4, 21]),
    ("bf16", 4, 2, 256, 7, 4, [4, 150]),             # pages that end inside a tile
    ("bf16", 4, 2, 128, 24, 33, [33, 290]),
    ("bf16", 4, 2, 64, 32, 6, [6, 95]),
    ("bf16", 3, 1, 64, 64, 2, [2, 200]),
    ("f32", 4, 1, 64, 16, 5, [5, 77, 200, 129]),
    ("f32", 4, 2, 128, 4, 7, [7, 90]),
    ("f32", 2, 2, 256, 16, 1, [1, 300]),
]


def _attention_inputs(case, seed, spread=2):
    dtype, hq, hkv, d, bs, t, lens = case
    rng = np.random.default_rng(seed)
    b = len(lens)
    p = Pool(rng, b, bs, hkv, d, cols=-(-max(lens) // bs))
    n = max(lens)
    k = rng.standard_normal((b, n, hkv, d)) * np.exp2(rng.integers(-spread, 1, (b, n, hkv, 1)))
    v = rng.standard_normal((b, n, hkv, d)) * np.exp2(rng.integers(-4 * spread, 4 * spread, (b, n, hkv, 1)))
    p.append(lens, k, v, lens, "bf16")
    q = _round(rng.standard_normal((b, t, hq, d)), dtype)
    ql = np.array([t if i % 3 != 1 else max(t - 2, 0) for i in range(b)])
    return p, q, ql


def _tolerance(case, q, p, lens, mass, size, ref):
    """Error of the output, relative to what it sums up.  With A = sum_j w_j |V_j| and S the largest
    scale * sum |q| |k| of the row:
      scores: D products and sums in fp32, the 16-bit form of q (2^-25 of the row's largest, bf16 only) and
              the exponential's own argument and result: ds <= (D + 8) 2^-24 S + 2^-21 + 2^-22 S, and 2^-25
              D terms for q;  a weight's relative error is at most 2 ds, and the
              normaliser's too, so 4 ds A in all;
      weights as 16-bit operands (bf16 only): 2^-11 A, and below 2^-14 of the row's largest contribution an
              absolute 2^-25 each: n 2^-25 448 of the largest w_j 2^c(j);
      sums over n positions in fp32: (n + 64) 2^-24 A;
      the output: half a step."""
    dtype, hq, hkv, d, bs, t, _ = case
    n = max(lens)
    ds = ((d + 8) * 2.0 ** -24 + 2.0 ** -22) * size + 2.0 ** -21
    tol = (4 * ds + (n + 64) * 2.0 ** -24) * mass + EPS[dtype] * np.abs(ref)
    if dtype == "bf16":
        big = np.abs(p.vals[~np.isnan(p.vals)]).max()
        top = np.exp2(p.exps[1][p.exps[1] < 120].max().astype(np.float64)) if (p.exps[1] < 120).any() else 1.0
        tol = tol + 2.0 ** -11 * mass + n * 2.0 ** -25 * 448 * np.minimum(top, mass.max(-1, keepdims=True) * 2)
        tol = tol + 4 * d * 2.0 ** -25 * size / max(big, 1) * mass
    return tol


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
def test_attention_matches_the_oracle(cuda, case):
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    dtype, hq, hkv, d, bs, t, lens = case
    p, q, ql = _attention_inputs(case, seed=hq * d + t + bs)
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    scale = 1 / math.sqrt(d)
    got = paged_kv8_attention(torch.tensor(q).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, i(lens), q_lens=i(ql))
    ref, mass, size = o.attention(q, p.vals, p.exps, p.tables, lens, ql, scale)
    got = got.float().cpu().numpy()
    tol = _tolerance(case, q, p, lens, mass, size, ref)
    bad = np.abs(got - ref) > tol
    assert not bad.any(), (np.abs(got - ref) / np.maximum(tol, 1e-300)).max()
    for r in range(len(lens)):
        assert (got[r, ql[r]:] == 0).all()


@pytest.mark.parametrize("hq,hkv,d,bs,t", [(8, 1, 256, 16, 1), (16, 16, 256, 16, 5), (4, 2, 64, 4, 6), (8, 1, 256, 16, 40)])
def test_attention_without_positions(cuda, hq, hkv, d, bs, t):
    """Lengths of zero, no new tokens, more new tokens than the sequence has: zero rows, nothing read."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, _ = _torch()
    rng = np.random.default_rng(3)
    p = Pool(rng, 4, bs, hkv, d, cols=-(-400 // bs))
    lens = [0, 300, 2, 0]
    k = _round(rng.standard_normal((4, 300, hkv, d)), "bf16")
    p.append(lens, k, k, lens, "bf16")
    p.dev_tables[0] = -1
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    q = _round(rng.standard_normal((4, t, hq, d)), "bf16")
    ql = [t, 0, t, 0]
    got = paged_kv8_attention(torch.tensor(q).bfloat16().cuda(), p.cache, 1, p.dev_tables, i(lens), q_lens=i(ql))
    got = got.float().cpu().numpy()
    assert (got[[0, 1, 3]] == 0).all()
    ref, mass, _ = o.attention(q, p.vals, p.exps, p.tables, lens, ql, 1 / math.sqrt(d))
    dead = max(0, t - 2)
    assert (got[2, :dead] == 0).all()
    assert (np.abs(got[2, dead:] - ref[2, dead:]) <= 2.0 ** -7 * mass[2, dead:]).all()  # 2^-8 out, 2^-11 weights, scores


@pytest.mark.parametrize("dtype,hq,hkv,d,t", [("bf16", 4, 1, 256, 2), ("bf16", 8, 8, 64, 5), ("f32", 4, 1, 64, 3),
                                              ("bf16", 8, 1, 128, 30)])
def test_attention_masks_nan_of_later_tokens(cuda, dtype, hq, hkv, d, t):
    """A new token with NaN in K and V reaches its own and later rows only, V's by dimension."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    rng = np.random.default_rng(8)
    n = 130 + t
    p = Pool(rng, 1, 16, hkv, d, cols=-(-n // 16))
    k = _round(rng.standard_normal((1, n, hkv, d)), "bf16")
    v = _round(rng.standard_normal((1, n, hkv, d)), "bf16")
    v[0, n - 1, 0, 3] = np.nan          # the last token
    v[0, n - 2, hkv - 1, 7] = np.inf    # the one before it, in the last head
    p.append([n], k, v, [n], "bf16")
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    q = _round(rng.standard_normal((1, t, hq, d)), dtype)
    got = paged_kv8_attention(torch.tensor(q).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, i([n]))[0]
    nan = got.isnan().cpu().numpy()
    want = np.zeros_like(nan)
    g = hq // hkv
    want[t - 1, :g, 3] = True
    want[t - 2:, (hkv - 1) * g:, 7] = True
    np.testing.assert_array_equal(nan, want)
    # K: a NaN score spoils the rows that see it, all of their dimensions
    k[0, n - 1, 0, 0] = np.nan
    p.append([n], k, np.nan_to_num(v, posinf=1.0), [n], "bf16")
    got = paged_kv8_attention(torch.tensor(q).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, i([n]))[0]
    nan = got.isnan().cpu().numpy()
    want = np.zeros_like(nan)
    want[t - 1, :g] = True
    np.testing.assert_array_equal(nan, want)


def test_attention_of_pages_whose_scales_lie_far_apart(cuda):
    """V pages at 2^-100 and 2^60, all-zero pages between: no overflow, small pages count where they are all there is."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, _ = _torch()
    rng = np.random.default_rng(9)
    p = Pool(rng, 3, 16, 1, 64, cols=20)
    lens = [320, 320, 320]
    k = _round(rng.standard_normal((3, 320, 1, 64)), "bf16")
    v = rng.standard_normal((3, 320, 1, 64))
    v[0] *= 2.0 ** -100
    v[1, :160] *= 2.0 ** 60
    v[2] = 0
    p.append(lens, k, _round(v, "bf16"), lens, "bf16")
    q = _round(rng.standard_normal((3, 2, 8, 64)), "bf16")
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    got = paged_kv8_attention(torch.tensor(q).bfloat16().cuda(), p.cache, 1, p.dev_tables, i(lens)).float().cpu().numpy()
    ref, mass, size = o.attention(q, p.vals, p.exps, p.tables, lens, [2, 2, 2], 1 / 8)
    assert (got[2] == 0).all()
    # weights' 2^-11 and scores (64 + 16) 2^-24 * 4 S (S < 60) relative to the mass, the output's 2^-8
    assert (np.abs(got - ref)[:2] <= 2.0 ** -8 * np.abs(ref[:2]) + 2.0 ** -10 * mass[:2]).all()


@pytest.mark.parametrize("hq,hkv,d", [(16, 16, 256), (8, 1, 256), (8, 2, 128)])
def test_attention_is_batch_invariant(cuda, hq, hkv, d):
    """A query's bits do not depend on how many new tokens (up to the few-row kernel's rows) or sequences stand
    beside it, nor on max_seq_len."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, _ = _torch()
    rng = np.random.default_rng(12)
    t = 5
    p = Pool(rng, 2, 16, hkv, d, cols=64)
    lens = [777, 400]
    k = _round(rng.standard_normal((2, 777, hkv, d)), "bf16")
    p.append(lens, k, 0.5 * k, lens, "bf16")
    q = torch.tensor(_round(rng.standard_normal((2, t, hq, d)), "bf16")).bfloat16().cuda()
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    full = paged_kv8_attention(q, p.cache, 1, p.dev_tables, i(lens), max_seq_len=1024)
    for j in range(t):
        one = paged_kv8_attention(q[:1, j:j + 1].contiguous(), p.cache, 1, p.dev_tables[:1].contiguous(),
                                  i([lens[0] - t + j + 1]), max_seq_len=800)
        assert torch.equal(one[0, 0], full[0, j])


def test_calls_on_two_streams_and_in_a_graph(cuda):
    """Two streams at once, and a captured step (append, attention) replayed while eager calls run."""
    from ssd_b200.kernels.kv8_cache import append_kv8, paged_kv8_attention

    torch, _ = _torch()
    rng = np.random.default_rng(4)
    b, hq, hkv, d, n = 4, 8, 2, 128, 2000
    p = Pool(rng, b, 16, hkv, d, cols=n // 16 + 1)
    k = _round(rng.standard_normal((b, n, hkv, d)), "bf16")
    p.append([n] * b, k, k, [n] * b, "bf16")
    sl = torch.full((b,), n, dtype=torch.int32, device="cuda")
    qs = [torch.randn((b, 3, hq, d), device="cuda").bfloat16() for _ in range(2)]
    want = [paged_kv8_attention(x, p.cache, 1, p.dev_tables, sl) for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for s, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[s].append(paged_kv8_attention(qs[s], p.cache, 1, p.dev_tables, sl))
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(x, want[s]) for x in outs[s])
    kk = torch.randn((b, 1, hkv, d), device="cuda").bfloat16()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append_kv8(p.cache, 1, p.dev_tables, sl, kk, kk)
        cap = paged_kv8_attention(qs[0], p.cache, 1, p.dev_tables, sl)
    kk.normal_()
    graph.replay()
    torch.cuda.synchronize()
    got = cap.clone()
    append_kv8(p.cache, 1, p.dev_tables, sl, kk, kk)
    assert torch.equal(got, paged_kv8_attention(qs[0], p.cache, 1, p.dev_tables, sl))
    # a larger eager call in between leaves the captured call's memory alone
    big = paged_kv8_attention(torch.randn((b, 40, hq, d), device="cuda").bfloat16(), p.cache, 1, p.dev_tables, sl)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(cap, got) and big.isfinite().all()


def test_strided_rows_and_refusals(cuda):
    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, gather_kv8, paged_kv8_attention

    torch, _ = _torch()
    cache = KV8CacheState.allocate(1, 8, 16, 2, 64)
    tab = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
    sl = torch.tensor([20], dtype=torch.int32, device="cuda")
    qkv = torch.randn((1, 20, 8, 64), device="cuda").bfloat16()
    append_kv8(cache, 0, tab, sl, qkv[:, :, 4:6], qkv[:, :, 6:8])  # views into wider rows
    other = KV8CacheState.allocate(1, 8, 16, 2, 64)
    append_kv8(other, 0, tab, sl, qkv[:, :, 4:6].contiguous(), qkv[:, :, 6:8].contiguous())
    assert torch.equal(cache.pages.view(torch.uint8), other.pages.view(torch.uint8))
    odd = torch.empty(1 * 1 * 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(1, 1, 4, 64)
    odd.copy_(qkv[:, 19:, :4])
    assert torch.equal(paged_kv8_attention(odd, cache, 0, tab, sl),
                       paged_kv8_attention(odd.clone(), cache, 0, tab, sl))
    pos = torch.arange(20, dtype=torch.int32, device="cuda")[None]
    k, _ = gather_kv8(cache, 0, tab, pos, dtype=torch.float32)
    x = qkv[:, :, 4:6].float()
    assert ((k - x).abs() <= 2.0 ** -4 * x.abs() + cache.scales.max() * 2.0 ** -10).all()  # one e4m3 rounding
    q = qkv[:, 19:, :4].contiguous()
    for bad in (lambda: append_kv8(cache, 0, tab, sl.long(), x, x),
                lambda: append_kv8(cache, 0, tab[:, ::2], sl, x, x),
                lambda: append_kv8(cache, 0, tab, sl, x[:, :, :1], x[:, :, :1]),
                lambda: append_kv8(cache, 0, tab, sl, x.cpu(), x.cpu()),
                lambda: append_kv8(cache, 0, tab, sl, x, x.bfloat16()),
                lambda: append_kv8(KV8CacheState(cache.pages, cache.scales[:, :, :4], 16), 0, tab, sl, x, x),
                lambda: append_kv8(KV8CacheState(cache.pages, cache.scales, 8), 0, tab, sl, x, x),
                lambda: paged_kv8_attention(q[..., :32], cache, 0, tab, sl),
                lambda: paged_kv8_attention(q, cache, 0, tab, sl.cpu()),
                lambda: paged_kv8_attention(q, cache, 0, tab, sl, out=q.float())):
        with pytest.raises(ValueError):
            bad()
    from ssd_b200._lib import SSDError

    with pytest.raises(SSDError):
        append_kv8(cache, 1, tab, sl, x, x)  # no such layer
    with pytest.raises(SSDError):
        paged_kv8_attention(q.half(), cache, 0, tab, sl)
    with pytest.raises(SSDError):
        paged_kv8_attention(q, cache, 0, tab, sl, max_seq_len=1000)  # more than the table holds


@pytest.mark.parametrize("dtype,hq,hkv,d,t", [("bf16", 8, 2, 256, 1), ("bf16", 16, 2, 64, 3), ("bf16", 8, 2, 128, 30),
                                              ("f32", 8, 2, 64, 3)])
@pytest.mark.parametrize("n", [40, 2000])
def test_attention_of_non_finite_queries(cuda, dtype, hq, hkv, d, t, n):
    """An infinity or NaN in a row of q: that row is NaN (it has no finite score, or an infinite one less itself), also
    where every score is minus infinity; the rows beside it do not notice."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    rng = np.random.default_rng(n + d)
    p = Pool(rng, 1, 16, hkv, d, cols=n // 16 + 1)
    k = _round(rng.standard_normal((1, n, hkv, d)), "bf16")
    k[..., 0] = 1.0  # an infinity in dim 0 gives every score its sign
    p.append([n], k, k, [n], "bf16")
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    q = torch.tensor(_round(rng.standard_normal((1, t, hq, d)), dtype)).to(dts[dtype]).cuda()
    want = paged_kv8_attention(q, p.cache, 1, p.dev_tables, i([n]))
    bad = q.clone()
    rows = [(0, 0, 0, float("inf")), (0, 2, 0, float("-inf")), (t - 1, hq - 1, 5, float("nan")),
            (t - 1, hq // 2, d - 1, float("inf"))]
    dead = torch.zeros(want.shape, dtype=torch.bool, device="cuda")
    for tt, h, dim, x in rows:
        bad[0, tt, h, dim] = x
        dead[0, tt, h] = True
    got = paged_kv8_attention(bad, p.cache, 1, p.dev_tables, i([n]))
    assert torch.equal(got.isnan(), dead)
    assert torch.equal(got[~dead], want[~dead])


@pytest.mark.parametrize("dtype,hq,hkv,d,t", [("bf16", 8, 1, 256, 1), ("bf16", 4, 2, 64, 3), ("bf16", 8, 1, 128, 30),
                                              ("f32", 4, 1, 64, 3)])
def test_nan_at_a_position_of_vanishing_weight(cuda, dtype, hq, hkv, d, t):
    """NaN in V reaches every row that sees it, though its weight is e^-1000 and lies in another part of the context."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    rng = np.random.default_rng(2)
    n = 6000
    p = Pool(rng, 1, 16, hkv, d, cols=n // 16)
    k = np.zeros((1, n, hkv, d))
    k[0, 5000, :, 0] = 100.0
    v = _round(rng.standard_normal((1, n, hkv, d)), "bf16")
    v[0, 17, :, 3] = np.nan
    p.append([n], k, v, [n], "bf16")
    q = torch.zeros((1, t, hq, d), dtype=dts[dtype], device="cuda")
    q[..., 0] = 10.0
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    got = paged_kv8_attention(q, p.cache, 1, p.dev_tables, i([n]), scale=1.0)
    nan = got.isnan()
    assert nan[..., 3].all() and int(nan.sum()) == t * hq
    val = torch.tensor(p.vals[1, p.tables[0, 5000 // 16], 5000 % 16]).cuda()
    scale = np.exp2(p.exps[1, p.tables[0, 5000 // 16]].astype(np.float64))
    want = (val * torch.tensor(scale).cuda()[:, None]).repeat_interleave(hq // hkv, 0)
    keep = torch.arange(d, device="cuda") != 3
    assert torch.equal(got[0, :, :, keep].double(), want[None, :, keep].to(dts[dtype]).double().expand(t, -1, -1))


def test_cache_past_32_bit_offsets(cuda):
    """Planes of more than 4 GB: the highest pages hold and give what low pages of a small cache do, bit for bit."""
    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, gather_kv8, paged_kv8_attention, rope_append_kv8
    from ssd_b200.kernels.page_moves import copy_pages

    torch, dts = _torch()
    hkv, d, n, nb = 16, 256, 400, 66_000  # 64 KB a page and plane
    cols = -(-n // 16)
    small = KV8CacheState.allocate(1, cols, 16, hkv, d)
    big = KV8CacheState.allocate(1, nb, 16, hkv, d)
    assert big.pages[0].numel() > 2 ** 32
    lo = torch.arange(cols, dtype=torch.int32, device="cuda").view(1, -1)
    hi = (nb - 1 - lo).contiguous()
    sl = torch.tensor([n], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    k, v = rnd(1, n, hkv, d).bfloat16(), rnd(1, n, hkv, d).bfloat16()
    qkv, cos = rnd(4, 3 * hkv * d).bfloat16(), rnd(512, d // 2)
    at = torch.arange(n, dtype=torch.int32, device="cuda").view(1, -1)
    outs = []
    for c, tab in ((small, lo), (big, hi)):
        append_kv8(c, 0, tab, sl, k, v)
        outs.append([rope_append_kv8(qkv, c, 0, tab, sl, hkv, cos, cos), *gather_kv8(c, 0, tab, at)])
        for t, dt in ((1, "bf16"), (5, "bf16"), (100, "bf16"), (3, "f32")):
            g2 = torch.Generator(device="cuda").manual_seed(t)
            q = torch.randn((1, t, hkv, d), generator=g2, device="cuda").to(dts[dt])
            outs[-1].append(paged_kv8_attention(q, c, 0, tab, sl, max_seq_len=n))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    ids = hi[0, :5]
    copy_pages(big, ids, torch.arange(5, dtype=torch.int32, device="cuda") + 65_700)
    copy_pages(big, ids, torch.arange(5, dtype=torch.int32, device="cuda"))
    for first in (0, 65_700):
        assert torch.equal(big.pages[:, 0, first:first + 5].view(torch.uint8), small.pages[:, 0, :5].view(torch.uint8))
        assert torch.equal(big.scales[:, 0, first:first + 5], small.scales[:, 0, :5])


@pytest.mark.parametrize("case", [
    ("bf16", 4, 1, 64, 16, 9, [9 + 17 * i % 700 for i in range(70)]),       # three registers of lengths
    ("bf16", 8, 1, 64, 16, 12, [0, 12, 4000] + [15 + i for i in range(17)]),  # one sequence takes most of the splits
    ("bf16", 4, 2, 128, 16, 40, [0, 40, 1000, 41, 333]),
    ("bf16", 8, 1, 128, 4, 20, [20, 900, 0]),                               # pages smaller than a tile
    ("bf16", 2, 2, 256, 16, 33, [33, 700]),
], ids=lambda c: f"{len(c[6])}x{c[5]}-{c[3]}")
def test_many_rows_over_ragged_batches(cuda, case):
    """Splits that go by the sequences' own lengths: empty, short and long ones beside each other; a bound that is
    far above every length gives the same, and so does a second run."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    dtype, hq, hkv, d, bs, t, lens = case
    p, q, ql = _attention_inputs(case, seed=len(lens) + t)
    ql = np.minimum(ql, lens)
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    args = (torch.tensor(q).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, i(lens))
    got = paged_kv8_attention(*args, q_lens=i(ql))
    assert torch.equal(got, paged_kv8_attention(*args, q_lens=i(ql)))
    ref, mass, size = o.attention(q, p.vals, p.exps, p.tables, lens, ql, 1 / math.sqrt(d))
    tol = _tolerance(case, q, p, lens, mass, size, ref)
    err = np.abs(got.float().cpu().numpy() - ref)
    assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()
    for r in range(len(lens)):
        assert (got[r, ql[r]:] == 0).all()
    wide = torch.cat([p.dev_tables, torch.full_like(p.dev_tables, -1)], 1)
    far = paged_kv8_attention(*args[:3], wide, args[4], q_lens=i(ql)).float().cpu().numpy()
    assert (np.abs(far - ref) <= tol).all()


@pytest.mark.parametrize("case", [
    ("bf16", 8, 2, 64, 48, 3, [3, 700, 1300]),     # pages of three groups of 16
    ("bf16", 8, 2, 64, 48, 30, [30, 700, 1300]),
    ("bf16", 4, 1, 128, 512, 2, [2, 513, 1500]),   # pages longer than a tile, and than a split
    ("bf16", 4, 1, 128, 512, 40, [40, 513, 1500]),
    ("f32", 4, 1, 64, 512, 3, [3, 513, 700]),
], ids=lambda c: f"{c[0]}-{c[4]}-{c[5]}")
def test_page_sizes_beside_the_tiles(cuda, case):
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    dtype, hq, hkv, d, bs, t, lens = case
    p, q, ql = _attention_inputs(case, seed=bs + t)
    p.check()
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    got = paged_kv8_attention(torch.tensor(q).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, i(lens), q_lens=i(ql))
    ref, mass, size = o.attention(q, p.vals, p.exps, p.tables, lens, ql, 1 / math.sqrt(d))
    err, tol = np.abs(got.float().cpu().numpy() - ref), _tolerance(case, q, p, lens, mass, size, ref)
    assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("hq,hkv,d,t", [(8, 1, 256, 3), (8, 1, 256, 40), (4, 2, 64, 3), (4, 2, 64, 40)])
def test_small_weights_on_large_values(cuda, hq, hkv, d, t):
    """The position that takes nearly all of the softmax holds V values far below its page's scale, so that positions
    of weight 2^-20 count as much: their weights must not be rounded to a few bits.

    Scores are exact products (one dimension), so ds is the exponential's own: at most 4 roundings of arguments below
    32, and 2^-22, ds <= 2^-16.  Weights: 2^-11 relative, and 2^-32 of the largest below 2^-21 of it.  n sums in fp32."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, _ = _torch()
    rng = np.random.default_rng(d + t)
    n = 64 + t
    p = Pool(rng, 1, 16, hkv, d, cols=-(-n // 16))
    k = np.zeros((1, n, hkv, d))
    k[..., 0] = np.exp2(rng.integers(-6, -2, (1, n, hkv)))  # scores 16 * that, small
    k[0, 5, :, 0] = 1.0
    v = rng.uniform(-448, 448, (1, n, hkv, d))
    v[0, ::16, :, 0] = 448                                  # every page's scale is 1
    v[0, 5] = rng.integers(-7, 8, (hkv, d)) * 2.0 ** -9
    p.append([n], k, v, [n], "bf16")
    q = np.zeros((1, t, hq, d))
    q[..., 0] = 16.0
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    got = paged_kv8_attention(torch.tensor(q).bfloat16().cuda(), p.cache, 1, p.dev_tables, i([n]), scale=1.0)
    ref, mass, _ = o.attention(q, p.vals, p.exps, p.tables, [n], [t], 1.0)
    tol = EPS["bf16"] * np.abs(ref) + (2.0 ** -11 + 4 * 2.0 ** -16 + n * 2.0 ** -24) * mass + n * 2.0 ** -32 * 448
    err = np.abs(got.float().cpu().numpy() - ref)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype,hq,hkv,d,bs,t", [("bf16", 8, 1, 256, 16, 3), ("bf16", 8, 1, 256, 16, 40),
                                                 ("bf16", 4, 2, 64, 4, 40), ("f32", 4, 2, 64, 16, 3)])
@pytest.mark.parametrize("qmag", [0.0, 2.0 ** -100, 2.0 ** -30, 1.0])
def test_zero_keys_and_small_queries(cuda, dtype, hq, hkv, d, bs, t, qmag):
    """Pages whose K is zero carry the smallest scale; with it, rows of q of any size, zero included, weigh every
    position they see alike."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    rng = np.random.default_rng(t)
    n = 130 + t  # ends inside a page and a tile
    p = Pool(rng, 1, bs, hkv, d, cols=-(-n // bs))
    v = _round(rng.standard_normal((1, n, hkv, d)), "bf16")
    p.append([n], np.zeros((1, n, hkv, d)), v, [n], "bf16")
    q = _round(qmag * rng.standard_normal((1, t, hq, d)), dtype)
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    got = paged_kv8_attention(torch.tensor(q).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, i([n]))
    ref, mass, _ = o.attention(q, p.vals, p.exps, p.tables, [n], [t], 1 / math.sqrt(d))
    # equal weights: exact but for V's page exponents, 2^-11; n sums in fp32, the output's rounding
    tol = EPS[dtype] * np.abs(ref) + (2.0 ** -11 + 2 * n * 2.0 ** -24) * mass
    assert (np.abs(got.float().cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("hq,hkv,d,t", [(4, 2, 64, 3), (4, 2, 64, 40), (8, 1, 256, 2), (8, 1, 256, 12)])
def test_small_elements_beside_a_large_one_in_q(cuda, hq, hkv, d, t):
    """One element of q lies 2^18 above the others, on a dimension where K is zero: the others decide, with all of
    their bits."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, _ = _torch()
    rng = np.random.default_rng(d * t)
    n = 100 + t
    p = Pool(rng, 1, 16, hkv, d, cols=-(-n // 16))
    k, v = 16 * rng.standard_normal((1, n, hkv, d)), rng.standard_normal((1, n, hkv, d))
    k[..., 0] = 0
    p.append([n], k, v, [n], "bf16")
    q = 2.0 ** -5 * rng.standard_normal((1, t, hq, d))
    q[..., 0] = 8192
    q = _round(q, "bf16")
    i = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    scale = 8 / d ** 0.5
    got = paged_kv8_attention(torch.tensor(q).bfloat16().cuda(), p.cache, 1, p.dev_tables, i([n]), scale=scale)
    ref, mass, size = o.attention(q, p.vals, p.exps, p.tables, [n], [t], scale)
    # scores: products exact in f16, d sums in fp32, the exponential; weights' 2^-11 and n sums; the output's half step
    ds = ((d + 8) * 2.0 ** -24 + 2.0 ** -22) * size + 2.0 ** -21
    tol = EPS["bf16"] * np.abs(ref) + (4 * ds + 2.0 ** -11 + n * 2.0 ** -24) * mass
    err = np.abs(got.float().cpu().numpy() - ref)
    assert (err <= tol).all(), (err / tol).max()
