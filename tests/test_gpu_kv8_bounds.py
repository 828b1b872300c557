"""GPU: attention over the 8-bit cache against 64 bits, at the bounds that its arithmetic states."""

from __future__ import annotations

import math

import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import CASES, Pool, _attention_inputs, _round, _torch

pytestmark = pytest.mark.gpu


def _i(a):
    import torch

    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def _run(p, q, lens, ql, dtype="bf16", **kw):
    """(output on the host, its tensor) for the numpy queries."""
    from ssd_b200.kernels.kv8_cache import paged_kv8_attention

    torch, dts = _torch()
    out = paged_kv8_attention(torch.tensor(q).to(dts[dtype]).cuda(), p.cache, 1, p.dev_tables, _i(lens), q_lens=_i(ql),
                              **kw)
    return out.float().cpu().numpy(), out


def _near(got, r, p, dtype="bf16"):
    tol = ref.bound(r, p.exps, dtype)
    off = np.abs(got - r["out"])
    assert (off <= tol).all(), f"{np.nanmax(off / np.maximum(tol, 1e-300)):.3g} times the bound, {np.isnan(off).sum()} NaN"


@pytest.mark.parametrize("hq,hkv,d,t", [(8, 1, 256, 40), (4, 4, 128, 40), (16, 4, 64, 33), (8, 2, 128, 5), (4, 1, 256, 1)])
@pytest.mark.parametrize("kind", ["zeros, large", "large, zeros", "one large page", "tiny, large", "large, tiny"])
@pytest.mark.parametrize("big", [18, 24, 30, 100])
def test_v_scales_far_apart_within_a_tile(cuda, hq, hkv, d, t, kind, big):
    """Runs of 32 positions whose V is all zero, or tiny, beside runs of |V| near 2^big: every position counts in
    the normaliser, at 512 positions (one split) and at 1100."""
    rng = np.random.default_rng(big)
    lens = [512, 1100, 470]
    ql = [t, t, max(t - 1, 1)]
    p = Pool(rng, 3, 16, hkv, d, cols=70)
    k = _round(rng.standard_normal((3, 1100, hkv, d)), "bf16")
    v = rng.standard_normal((3, 1100, hkv, d))
    run = np.arange(1100) // 32 % 2
    first, second = {"zeros, large": (0, 2.0 ** big), "large, zeros": (2.0 ** big, 0), "tiny, large": (2.0 ** -90, 2.0 ** big),
                     "large, tiny": (2.0 ** big, 2.0 ** -90), "one large page": (0, 0)}[kind]
    v *= np.where(run == 0, first, second)[None, :, None, None]
    if kind == "one large page":
        v[:, 208:224] = 2.0 ** big * rng.standard_normal((3, 16, hkv, d))
    p.append(lens, k, _round(v, "bf16"), lens, "bf16")
    q = _round(rng.standard_normal((3, t, hq, d)), "bf16")
    scale = 1 / math.sqrt(d)
    r = ref.attention(q, p.vals, p.exps, p.tables, lens, ql, scale)
    _near(_run(p, q, lens, ql)[0], r, p)
    few = dict(lens=[512, 500, 470], cols=32)  # a bound of 512: one split
    p.dev_tables = p.dev_tables[:, :few["cols"]].contiguous()
    r = ref.attention(q, p.vals, p.exps, p.tables, few["lens"], ql, scale)
    _near(_run(p, q, few["lens"], ql)[0], r, p)


@pytest.mark.parametrize("hq,hkv,d,lens", [(8, 1, 256, [500, 300]), (8, 1, 256, [3000, 100]), (16, 4, 64, [512, 12]),
                                           (4, 2, 128, [1500, 700])])
def test_a_wait_that_runs_out_is_reported(cuda, hq, hkv, d, lens):
    """No polls allowed: every CTA gives up at its first wait.  Rows are NaN (those past q_lens zeros), the status says so
    once, and the next call is right."""
    from ssd_b200._lib import SSDError, lib
    from ssd_b200.kernels.kv8_cache import check_kv8_attention

    rng = np.random.default_rng(1)
    t, ql = 40, [40, 33]
    lens = [max(n, t) for n in lens]
    p = Pool(rng, 2, 16, hkv, d, cols=-(-max(lens) // 16))
    k = _round(rng.standard_normal((2, max(lens), hkv, d)), "bf16")
    p.append(lens, k, k, lens, "bf16")
    q = _round(rng.standard_normal((2, t, hq, d)), "bf16")
    check_kv8_attention()
    assert lib().ssd_kv8_attention_set_polls(-2) == 1
    try:
        assert lib().ssd_kv8_attention_set_polls(0) == 0
        got = _run(p, q, lens, ql)[0]
    finally:
        assert lib().ssd_kv8_attention_set_polls(-1) == 0
    with pytest.raises(SSDError, match="timed out"):
        check_kv8_attention()
    check_kv8_attention("cuda")
    for b in range(2):
        assert np.isnan(got[b, :ql[b]]).all() and (got[b, ql[b]:] == 0).all()
    r = ref.attention(q, p.vals, p.exps, p.tables, lens, ql, 1 / math.sqrt(d))
    _near(_run(p, q, lens, ql)[0], r, p)
    check_kv8_attention()


@pytest.mark.parametrize("dtype,hq,hkv,d,bs,t", [("bf16", 8, 1, 64, 16, 2), ("bf16", 8, 1, 64, 16, 40), ("bf16", 4, 2, 128, 4, 3),
                                                 ("bf16", 8, 2, 128, 4, 33), ("f32", 4, 1, 64, 16, 5)])
def test_scales_count_by_their_exponent_everywhere(cuda, dtype, hq, hkv, d, bs, t):
    """A stored scale that append would not have written -- zero, subnormal, negative, no power of two -- is the power of
    two at its exponent, 2^-118 at least, for every kernel that reads it; a scale of zero is no missing page."""
    from ssd_b200.kernels.kv8_cache import gather_kv8

    torch, _ = _torch()
    rng = np.random.default_rng(31)
    lens, ql = [200, 90], [t, t - 1]
    p = Pool(rng, 2, bs, hkv, d, cols=-(-200 // bs))
    k = _round(rng.standard_normal((2, 200, hkv, d)), "bf16")
    p.append(lens, k, _round(rng.standard_normal((2, 200, hkv, d)), "bf16"), lens, "bf16")
    for col, (stored, e) in enumerate([(0.0, -118), (1e-42, -118), (-2.0 ** -8, -8), (3 * 2.0 ** -8, -7)]):
        for plane in range(2):
            blk = p.tables[0, 2 * col + plane]
            p.cache.scales[plane, 1, blk] = stored
            p.exps[plane, blk] = e
    q = _round(rng.standard_normal((2, t, hq, d)), dtype)
    r = ref.attention(q, p.vals, p.exps, p.tables, lens, ql, 1 / math.sqrt(d))
    _near(_run(p, q, lens, ql, dtype)[0], r, p, dtype)
    pos = np.arange(200)
    gk, gv = gather_kv8(p.cache, 1, p.dev_tables[:1].contiguous(), _i(pos[None]), dtype=torch.float32)
    rk, rv = ref.o.rows_of(p.vals, p.exps, p.tables[0], pos)
    np.testing.assert_array_equal(gk[0].cpu().numpy(), rk)
    np.testing.assert_array_equal(gv[0].cpu().numpy(), rv)


@pytest.mark.parametrize("dtype,t,bs", [("bf16", 2, 16), ("bf16", 40, 16), ("bf16", 40, 4), ("f32", 5, 16)])
def test_infinite_queries_that_see_nothing(cuda, dtype, t, bs):
    """A row of q with an infinity is NaN where it sees a position, zeros where every page it could see is missing."""
    rng = np.random.default_rng(17)
    lens = [300, 300, 90]
    p = Pool(rng, 3, bs, 1, 64, cols=-(-300 // bs))
    k = _round(rng.standard_normal((3, 300, 1, 64)), "bf16")
    p.append(lens, k, k, lens, "bf16")
    p.tables[0] = -1
    p.tables[2, 1:] = 10 ** 6  # one page left
    import torch

    p.dev_tables = torch.tensor(p.tables, device="cuda")
    q = _round(rng.standard_normal((3, t, 8, 64)), dtype)
    q[:, 0, 3, 5] = np.inf
    q[:, t - 1, 4] = -np.inf
    got = _run(p, q, lens, [t] * 3, dtype)[0]
    assert (got[0] == 0).all()
    for b in (1, 2):
        assert np.isnan(got[b, 0, 3]).all() and np.isnan(got[b, t - 1, 4]).all()
    finite = np.isfinite(q).all(-1)
    q[~finite] = 0
    r = ref.attention(q, p.vals, p.exps, p.tables, lens, [t] * 3, 1 / 8)
    off, tol = np.abs(got - r["out"])[finite], ref.bound(r, p.exps, dtype)[finite]
    assert (off <= tol).all()


def test_long_prompts_allocate_their_output_alone(cuda):
    """600 rows of 16 heads against 8192 positions: unsplit, so a call's memory is its output."""
    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, paged_kv8_attention

    torch, _ = _torch()
    t, cols = 600, 512
    cache = KV8CacheState.allocate(1, cols, 16, 16, 64)
    table = torch.arange(cols, dtype=torch.int32, device="cuda")[None]
    q = torch.randn((1, t, 16, 64), device="cuda").bfloat16()
    append_kv8(cache, 0, table, _i([t]), q, q)
    paged_kv8_attention(q, cache, 0, table, _i([t]))
    n = _i([t])
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    paged_kv8_attention(q, cache, 0, table, n)
    assert torch.cuda.max_memory_allocated() - before <= q.numel() * 2 + (1 << 21)  # one block of the allocator beside it


def _sparse(seed, b, nb, cols, bs, hkv, d):
    """A pool as ``Pool`` has it, from ``ref.sparse_pool``; sequences share pages (they are only read)."""
    from types import SimpleNamespace

    from ssd_b200.kernels.kv8_cache import KV8CacheState

    torch, _ = _torch()
    rng = np.random.default_rng(seed)
    vals, exps = ref.sparse_pool(rng, nb, bs, hkv, d)
    cache = KV8CacheState.allocate(2, nb, bs, hkv, d)
    cache.pages.view(torch.uint8)[:, 0].fill_(0x7F)
    cache.pages.view(torch.uint8)[:, 1] = torch.tensor(ref.e4m3_bytes(vals)).cuda()
    cache.scales[:, 1] = torch.tensor(np.exp2(exps.astype(np.float32))).cuda()
    tables = np.stack([rng.permutation(nb)[np.arange(cols) % nb] for _ in range(b)]).astype(np.int32)
    return SimpleNamespace(cache=cache, vals=vals, exps=exps, tables=tables, dev_tables=torch.tensor(tables).cuda()), rng


LONG = [  # dtype, hq, hkv, d, bs, t, longest, sequences: split of the bound at 666 CTAs
    ("bf16", 16, 16, 64, 16, 1, 4096, 8),     # 832
    ("bf16", 16, 16, 64, 16, 5, 4096, 8),
    ("bf16", 16, 16, 64, 4, 5, 4096, 8),      # 832, a row and scales a position
    ("bf16", 16, 16, 128, 16, 5, 2500, 8),    # 512
    ("bf16", 8, 8, 256, 16, 3, 3000, 6),      # 256
    ("bf16", 4, 4, 256, 16, 2, 3333, 20),     # 448
    ("bf16", 8, 1, 64, 16, 8, 4096, 170),     # 1024, 64 rows a KV head
    ("bf16", 8, 1, 64, 1, 2, 4000, 170),
    ("bf16", 16, 2, 128, 24, 7, 4000, 90),    # 1024, pages of 24
    ("bf16", 8, 1, 256, 16, 64, 8192, 4),     # prompt chunks: by the lengths
    ("bf16", 8, 1, 128, 4, 33, 5000, 3),
    ("bf16", 16, 4, 64, 16, 200, 6000, 2),
    ("f32", 4, 1, 64, 16, 5, 3000, 5),
    ("f32", 2, 2, 256, 4, 3, 1500, 3),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(map(str, c)))
def test_long_contexts_at_their_bounds(cuda, case):
    """Contexts of many splits, of every length the rule gives; a position lost or counted twice would show.  A few
    heads and sequences are compared, the longest and the shortest among them."""
    dtype, hq, hkv, d, bs, t, top, b = case
    p, rng = _sparse(b * t, b, -(-top // bs), -(-top // bs), bs, hkv, d)
    lens = rng.integers(t, top + 1, b)
    lens[0], lens[1], lens[b - 1] = top, t, top - 1
    ql = np.where(np.arange(b) % 4 == 2, max(t - 1, 1), t)
    q = _round(0.25 * rng.standard_normal((b, t, hq, d)), dtype)  # weights alike: each position counts
    got, _ = _run(p, q, lens, ql, dtype)
    some = sorted({0, 1, min(2, b - 1), b - 1})
    heads = sorted({0, hq // 2, hq - 1})
    r = ref.attention(q[some], p.vals, p.exps, p.tables[some], lens[some], ql[some], 1 / math.sqrt(d), heads=heads)
    tol = ref.bound(r, p.exps, dtype)
    off = np.abs(got[some] - r["out"])[:, :, heads]
    assert (off <= tol[:, :, heads]).all(), (off / np.maximum(tol[:, :, heads], 1e-300)).max()
    assert all((got[i, ql[i]:] == 0).all() for i in range(b))


@pytest.mark.parametrize("hq,hkv,d,bs,t,top,b", [(16, 16, 64, 16, 5, 4096, 8), (16, 16, 64, 4, 5, 4096, 8),
                                                 (8, 1, 256, 16, 8, 8192, 3), (8, 1, 64, 16, 8, 4096, 170),
                                                 (16, 4, 128, 16, 6, 3000, 16)])
def test_bits_do_not_depend_on_the_tokens_beside(cuda, hq, hkv, d, bs, t, top, b):
    """At a given batch and bound, a verify step gives each token the bits that decoding it alone does, whatever the split
    (832, 832, 256, 1024 and 320 positions here)."""
    torch, _ = _torch()
    p, rng = _sparse(t, b, -(-top // bs), -(-top // bs), bs, hkv, d)
    lens = rng.integers(t, top + 1, b)
    lens[0], lens[1] = top, t
    q = _round(rng.standard_normal((b, t, hq, d)), "bf16")
    _, full = _run(p, q, lens, [t] * b)
    for j in range(t):
        _, one = _run(p, q[:, j:j + 1], lens - t + j + 1, [1] * b)
        assert torch.equal(one[:, 0], full[:, j]), j


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
def test_attention_at_its_bounds(cuda, case):
    """The shapes of the oracle's test, at the bounds of the present arithmetic."""
    dtype, hq, hkv, d, bs, t, lens = case
    p, q, ql = _attention_inputs(case, seed=hq * d + t + bs)
    r = ref.attention(q, p.vals, p.exps, p.tables, lens, ql, 1 / math.sqrt(d))
    _near(_run(p, q, lens, ql, dtype)[0], r, p, dtype)


@pytest.mark.parametrize("b,t", [(0, 3), (0, 0), (2, 0)])
def test_calls_on_nothing(cuda, b, t):
    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, gather_kv8, paged_kv8_attention, rope_append_kv8

    torch, _ = _torch()
    cache = KV8CacheState.allocate(1, 4, 16, 2, 64)
    table, lens = torch.zeros((b, 3), dtype=torch.int32, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda")
    x = torch.zeros((b, t, 2, 64), device="cuda").bfloat16()
    before = cache.pages.view(torch.uint8).clone()
    append_kv8(cache, 0, table, lens, x, x)
    cos = torch.ones((8, 32), device="cuda")
    qkv = torch.zeros((b * t, 8 * 64), device="cuda").bfloat16()
    # tokens a sequence are told from the rows: none without sequences
    assert rope_append_kv8(qkv, cache, 0, table, lens, 4, cos, cos).shape == (b, t if b else 0, 4, 64)
    at = torch.zeros((b, t), dtype=torch.int32, device="cuda")
    assert gather_kv8(cache, 0, table, at)[0].shape == (b, t, 2, 64)
    q = torch.zeros((b, t, 4, 64), device="cuda").bfloat16()
    assert paged_kv8_attention(q, cache, 0, table, lens).shape == q.shape
    assert torch.equal(cache.pages.view(torch.uint8), before)


@pytest.mark.parametrize("dtype,bs,hkv,d", [("bf16", 16, 2, 64), ("f32", 16, 1, 256), ("bf16", 7, 2, 128)])
@pytest.mark.parametrize("outlier", [2.0 ** 6, 2.0 ** 12, 2.0 ** 30])
def test_rows_beside_a_rejected_one(cuda, dtype, bs, hkv, d, outlier):
    """A draft row far larger than the others is appended, rejected (the length goes back) and other rows follow.  The
    page keeps the scale that it needed until its first row is appended again: its rows, earlier and later, are off by
    their own rounding, 2^-4 of a value at most, and by less than 2^-9 2^e in all (each growth to an exponent e_i
    rounds at most half a step 2^-10 2^e_i more, the e_i rise to e).  The pages beside it are not touched."""
    from ssd_b200.kernels.kv8_cache import gather_kv8

    torch, _ = _torch()
    rng = np.random.default_rng(41)
    p = Pool(rng, 2, bs, hkv, d, cols=-(-48 // bs))
    x = _round(rng.standard_normal((2, 48, hkv, d)), dtype)
    n = 2 * bs + 3  # the accepted length, inside the third page
    p.append([n, n], x[:, :n], x[:, :n], [n, n], dtype)
    top = np.abs(x).max()
    for step in (1.0, 4.0, outlier):  # the scale grows more than once
        draft = x[:, n:n + 2].copy()
        draft[:, 1] = _round(step * draft[:, 1], dtype)
        top = max(top, np.abs(draft).max())
        p.append([n + 2, n + 2], draft, draft, [2, 2], dtype)
        p.check()
    p.append([n + 4, n + 4], x[:, n:n + 4], x[:, n:n + 4], [4, 4], dtype)  # rejected: other rows in its place
    p.check()
    e = np.ceil(np.log2(top / 448))
    pos = np.arange(n + 4)
    got = gather_kv8(p.cache, 1, p.dev_tables, _i(np.tile(pos, (2, 1))), dtype=torch.float32)
    hurt = pos // bs == n // bs
    for g in got:
        off = np.abs(g.double().cpu().numpy() - x[:, pos])
        assert (off <= 2.0 ** -4 * np.abs(x[:, pos]) + 2.0 ** -9 * 2.0 ** e).all()
        own = np.ceil(np.log2(np.abs(x).max() / 448))
        assert (off <= 2.0 ** -4 * np.abs(x[:, pos]) + 2.0 ** -9 * 2.0 ** own)[:, ~hurt].all()
    q = _round(rng.standard_normal((2, 3, 2 * hkv, d)), dtype)
    r = ref.attention(q, p.vals, p.exps, p.tables, [n + 4] * 2, [3, 3], 1 / math.sqrt(d))
    _near(_run(p, q, [n + 4] * 2, [3, 3], dtype)[0], r, p, dtype)


@pytest.mark.parametrize("hq,hkv,d,bs,t", [(8, 1, 256, 16, 3), (16, 4, 64, 16, 40), (4, 2, 128, 4, 2), (4, 2, 128, 4, 40)])
@pytest.mark.parametrize("lens", [[450, 300], [2500, 1100]])
def test_v_near_the_smallest_scale(cuda, hq, hkv, d, bs, t, lens):
    """V of 2^-112 to 2^-100, page by page, under scores that spread over tens of powers of two: outputs are that small, and
    right (bf16 and fp32 hold numbers down to 2^-126)."""
    rng = np.random.default_rng(77)
    p = Pool(rng, 2, bs, hkv, d, cols=-(-max(lens) // bs))
    n = max(lens)
    mag = np.exp2(-rng.integers(100, 113, (2, -(-n // 16), hkv)).astype(float)).repeat(16, 1)[:, :n, :, None]
    k = _round(rng.standard_normal((2, n, hkv, d)), "bf16")
    p.append(lens, k, _round(mag * rng.standard_normal((2, n, hkv, d)), "bf16"), lens, "bf16")
    q = _round(4 * rng.standard_normal((2, t, hq, d)), "bf16")
    r = ref.attention(q, p.vals, p.exps, p.tables, lens, [t] * 2, 1 / math.sqrt(d))
    _near(_run(p, q, lens, [t] * 2)[0], r, p)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,bs,t,lens", [(16, 16, 256, 16, 256, [256, 300]), (8, 1, 256, 16, 200, [1999]),
                                                (6, 2, 64, 7, 33, [33, 40, 90]), (4, 4, 128, 100, 130, [131, 700]),
                                                (3, 1, 64, 1, 5, [5, 4, 0, 77])])
def test_rope_append_is_rotation_then_append(cuda, dtype, hq, hkv, d, bs, t, lens):
    """Byte for byte what append_kv8 makes of the rotated rows in fp32 (products and sums rounded one by one), a whole
    forward's rows among them; q is that rotation, rounded once."""
    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, rope_append_kv8

    torch, dts = _torch()
    g = torch.Generator(device="cuda").manual_seed(t + d)
    b, cols = len(lens), -(-max(lens) // bs)
    ql = [t if i % 2 == 0 else max(t - 3, 0) for i in range(b)]
    perm = torch.randperm(b * cols, generator=g, device="cuda")
    table = perm.to(torch.int32).view(b, cols)
    caches = [KV8CacheState.allocate(1, b * cols, bs, hkv, d) for _ in range(2)]
    old = torch.randn((b, max(lens), hkv, d), generator=g, device="cuda") * 0.3
    before = [max(n - m, 0) for n, m in zip(lens, ql)]
    for c in caches:
        append_kv8(c, 0, table, _i(before), old, old, q_lens=_i(before))
    qkv = torch.randn((b * t, (hq + 2 * hkv) * d), generator=g, device="cuda").to(dts[dtype])
    ang = torch.arange(max(lens) + 1, device="cuda")[:, None] * torch.exp(-torch.arange(d // 2, device="cuda") / 9)[None]
    cos, sin = ang.cos(), ang.sin()
    q = rope_append_kv8(qkv, caches[0], 0, table, _i(lens), hq, cos, sin, q_lens=_i(ql))
    x = qkv.float().view(b, t, hq + 2 * hkv, d)
    pos = (torch.tensor(lens, device="cuda") - torch.tensor(ql, device="cuda"))[:, None] + torch.arange(t, device="cuda")
    real = (torch.arange(t, device="cuda")[None] < torch.tensor(ql, device="cuda")[:, None]) & (pos >= 0)
    cc, ss = (a[pos.clamp(0, max(lens))][:, :, None] for a in (cos, sin))
    lo, hi = x[:, :, :hq + hkv, :d // 2], x[:, :, :hq + hkv, d // 2:]
    y = torch.cat([lo * cc - hi * ss, hi * cc + lo * ss], -1)
    append_kv8(caches[1], 0, table, _i(lens), y[:, :, hq:], x[:, :, hq + hkv:], q_lens=_i(ql))
    assert torch.equal(caches[0].pages.view(torch.uint8), caches[1].pages.view(torch.uint8))
    assert torch.equal(caches[0].scales, caches[1].scales)
    assert torch.equal(q, (y[:, :, :hq] * real[:, :, None, None]).to(dts[dtype]))
