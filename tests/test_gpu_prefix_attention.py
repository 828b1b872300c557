"""GPU: attention over shared prefixes against 64 bits, at bounds derived from the kernels' arithmetic."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.beams import prefix_attention

pytestmark = pytest.mark.gpu


def case(seed, sizes, prefixes, tails, T, hq, hkv, D, bs, dtype="bf16", q_lens=None, extra_cols=0, layers=1, layer=0):
    """Rows of forked tables: whole prefix pages shared, a partial one copied."""
    import torch

    from ssd_b200.kernels.kv_cache import KVCacheState

    rng = np.random.default_rng(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    B = sum(sizes)
    group = [i for i, n in enumerate(sizes) for _ in range(n)]
    lens = [prefixes[group[b]] + tails[b] for b in range(B)]
    cols = max(1, max(-(-n // bs) for n in lens)) + extra_cols
    nb = sum(p // bs for p in prefixes) + sum(-(-n // bs) for n in lens) + 2
    perm = rng.permutation(nb).astype(np.int32)
    pages = torch.from_numpy(rng.standard_normal((2, layers, nb, bs, hkv, D)).astype(np.float32)).to("cuda", dt)
    tables = np.full((B, cols), -1, np.int32)
    at = row = 0
    starts = [0]
    for n, P in zip(sizes, prefixes):
        full, part = P // bs, P % bs
        shared = perm[at:at + full]
        at += full
        for i in range(n):
            rest = max(0, -(-lens[row] // bs) - full)
            tables[row, :full] = shared
            tables[row, full:full + rest] = perm[at:at + rest]
            if part and i and rest:
                pages[:, :, tables[row, full], :part] = pages[:, :, tables[row - i, full], :part]
            at += rest
            row += 1
        starts.append(row)
    q = torch.from_numpy(rng.standard_normal((B, T, hq, D)).astype(np.float32)).to("cuda", dt)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ql = None if q_lens is None else i32(q_lens)
    return dict(q=q, cache=KVCacheState(pages=pages, block_size=bs), layer=layer, block_tables=i32(tables),
                seq_lens=i32(lens), group_starts=i32(starts), prefix_lens=i32(prefixes), q_lens=ql)


def oracle(c, scale=None):
    host = lambda t: t.float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()  # noqa: E731
    q = host(c["q"])
    return prefix_attention(q, host(c["cache"].pages[:, c["layer"]]), host(c["block_tables"]), host(c["seq_lens"]),
                            None if c["q_lens"] is None else host(c["q_lens"]), host(c["group_starts"]),
                            host(c["prefix_lens"]), q.shape[-1] ** -0.5 if scale is None else scale)


def bound(c, want, size, slack):
    """fp32 scores: D products summed, off by (D + 2) 2^-24 of sum |q k|, twice (the score and its maximum); weights:
    2^-21 of the exponentials and their arguments' rounding (up to 2^-23 of a score of `slack`); sums of up to n
    terms in fp32, at most 2^-24 n each of the weights' and the products' (n: the longest context); bf16 weights: 2^-8.
    The output: half a step of its type."""
    D = c["q"].shape[-1]
    n = int(c["seq_lens"].max())
    bf = c["q"].element_size() == 2
    rel = (2 * (D + 2) * 2.0 ** -24 + 2.0 ** -22) * slack + 2.0 ** -21 + 2 * n * 2.0 ** -24 + (2.0 ** -8 if bf else 0)
    return size * rel[..., None] + np.abs(want) * (2.0 ** -8 if bf else 2.0 ** -24) + 1e-30


def check(c, **kw):
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    got = shared_prefix_attention(**c, **kw)
    torch.cuda.synchronize()
    got = got.double().cpu().numpy()
    want, size, slack = oracle(c, kw.get("scale"))
    lim = bound(c, want, size, slack)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    bad = np.abs(np.where(nan, 0, got - want)) > lim
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want).max())
    return got


SHAPES = [  # sizes, prefixes, tails, T, hq, hkv, D
    ([4], [137], [3, 9, 1, 5], 1, 8, 1, 256),
    ([1], [0], [1], 1, 8, 1, 256),                         # one token, nothing shared
    ([3, 1, 2], [64, 0, 33], [1, 17, 2, 40, 5, 6], 1, 16, 16, 256),
    ([2, 4], [300, 511], [7, 8, 70, 9, 300, 12], 7, 4, 4, 128),
    ([15], [200], list(range(2, 17)), 2, 8, 2, 64),
    ([2], [1000], [40, 64], 40, 8, 1, 256),                # more query rows a sequence than a row tile holds
    ([40], [100], [1 + i % 23 for i in range(40)], 1, 1, 1, 64),
    ([33, 5], [16, 48], [4 + 3 * (i % 5) for i in range(38)], 4, 8, 1, 128),
    ([1] * 9, [0, 1, 15, 16, 17, 31, 32, 100, 5], [1, 2, 3, 4, 5, 6, 7, 8, 9], 1, 4, 2, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bs", [16, 32, 4])
@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
def test_matches_64_bits(cuda, shape, bs, dtype):
    sizes, prefixes, tails, T, hq, hkv, D = shape
    check(case(1, sizes, prefixes, tails, T, hq, hkv, D, bs, dtype))


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("bf16", 3), ("f32", 16)])
def test_long_contexts_in_several_parts(cuda, dtype, bs):
    check(case(2, [3, 2], [2500, 901], [5, 700, 90, 1, 333], 2, 4, 1, 128, bs, dtype))
    check(case(3, [3], [4100], [3, 50, 9], 1, 2, 2, 256, bs, dtype))


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("bf16", 4), ("f32", 16)])
def test_ragged_new_tokens_and_empty_rows(cuda, dtype, bs):
    """q_lens of 0 to T; rows past q_lens are zeros, also in an output that held something else."""
    import torch

    c = case(4, [3, 2], [40, 7], [6, 4, 9, 4, 5], 4, 8, 2, 64, bs, dtype, q_lens=[4, 0, 1, 3, 2])
    out = torch.full_like(c["q"], float("nan"))
    got = check(c, out=out)
    for b, n in enumerate([4, 0, 1, 3, 2]):
        assert (got[b, n:] == 0).all()


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("bf16", 4), ("f32", 16)])
def test_rows_inside_the_prefix(cuda, dtype, bs):
    """A row sees the positions up to its own, also where the prefix goes on (and where its length is 0)."""
    import torch

    c = case(5, [3], [50], [4, 4, 4], 4, 4, 1, 64, bs, dtype)
    c["seq_lens"] = torch.tensor([20, 54, 3], dtype=torch.int32, device="cuda")  # row 2: tokens before position 0
    check(c)
    c["seq_lens"] = torch.tensor([0, 54, 50], dtype=torch.int32, device="cuda")
    check(c)


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("bf16", 4), ("f32", 16)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_does_not_reach_it(cuda, dtype, bs, value):
    """Infinities and NaN behind a row's end, in other rows' tails and in pages of no row."""
    import torch

    c = case(6, [3, 2], [37, 20], [5, 12, 3, 8, 2], 2, 4, 2, 64, bs, dtype)
    pages = c["cache"].pages
    for b, n in enumerate(c["seq_lens"].tolist()):
        blk, at = c["block_tables"][b, (n - 1) // bs], (n - 1) % bs
        pages[:, :, blk, at + 1:] = value
    used = torch.unique(c["block_tables"][c["block_tables"] >= 0]).long()
    free = torch.ones(pages.shape[2], dtype=torch.bool, device="cuda")
    free[used] = False
    pages[:, :, free] = value
    check(c)
    # row 1's own tail: its last token's row reaches that token alone
    n = int(c["seq_lens"][1])
    pages[:, :, c["block_tables"][1, (n - 1) // bs], (n - 1) % bs] = value
    check(c)


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("bf16", 4), ("f32", 16)])
def test_missing_pages_hold_nothing(cuda, dtype, bs):
    c = case(7, [2, 1], [64, 40], [9, 20, 3], 1, 4, 1, 64, bs, dtype)
    c["block_tables"][0, 1] = -1                       # in the prefix, read through the group's first row
    c["block_tables"][1, -(-84 // bs) - 1] = 1 << 20   # row 1's last page
    c["block_tables"][2, :] = -1                       # a row without any page
    got = check(c)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("f32", 16)])
def test_extreme_scores(cuda, dtype, bs):
    """Scores far apart: weights underflow, sums do not overflow; negative and zero scales."""
    c = case(8, [4], [300], [5, 70, 9, 2], 1, 4, 1, 64, bs, dtype)
    check(c, scale=-0.3)
    check(c, scale=0.0)
    c["q"].mul_(30)
    check(c)


def test_layers_strides_and_table_columns(cuda):
    import torch

    c = case(9, [2], [40], [5, 6], 1, 4, 1, 64, 16, layers=3, layer=2, extra_cols=5)
    check(c, max_seq_len=46)
    wide = torch.zeros((2, 1, 4, 130), dtype=torch.bfloat16, device="cuda")
    wide[..., 3:67] = c["q"]
    ref = check(c)
    c["q"] = wide[..., 3:67]
    assert np.array_equal(check(c), ref)


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("bf16", 4), ("f32", 16)])
def test_equals_attention_by_rows(cuda, dtype, bs):
    """Within the sum of both kernels' bounds of the attention that reads every row's pages by themselves."""
    from ssd_b200.kernels.kv_cache import paged_verify_attention

    c = case(10, [5, 3], [250, 77], [9, 3, 30, 2, 8, 4, 4, 19], 2, 8, 2, 128, bs, dtype)
    got = check(c)
    rows = paged_verify_attention(c["q"], c["cache"], 0, c["block_tables"], c["seq_lens"]).double().cpu().numpy()
    assert (np.abs(got - rows) <= 2 * bound(c, *oracle(c))).all()


def test_graphs_and_streams(cuda):
    """Two captured calls side by side, replayed after the lengths have changed, and a call on another stream."""
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c1 = case(11, [4], [600], [8, 8, 8, 8], 1, 8, 1, 256, 16)
    c2 = case(12, [2, 3], [50, 300], [4, 5, 6, 7, 8], 2, 8, 8, 64, 16)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        a = shared_prefix_attention(**c1)
    with torch.cuda.stream(s2):
        b = shared_prefix_attention(**c2)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = shared_prefix_attention(**c1)
    with torch.cuda.graph(g2):
        o2 = shared_prefix_attention(**c2)
    for _ in range(3):
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, a) and torch.equal(o2, b)
    c1["seq_lens"] -= 3
    g1.replay()
    torch.cuda.synchronize()
    assert torch.equal(o1, shared_prefix_attention(**c1))


WIDE = [  # more than a row tile, or than the tensor-core kernel's plan, holds; heads that fill no tile
    (([300], [70], [1 + i % 9 for i in range(300)], 1, 8, 1, 64), 16),
    (([1] * 270, [i % 40 for i in range(270)], [2] * 270, 2, 4, 2, 64), 16),
    (([256], [33], [1 + i % 5 for i in range(256)], 1, 4, 4, 64), 16),
    (([5, 2], [90, 17], [3, 4, 30, 6, 7, 3, 50], 3, 6, 2, 128), 48),
    (([3], [200], [13, 40, 90], 13, 20, 2, 256), 32),
    (([2], [100], [300, 310], 300, 8, 1, 64), 16),
    (([3, 2], [40, 20], [1, 2, 3, 4, 5], 1, 256, 1, 64), 16),
    (([2, 3], [2000, 40], [1, 900, 3, 1500, 8], 1, 130, 1, 128), 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,bs", WIDE, ids=range(len(WIDE)))
def test_wide_batches_and_odd_heads(cuda, shape, bs, dtype):
    check(case(41, *shape, bs, dtype))


@pytest.mark.parametrize("dtype,bs", [("bf16", 16), ("bf16", 4), ("f32", 16)])
def test_lengths_past_their_bounds_count_as_the_bounds(cuda, dtype, bs):
    """q_lens above T are T; positions from max_seq_len on are not read, whatever lengths and prefixes say."""
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c = case(42, [3, 1], [64, 40], [9, 8, 20, 5], 2, 8, 2, 64, bs, dtype)
    want = shared_prefix_attention(**c)
    assert torch.equal(shared_prefix_attention(**{**c, "q_lens": torch.full_like(c["seq_lens"], 9)}), want)
    short = shared_prefix_attention(**c, max_seq_len=48).double().cpu().numpy()
    keys = {**c, "block_tables": c["block_tables"].clone()}
    keys["block_tables"][:, 48 // bs:] = -1  # the same positions missing
    w, size, slack = oracle(keys)
    assert (np.abs(short - w) <= bound(keys, w, size, slack)).all()


@pytest.mark.parametrize("hq,hkv,d,prefix", [(8, 1, 256, 40), (8, 1, 256, 3000), (16, 4, 64, 700), (4, 2, 128, 1500)])
def test_a_wait_that_runs_out_is_reported(cuda, hq, hkv, d, prefix):
    """No polls allowed: every CTA gives up at its first wait.  Rows are NaN (those past q_lens zeros), the status says so
    once, and the next call is right."""
    from ssd_b200._lib import SSDError, lib
    from ssd_b200.kernels.prefix_attention import check_shared_prefix_attention, shared_prefix_attention

    c = case(43, [3, 2], [prefix, 20], [9, 8, 20, 30, 6], 2, hq, hkv, d, 16, q_lens=[2, 1, 2, 2, 0])
    check_shared_prefix_attention()
    assert lib().ssd_shared_prefix_attention_set_polls(-2) == 1
    try:
        assert lib().ssd_shared_prefix_attention_set_polls(0) == 0
        got = shared_prefix_attention(**c).float().cpu().numpy()
    finally:
        assert lib().ssd_shared_prefix_attention_set_polls(-1) == 0
    with pytest.raises(SSDError, match="timed out"):
        check_shared_prefix_attention()
    check_shared_prefix_attention("cuda")
    for b, n in enumerate([2, 1, 2, 2, 0]):
        assert np.isnan(got[b, :n]).all() and (got[b, n:] == 0).all()
    check(c)
    check_shared_prefix_attention()


@pytest.mark.parametrize("shape", [SHAPES[3], SHAPES[4], SHAPES[7], ([2, 1], [3000, 1000], [70, 8, 5], 2, 8, 2, 256)],
                         ids=range(4))
def test_repeats_are_equal_to_the_bit(cuda, shape):
    """Sums are taken in one order: threads that came in another would show in a few of many calls."""
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c = case(44, *shape, 16)
    want = shared_prefix_attention(**c)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(2500):
        differ += (shared_prefix_attention(**c) != want).any()
    assert int(differ) == 0


def test_nothing_to_do(cuda):
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c = case(13, [2], [20], [3, 4], 1, 4, 1, 64, 16)
    assert shared_prefix_attention(**{**c, "q": c["q"][:, :0]}).shape == (2, 0, 4, 64)
    empty = {k: (v[:0] if k in ("q", "block_tables", "seq_lens") else v) for k, v in c.items()}
    empty["group_starts"], empty["prefix_lens"] = torch.zeros(1, dtype=torch.int32, device="cuda"), c["prefix_lens"][:0]
    assert shared_prefix_attention(**empty).shape == (0, 1, 4, 64)


def test_refusals(cuda):
    import torch

    from ssd_b200._lib import SSDError
    from ssd_b200.kernels.kv_cache import KVCacheState
    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c = case(14, [2], [20], [3, 4], 1, 4, 1, 64, 16)
    bad = [("q", c["q"].float()), ("q", c["q"][0]), ("q", c["q"].cpu()), ("q", c["q"][..., :32]),
           ("seq_lens", c["seq_lens"].long()), ("seq_lens", c["seq_lens"][:1]), ("seq_lens", c["seq_lens"].cpu()),
           ("group_starts", c["group_starts"][:1]), ("prefix_lens", c["prefix_lens"].float()),
           ("prefix_lens", c["prefix_lens"][0]), ("block_tables", c["block_tables"][0]),
           ("cache", KVCacheState(pages=c["cache"].pages[0], block_size=16))]
    for k, v in bad:
        with pytest.raises((ValueError, SSDError)):
            shared_prefix_attention(**{**c, k: v})
    for kw in (dict(max_seq_len=1 << 20), dict(out=c["q"].float()), dict(out=c["q"][:1])):
        with pytest.raises((ValueError, SSDError)):
            shared_prefix_attention(**c, **kw)
    with pytest.raises(SSDError):
        shared_prefix_attention(**{**c, "layer": 1})
    odd = case(15, [2], [20], [3, 4], 1, 4, 1, 64, 16)
    odd["cache"] = KVCacheState(pages=torch.zeros((2, 1, 8, 16, 1, 96), dtype=torch.bfloat16, device="cuda"), block_size=16)
    odd["q"] = torch.zeros((2, 1, 4, 96), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(SSDError):
        shared_prefix_attention(**odd)
