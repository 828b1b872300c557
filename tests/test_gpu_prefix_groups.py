"""GPU: the groups of the shared-prefix attention where they do not cover the batch in order."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_prefix_attention import case, check

pytestmark = pytest.mark.gpu

KINDS = [("bf16", 16), ("bf16", 4), ("f32", 16)]


def poison():
    """What a later allocation finds in its memory: large numbers, as addresses and as sums."""
    import torch

    for n in (1 << 16, 1 << 20, 1 << 24):
        torch.full((n,), 0x70707070, dtype=torch.int32, device="cuda")


PARTIAL = [  # sizes, prefixes, tails, T, hq, hkv, D
    ([3, 2, 2], [20, 40, 7], [6, 4, 9, 4, 5, 8, 3], 2, 8, 2, 64),                      # lists that are not cut
    ([3, 2, 2], [300, 2500, 90], [5, 700, 90, 300, 33, 8, 9], 2, 4, 2, 128),           # joined parts
    ([2, 1, 2], [100, 1000, 30], [50, 60, 70, 41, 45], 40, 8, 1, 256),                 # several tiles a sequence
    ([5, 32, 2], [64, 1500, 9], [3 + i % 40 for i in range(39)], 4, 16, 2, 64),        # two tiles a group: a team
]


@pytest.mark.parametrize("dtype,bs", KINDS)
@pytest.mark.parametrize("shape", PARTIAL, ids=range(len(PARTIAL)))
def test_rows_of_no_group_are_zeros(cuda, shape, dtype, bs):
    """Groups that begin above row 0 and end below the last one, and that hold no rows at all."""
    import torch

    c = case(21, *shape, bs, dtype)
    sizes = shape[0]
    starts = c["group_starts"]
    out = torch.full_like(c["q"], float("nan"))
    for lo, hi in ((1, 2), (1, 3), (0, 2)):
        part = {**c, "group_starts": starts[lo:hi + 1].contiguous(), "prefix_lens": c["prefix_lens"][lo:hi].contiguous()}
        poison()
        got = check(part, out=out.fill_(float("nan")))
        first, end = sum(sizes[:lo]), sum(sizes[:hi])
        assert (got[:first] == 0).all() and (got[end:] == 0).all()
    none = {**c, "group_starts": torch.tensor([2, 2, 2], dtype=torch.int32, device="cuda"), "prefix_lens": c["prefix_lens"][:2]}
    poison()
    assert (check(none, out=out.fill_(float("nan"))) == 0).all()


def test_rows_of_no_group_in_a_replayed_graph(cuda):
    """The groups shrink between replays of one captured call."""
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c = case(22, *PARTIAL[1], 16)
    g = torch.cuda.CUDAGraph()
    shared_prefix_attention(**c)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        o = shared_prefix_attention(**c)
    c["group_starts"].copy_(torch.tensor([3, 5, 5, 5], dtype=torch.int32))
    c["prefix_lens"].copy_(torch.tensor([2500, 0, 0], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(o.double().cpu().numpy(), check(c))
    assert (o[:3] == 0).all() and (o[5:] == 0).all()


@pytest.mark.parametrize("dtype,bs", KINDS)
@pytest.mark.parametrize("starts", [[0, 5, 3, 7], [4, 0, 2, 7], [0, 3, 7, 5], [7, 3, 1, 0], [-4, 2, 1, 90], [0, 2, -1, 7]])
@pytest.mark.parametrize("shape", PARTIAL[:3], ids=range(3))
def test_starts_that_descend_count_as_the_largest_before(cuda, shape, starts, dtype, bs):
    """No row is in two groups, whatever the starts say: the same bits as with ascending ones."""
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c = case(23, *shape, bs, dtype)
    B = c["q"].shape[0]
    c["prefix_lens"][:] = torch.tensor([3, 0, 5], dtype=torch.int32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    upright = np.maximum.accumulate(np.clip(starts, 0, B)).tolist()
    poison()
    got = shared_prefix_attention(**{**c, "group_starts": i32(starts)})
    assert torch.equal(got, shared_prefix_attention(**{**c, "group_starts": i32(upright)}))
    check({**c, "group_starts": i32(upright)})


def test_many_starts_that_descend(cuda):
    """More groups than a warp takes at once, with steps back inside and between its batches."""
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    rng = np.random.default_rng(24)
    for dtype, bs in KINDS:
        c = case(25, [1] * 90, [0] * 90, [1 + i % 50 for i in range(90)], 1, 4, 2, 64, bs, dtype)
        for _ in range(4):
            starts = np.sort(rng.integers(0, 91, 91))
            starts[rng.integers(0, 91, 12)] = rng.integers(-5, 99, 12)
            upright = np.maximum.accumulate(np.clip(starts, 0, 90))
            i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
            got = shared_prefix_attention(**{**c, "group_starts": i32(starts)})
            assert torch.equal(got, shared_prefix_attention(**{**c, "group_starts": i32(upright)}))
            check({**c, "group_starts": i32(upright)})


@pytest.mark.parametrize("dtype,bs", KINDS)
@pytest.mark.parametrize("prefix", [0, 37, 1200])
def test_scores_of_minus_infinity_weigh_nothing(cuda, prefix, dtype, bs):
    """Some of a row's scores -inf: the others make the row.  All of them: zeros, as where nothing is seen."""
    import torch

    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    c = case(26, [2, 1], [prefix, 20], [9, 300, 5], 1, 4, 2, 64, bs, dtype)
    c["q"][..., 0] = 1.0
    keys = c["cache"].pages[0]
    for j in range(prefix, prefix + 9, 2):       # every second one of row 0's tail
        keys[:, c["block_tables"][0, j // bs].long(), j % bs, :, 0] = float("-inf")
    keys[:, c["block_tables"][2, :-(-25 // bs)].long(), :, :, 0] = float("-inf")  # all that row 2 sees
    got = shared_prefix_attention(**c)
    assert (got[2] == 0).all()
    check({**c, "group_starts": c["group_starts"][:2].contiguous(), "prefix_lens": c["prefix_lens"][:1]})
