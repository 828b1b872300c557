"""GPU: page copies and pool compaction against a plain restatement (exact: bytes and whole numbers)."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _cache(kind, nl, nb, bs, hkv, d, seed):
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.kernels.kv_cache import KVCacheState

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if kind == "kv8":
        c = KV8CacheState.allocate(nl, nb, bs, hkv, d)
        c.pages.view(torch.uint8).random_(0, 256, generator=g)
        c.scales.uniform_(generator=g)
    else:
        c = KVCacheState.allocate(nl, nb, bs, hkv, d, dtype=torch.bfloat16 if kind == "bf16" else torch.float32)
        c.pages.normal_(generator=g)
    return c


def _bytes(c):
    import torch

    return [c.pages.view(torch.uint8).clone()] + ([c.scales.clone()] if hasattr(c, "scales") else [])


@pytest.mark.parametrize("kind", ["bf16", "f32", "kv8"])
@pytest.mark.parametrize("nl,nb,bs,hkv,d,n", [(1, 8, 16, 1, 64, 1), (3, 50, 16, 2, 256, 20), (2, 40, 1, 1, 64, 13),
                                              (2, 9, 3, 5, 128, 4), (1, 6, 64, 16, 256, 3)])
def test_copy_pages(cuda, kind, nl, nb, bs, hkv, d, n):
    import torch

    from ssd_b200.kernels.page_moves import copy_pages

    c = _cache(kind, nl, nb, bs, hkv, d, n)
    rng = np.random.default_rng(n)
    ids = torch.tensor(rng.permutation(nb).astype(np.int32), device="cuda")
    src, dst = ids[:n].clone(), ids[n:2 * n].clone()
    if n > 2:
        src[1], dst[2] = -1, nb  # skipped pairs
    want = _bytes(c)
    for w in want:
        for s, t in zip(src.tolist(), dst.tolist()):
            if 0 <= s < nb and 0 <= t < nb:
                w[:, :, t] = w[:, :, s]
    copy_pages(c, src, dst)
    assert all(torch.equal(a, w) for a, w in zip(_bytes(c), want))
    copy_pages(c, src[:0], dst[:0])  # nothing to copy
    assert all(torch.equal(a, w) for a, w in zip(_bytes(c), want))


def test_copy_one_page_to_many_and_into_another_cache(cuda):
    import torch

    from ssd_b200.kernels.page_moves import copy_pages

    for kind in ("bf16", "kv8"):
        a, b = _cache(kind, 2, 20, 16, 2, 64, 1), _cache(kind, 2, 33, 16, 2, 64, 2)
        ids = torch.tensor([[4, 9], [7, 3], [-1, 2]], dtype=torch.int32, device="cuda")
        want = _bytes(a)
        for w in want:
            w[:, :, 9], w[:, :, 3], w[:, :, 2] = w[:, :, 4], w[:, :, 4], w[:, :, 4]
        copy_pages(a, ids[0, 0:1].expand(3), ids[:, 1])  # an expanded source, a strided destination
        assert all(torch.equal(x, w) for x, w in zip(_bytes(a), want))
        src = torch.arange(20, dtype=torch.int32, device="cuda")
        assert copy_pages(a, src, src + 13, dst_cache=b) is b
        for x, y in zip(_bytes(a), _bytes(b)):
            assert torch.equal(y[:, :, 13:], x)
        with pytest.raises(ValueError):
            copy_pages(a, src, src, dst_cache=_cache(kind, 1, 33, 16, 2, 64, 2))
        with pytest.raises(ValueError):
            copy_pages(a, src, src.long())
        with pytest.raises(ValueError):
            copy_pages(a, src, src[:3])


def _plain_compact(nb, free, ref, tables, lens):
    isfree = np.zeros(nb, bool)
    isfree[free] = True
    u = int((~isfree).sum())
    src = [i for i in range(u, nb) if not isfree[i]]
    dst = [i for i in range(u) if isfree[i]]
    remap = np.where(isfree, -1, np.arange(nb))
    remap[src] = dst
    nref = ref.copy()
    nref[dst], nref[src] = ref[src], 0
    out = np.full_like(tables, -1)
    for b, n in enumerate(lens):
        for i in range(n):
            if 0 <= tables[b, i] < nb:
                out[b, i] = remap[tables[b, i]]
    fl = np.full(nb, -1)
    fl[:nb - u] = np.arange(nb - 1, u - 1, -1)
    return u, src, dst, remap, nref, out, fl


@pytest.mark.parametrize("kind", ["bf16", "kv8"])
@pytest.mark.parametrize("nb,used", [(1, 0), (1, 1), (2, 1), (40, 17), (40, 0), (40, 40), (1500, 700), (5000, 2600)])
@pytest.mark.parametrize("inplace", [False, True])
def test_compact_pages(cuda, kind, nb, used, inplace):
    import torch

    from ssd_b200.kernels.page_moves import compact_pages

    rng = np.random.default_rng(nb + used)
    c = _cache(kind, 2, nb, 2, 1, 64, nb)
    perm = rng.permutation(nb)
    rows, cols = 5, used // 5 + 3
    tables, lens = np.full((rows, cols), 12345, np.int32), np.zeros(rows, np.int32)  # dead entries: garbage
    for j, blk in enumerate(perm[:used]):
        tables[j % rows, lens[j % rows]] = blk
        lens[j % rows] += 1
    ref = np.zeros(nb, np.int32)
    ref[perm[:used]] = rng.integers(0, 3, used)  # a block in use may have no count
    free = np.full(nb, -1, np.int32)
    free[:nb - used] = perm[used:]
    u, src, dst, remap, nref, ntab, fl = _plain_compact(nb, perm[used:], ref, tables, lens)
    t = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    args = [t(tables), t(lens), t(ref), t(free), t([nb - used])]
    kept = [a.clone() for a in args]
    want = _bytes(c)
    for w in want:
        w[:, :, dst] = w[:, :, src]
    r = compact_pages(c, *args, inplace=inplace)
    assert all(torch.equal(a, w) for a, w in zip(_bytes(c), want))
    assert r.remap.tolist() == remap.tolist() and r.ref_counts.tolist() == nref.tolist()
    assert r.tables.tolist() == ntab.tolist()
    assert r.free_list.tolist() == fl.tolist() and r.free_top.tolist() == [nb - u]
    if inplace:
        assert r.tables is args[0] and r.free_top is args[4]
    else:
        assert all(torch.equal(a, k) for a, k in zip(args, kept))


@pytest.mark.parametrize("nb,rows,cols", [(50_000, 64, 600), (200_000, 3, 20_000)])
def test_compact_large_pools(cuda, nb, rows, cols):
    """Pools whose flags take more than the default shared memory, or more than there is; tables that get a launch of
    their own, the draft's among them."""
    import torch

    from ssd_b200.kernels.page_moves import compact_pages

    rng = np.random.default_rng(nb)
    c = _cache("kv8", 1, nb, 1, 1, 64, 3)
    perm = rng.permutation(nb)
    used = nb // 2 + 17
    tables = rng.permutation(perm[:used])[rng.integers(0, used, (rows, cols))].astype(np.int32)
    draft = perm[rng.integers(0, used, (2, cols))].astype(np.int32)
    lens, dlens = rng.integers(0, cols + 1, rows).astype(np.int32), np.array([cols, 5], np.int32)
    ref = rng.integers(0, 4, nb).astype(np.int32)
    free = np.full(nb, -1, np.int32)
    free[:nb - used] = perm[used:]
    ref[perm[used:]] = 0
    u, src, dst, remap, nref, ntab, fl = _plain_compact(nb, perm[used:], ref, tables, lens)
    dtab = np.where(np.arange(cols)[None] < dlens[:, None], remap[draft], -1)
    t = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    want = _bytes(c)
    for w in want:
        w[:, :, dst] = w[:, :, src]
    r = compact_pages(c, t(tables), t(lens), t(ref), t(free), t([nb - used]), t(draft), t(dlens))
    assert all(torch.equal(a, w) for a, w in zip(_bytes(c), want))
    for got, exp in ((r.remap, remap), (r.ref_counts, nref), (r.tables, ntab), (r.draft_tables, dtab),
                     (r.free_list, fl), (r.free_top, np.array([nb - u]))):
        np.testing.assert_array_equal(got.cpu().numpy(), exp)


def test_compact_refuses_one_table_for_both(cuda):
    import torch

    from ssd_b200.kernels.page_moves import compact_pages

    c = _cache("bf16", 1, 8, 16, 1, 64, 1)
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    tab, lens = z(2, 4), z(2)
    with pytest.raises(ValueError):
        compact_pages(c, tab, lens, z(8), z(8), z(1), tab, lens, inplace=True)


def test_moves_in_a_graph_and_on_another_stream(cuda):
    """A captured copy and compaction, replayed on fresh contents; the same on a side stream."""
    import torch

    from ssd_b200.kernels.page_moves import compact_pages, copy_pages

    nb, rows, cols = 60, 3, 12
    t = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731

    def state(seed):
        r = np.random.default_rng(seed)
        perm = r.permutation(nb)
        tables, lens = np.full((rows, cols), -1, np.int32), np.full(rows, 8, np.int32)
        tables[:, :8] = perm[:24].reshape(rows, 8)
        ref = np.zeros(nb, np.int32)
        ref[perm[:24]] = 1
        free = np.full(nb, -1, np.int32)
        free[:nb - 24] = perm[24:]
        return perm, tables, lens, ref, free

    c = _cache("kv8", 2, nb, 16, 2, 64, 5)
    fill = [_cache("kv8", 2, nb, 16, 2, 64, 6 + i) for i in range(2)]
    src, dst = t([3, 5, 3]), t([10, 11, -1])
    args = [t(x) for x in state(0)[1:]] + [t([nb - 24])]
    compact_pages(c, *args)  # loads the kernels
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_pages(c, src, dst)
        r = compact_pages(c, *args)
    side = torch.cuda.Stream()
    for seed in (1, 2):
        perm, *new = state(seed)
        for a, x in zip(args, new):
            a.copy_(t(x))
        for x, y in ((c.pages.view(torch.uint8), fill[seed - 1].pages.view(torch.uint8)), (c.scales, fill[seed - 1].scales)):
            x.copy_(y)
        want = _bytes(c)
        u, s, d, remap, nref, ntab, fl = _plain_compact(nb, perm[24:], new[2], new[0], new[1])
        for w in want:
            w[:, :, 10], w[:, :, 11] = w[:, :, 3].clone(), w[:, :, 5].clone()
            w[:, :, d] = w[:, :, s]
        torch.cuda.synchronize()
        if seed == 1:
            graph.replay()
        else:
            with torch.cuda.stream(side):
                copy_pages(c, src, dst)
                r = compact_pages(c, *args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(_bytes(c), want))
        assert r.tables.tolist() == ntab.tolist() and r.free_list.tolist() == fl.tolist()
        assert r.remap.tolist() == remap.tolist() and r.ref_counts.tolist() == nref.tolist()
