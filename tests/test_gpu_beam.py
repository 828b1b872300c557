"""GPU: beam search's selection and the re-ordering of paged rows against 64 bits and whole numbers."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import beams

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ selection
def select(logits, scores, lengths=None, finished=None, eos=None, alpha=0.0):
    """The call's outputs, checked against the oracle: whole numbers equal, scores within rounding.

    A score is base + (x - lse) rounded once to fp32 (2^-24 of it); lse: the exponentials' error (2^-21, and the
    rounding of arguments up to 2^-23 of the spread) and sums of 32 terms in a thread and ten levels above (42 2^-24)."""
    import torch

    from ssd_b200.algorithm.beam import beam_select

    r = beam_select(logits, scores, lengths, finished, eos_token_id=eos, length_penalty=alpha)
    torch.cuda.synchronize()
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    x = host(logits)
    want = beams.beam_select(x, host(scores), host(lengths), host(finished), -1 if eos is None else eos, alpha)
    got = [host(t) for t in (r.scores, r.parents, r.tokens, r.lengths, r.finished)]
    for a, b in zip(got[1:], want[1:]):
        assert np.array_equal(a, b), (a, b)
    fin = x[np.isfinite(x)]
    spread = float(fin.max() - fin.min()) if fin.size else 0.0
    lim = 2.0 ** -24 * np.abs(np.where(np.isfinite(want[0]), want[0], 0)) + 2.0 ** -21 + spread * 2.0 ** -23 + 42 * 2.0 ** -24
    inf = np.isinf(want[0])
    assert np.array_equal(got[0][inf], want[0][inf])
    assert (np.abs(np.where(inf, 0, got[0] - np.where(inf, 0, want[0]))) <= lim).all()
    return r


def inputs(seed, G, W, V, std=3.0):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    logits = std * torch.randn((G, W, V), generator=g, device="cuda")
    scores = -10 * torch.rand((G, W), generator=g, device="cuda")
    lengths = torch.randint(1, 40, (G, W), generator=g, device="cuda", dtype=torch.int32)
    finished = (torch.rand((G, W), generator=g, device="cuda") < 0.3).to(torch.uint8)
    return logits, scores, lengths, finished


@pytest.mark.parametrize("G,W,V", [(1, 1, 1), (1, 4, 3), (2, 3, 1021), (3, 2, 8192), (1, 4, 8193), (5, 8, 16384),
                                   (2, 5, 33333), (1, 32, 40), (2, 32, 5000), (1, 4, 256000), (7, 16, 20001),
                                   (300, 1, 64), (37, 8, 32768)])
def test_select_matches(cuda, G, W, V):
    x, s, n, f = inputs(G * 1000 + W, G, W, V)
    select(x, s)
    select(x, s, n, None, None, 0.6)
    select(x, s, n, f, V // 2, 0.0)
    select(x, s, n, f.bool(), V - 1, 1.7)
    select(x, s, n, f, 0, -0.5)


@pytest.mark.parametrize("G,W,V", [(1, 2, 3000001), (2, 31, 70000), (60, 17, 9000)])
def test_select_large(cuda, G, W, V):
    x, s, n, f = inputs(G * 1000 + W, G, W, V)
    select(x, s, n, f, V // 2, 0.7)


def test_select_first_step_and_dead_beams(cuda):
    x, s, n, f = inputs(1, 3, 6, 5000)
    s[:] = float("-inf")
    s[:, 0] = 0
    select(x, s)
    s[1] = float("-inf")                   # a request without a live beam
    s[2, 3] = -2.0
    f[:] = 0
    f[2, 0] = 1                            # and one beam that has finished
    select(x, s, n, f, 7, 1.0)


def test_select_masks(cuda):
    """Masked tokens are never taken; beams whose mask leaves fewer tokens than places, one, or none."""
    x, s, n, f = inputs(2, 4, 4, 3001)
    x[0, :, 5:] = float("-inf")
    x[1] = float("-inf")
    x[1, 2, 77] = -1e30
    x[2, :, :] = float("-inf")
    x[3, 1] = float("nan")
    x[3, 2, 100] = float("inf")
    x[3, 0, 3] = float("nan")
    select(x, s)
    x[3, 3] = -3.4028234663852886e38     # masks of the type's lowest value: a uniform beam
    select(x, s)
    select(x, s, n, f, 3, 0.6)


@pytest.mark.parametrize("V", [37, 5000, 40000])
def test_select_ties(cuda, V):
    """Equal logits over whole beams, equal beams, zeros of both signs: the lowest beam and token first."""
    import torch

    x = torch.zeros((2, 4, V), device="cuda")
    x[:, :, 1::3] = -0.0
    s = torch.zeros((2, 4), device="cuda")
    select(x, s)
    x[1] = x[1] + torch.arange(V, device="cuda") // 700
    select(x, s)
    n = torch.full((2, 4), 5, dtype=torch.int32, device="cuda")
    f = torch.tensor([[0, 1, 1, 0], [1, 1, 1, 1]], dtype=torch.uint8, device="cuda")
    select(x, s, n, f, 0, 1.0)


@pytest.mark.parametrize("order", ["up", "down"])
def test_select_sorted_rows(cuda, order):
    import torch

    v = torch.arange(50001, device="cuda", dtype=torch.float32) * 1e-3
    x = (v if order == "up" else v.flip(0)).expand(2, 8, -1).contiguous()
    select(x, -torch.arange(16, device="cuda", dtype=torch.float32).view(2, 8))


def test_select_strides(cuda):
    """Rows at a stride, rows that start off 16 bytes, and rows that have to be copied first."""
    import torch

    x, s, n, f = inputs(3, 2, 3, 2003)
    wide = torch.full((2, 3, 2048), float("nan"), device="cuda")
    wide[:, :, 1:2004] = x
    a = select(x, s)
    b = select(wide[:, :, 1:2004], s)
    c = select(x.permute(2, 0, 1).contiguous().permute(1, 2, 0), s)
    for r in (b, c):
        assert torch.equal(a.scores, r.scores) and torch.equal(a.tokens, r.tokens)


def test_select_graph_and_streams(cuda):
    import torch

    from ssd_b200.algorithm.beam import beam_select

    x, s, n, f = inputs(4, 4, 4, 30000)
    y, t, _, _ = inputs(5, 1, 4, 256000)
    a, b = beam_select(x, s), beam_select(y, t)
    graphs = []
    for args in ((x, s), (y, t)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = beam_select(*args)
        graphs.append((g, r, torch.cuda.Stream()))
    for _ in range(3):
        for g, _, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (_, r, _), want in zip(graphs, (a, b)):
            assert torch.equal(r.scores, want.scores) and torch.equal(r.tokens, want.tokens)


def test_select_refusals(cuda):
    import torch

    from ssd_b200._lib import SSDError
    from ssd_b200.algorithm.beam import beam_select

    x, s, n, f = inputs(6, 2, 3, 50)
    ok = dict(logits=x, scores=s, lengths=n, finished=f, eos_token_id=1)
    beam_select(**ok)
    for k, v in [("logits", x.double()), ("logits", x[0]), ("logits", x.cpu()), ("scores", s.double()),
                 ("scores", s[:1]), ("scores", s.cpu()), ("lengths", n.long()), ("lengths", n[:, :2]),
                 ("finished", f.int()), ("finished", f[:1]), ("eos_token_id", None), ("eos_token_id", 50),
                 ("eos_token_id", -1)]:
        with pytest.raises((ValueError, SSDError)):
            beam_select(**{**ok, k: v})
    with pytest.raises(ValueError):
        beam_select(x, s, length_penalty=1.0)
    with pytest.raises(SSDError):
        beam_select(x, s, n, length_penalty=float("nan"))
    with pytest.raises(ValueError):
        beam_select(torch.zeros((1, 33, 50), device="cuda"), torch.zeros((1, 33), device="cuda"))
    assert beam_select(x[:0], s[:0]).tokens.shape == (0, 3)


# ------------------------------------------------------------------------------------------------ re-ordering
def pool(seed, G, W, bs, lo, hi, nb_free, kind="bf16", layers=2, hkv=2, D=64, held=None):
    """Requests of W rows that share their prompt's whole pages; (cache, PageManager, tokens held by each row)."""
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.kernels.kv_cache import KVCacheState
    from ssd_b200.runtime.page_manager import PageManager

    rng = np.random.default_rng(seed)
    n = [int(rng.integers(lo, hi + 1)) for _ in range(G)] if held is None else held
    prompt = [int(rng.integers(0, x + 1)) for x in n]
    rows, need = [], 0
    for x, p in zip(n, prompt):
        full, all_ = p // bs, -(-x // bs)
        shared = list(range(need, need + full))
        need += full
        for _ in range(W):
            rows.append(shared + list(range(need, need + all_ - full)))
            need += all_ - full
    nb = need + nb_free
    perm = rng.permutation(nb)
    rows = [[int(perm[b]) for b in r] for r in rows]
    free = [int(b) for b in perm[need:]]
    cols = max(1, max(len(r) for r in rows)) + 2
    pm = PageManager(bs, nb, max_seqs=G * W, max_blocks_per_seq=cols)
    refs = np.zeros(nb, np.int32)
    for i, r in enumerate(rows):
        if r:
            pm.tables[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        pm.lens[i] = len(r)
        for b in r:
            refs[b] += 1
    pm.ref_counts_dev.copy_(torch.from_numpy(refs))
    pm.free_list.fill_(-1)
    if free:
        pm.free_list[:len(free)] = torch.tensor(free, dtype=torch.int32)
    pm.free_top[0] = len(free)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if kind == "kv8":
        c = KV8CacheState.allocate(layers, nb, bs, hkv, D)
        c.pages.view(torch.uint8).random_(0, 256, generator=g)
        c.scales.uniform_(generator=g)
    else:
        c = KVCacheState.allocate(layers, nb, bs, hkv, D, dtype=torch.bfloat16 if kind == "bf16" else torch.float32)
        c.pages.normal_(generator=g)
    return c, pm, [x for x in n for _ in range(W)]


def state(pm):
    import torch

    torch.cuda.synchronize()
    lens = pm.lens.tolist()
    t = pm.tables.cpu().numpy()
    for i, n in enumerate(lens):
        assert (t[i, n:] == -1).all()
    return [t[i, :n].tolist() for i, n in enumerate(lens)], lens, pm.ref_counts, pm.free_blocks


def reorder(c, pm, held, parents):
    import torch

    from ssd_b200.kernels.page_moves import reorder_pages

    tables, lens, refs, free = state(pm)
    parents = np.asarray(parents, np.int32)
    want, w_refs, w_free, w_ok, copies = beams.reorder(tables, lens, refs, free, parents, held, pm.block_size)
    caches = c if isinstance(c, list) else [c]
    raw = [x.pages.view(torch.uint8).clone() for x in caches]
    for r in raw:
        for _, s, d, n in copies:
            r[:, :, d, :n] = r[:, :, s, :n]
    scales = [x.scales.clone() if hasattr(x, "scales") else None for x in caches]
    for sc in scales:
        if sc is not None:
            for _, s, d, _ in copies:
                sc[:, :, d] = sc[:, :, s]
    ok = reorder_pages(c, pm.tables, pm.lens, pm.ref_counts_dev, pm.free_list, pm.free_top,
                       torch.from_numpy(parents).cuda(), torch.tensor(held, dtype=torch.int32, device="cuda"))
    got = state(pm)
    assert got[0] == want and got[2] == w_refs and got[3] == w_free and ok.tolist() == w_ok
    assert (pm.free_list[len(w_free):] == -1).all()
    for x, r, sc in zip(caches, raw, scales):
        assert torch.equal(x.pages.view(torch.uint8), r)
        assert sc is None or torch.equal(x.scales, sc)
    W = parents.shape[1]
    return [held[b // W * W + p] if 0 <= p < W else 0 for b, p in enumerate(parents.flat)]


@pytest.mark.parametrize("kind", ["bf16", "f32", "kv8"])
@pytest.mark.parametrize("G,W,bs,lo,hi", [(1, 4, 16, 45, 45), (1, 1, 16, 20, 20), (5, 3, 16, 1, 200), (3, 8, 4, 0, 60),
                                          (2, 2, 1, 1, 40), (32, 8, 16, 100, 900), (4, 5, 5, 3, 90), (128, 8, 16, 1, 50)])
def test_reorder_matches(cuda, kind, G, W, bs, lo, hi):
    c, pm, held = pool(G + W, G, W, bs, lo, hi, 2 * G * W + 3, kind)
    rng = np.random.default_rng(G)
    for step in range(4):
        parents = rng.integers(0, W, (G, W)) if step else np.tile(np.arange(W), (G, 1))
        held = reorder(c, pm, held, parents)


@pytest.mark.parametrize("G,W,bs,lo,hi,free", [
    (3, 9, 16, 1, 120, 40), (2, 16, 4, 30, 90, 90), (32, 32, 16, 1, 70, 2100), (5, 32, 8, 200, 900, 400),  # many beams
    (4, 3, 4, 100, 400, 40000), (20, 8, 1, 200, 700, 33000),  # pools of which a thread looks through many blocks
    (1024, 1, 1, 500, 560, 8)])                               # more columns than fit a thread's marks
def test_reorder_wide_and_large(cuda, G, W, bs, lo, hi, free):
    c, pm, held = pool(G + W + bs, G, W, bs, lo, hi, free, layers=1, hkv=1)
    rng = np.random.default_rng(G)
    for step in range(2):
        held = reorder(c, pm, held, rng.integers(-1 if step else 0, W, (G, W)))


def test_reorder_all_children_of_one_and_back(cuda):
    c, pm, held = pool(1, 2, 4, 16, 37, 37, 9)
    for parents in ([[3] * 4, [0] * 4], [[1, 0, 3, 2], [3, 2, 1, 0]], [[0, 1, 2, 3]] * 2):
        held = reorder(c, pm, held, parents)


def test_reorder_whole_pages_only(cuda):
    """Tokens that end with a page: nothing is copied; and rows without tokens."""
    c, pm, held = pool(2, 2, 3, 16, 0, 0, 4, held=[48, 0])
    reorder(c, pm, held, [[2, 2, 0], [1, 1, 1]])


def test_reorder_rows_with_blocks_ahead(cuda):
    """Blocks past a row's tokens (allocated for tokens that were not kept) are let go."""
    c, pm, held = pool(3, 2, 3, 16, 60, 100, 9)
    held = [h - 30 for h in held]
    held = reorder(c, pm, held, [[0, 0, 2], [1, 2, 2]])
    reorder(c, pm, held, [[0, 1, 2], [0, 1, 2]])


def test_reorder_empties_rows(cuda):
    c, pm, held = pool(4, 3, 3, 16, 30, 70, 9)
    held = reorder(c, pm, held, [[-1, 0, 0], [-1, -1, -1], [2, 3, -7]])
    reorder(c, pm, held, [[1, 1, 1], [0, 1, 2], [0, 0, 0]])


def test_reorder_out_of_blocks(cuda):
    """Freed blocks serve first; rows that get none are empty, the others as they should be."""
    c, pm, held = pool(5, 2, 4, 16, 40, 40, 0, held=[41, 43])
    held = reorder(c, pm, held, [[0, 0, 0, 0], [0, 1, 2, 3]])
    c, pm, held = pool(6, 1, 3, 16, 40, 40, 0, held=[41])
    pm.ref_counts_dev += (pm.ref_counts_dev > 0).int()  # every block also held elsewhere: nothing is freed
    reorder(c, pm, held, [[0, 0, 0]])


def test_reorder_two_caches_of_one_pool(cuda):
    c, pm, held = pool(7, 2, 3, 16, 20, 90, 9)
    d, _, _ = pool(7, 2, 3, 16, 20, 90, 9, layers=1, hkv=1, D=128, kind="f32")
    reorder([c, d], pm, held, [[0, 0, 2], [1, 1, 1]])


def test_reorder_graph(cuda):
    """Captured once, replayed: the same as the calls in turn."""
    import torch

    from ssd_b200.kernels.page_moves import reorder_pages

    runs = []
    for captured in (False, True):
        c, pm, held = pool(8, 4, 4, 16, 20, 90, 40)
        p = torch.tensor([[0, 0, 1, 2], [3, 3, 3, 3], [0, 1, 2, 3], [1, 1, 2, 2]], dtype=torch.int32, device="cuda")
        h = torch.tensor(held, dtype=torch.int32, device="cuda")
        call = lambda: reorder_pages(c, pm.tables, pm.lens, pm.ref_counts_dev, pm.free_list, pm.free_top, p, h)  # noqa: E731
        torch.cuda.synchronize()
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            call = g.replay
        for _ in range(3):
            call()
        runs.append(state(pm) + (c.pages.clone(),))
    assert runs[0][:4] == runs[1][:4] and torch.equal(runs[0][4], runs[1][4])


def test_reorder_refusals(cuda):
    import torch

    from ssd_b200._lib import SSDError
    from ssd_b200.kernels.page_moves import reorder_pages

    c, pm, held = pool(9, 2, 2, 16, 20, 90, 9)
    p = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    h = torch.tensor(held, dtype=torch.int32, device="cuda")
    ok = dict(cache=c, tables=pm.tables, lens=pm.lens, ref_counts=pm.ref_counts_dev, free_list=pm.free_list,
              free_top=pm.free_top, parents=p, num_tokens=h)
    before = state(pm)
    for k, v in [("cache", []), ("tables", pm.tables[:3]), ("tables", pm.tables.long()), ("lens", pm.lens[:3]),
                 ("ref_counts", pm.ref_counts_dev[1:]), ("free_list", pm.free_list.cpu()), ("free_top", pm.free_top.long()),
                 ("parents", p[0]), ("parents", p.long()), ("parents", p.cpu()), ("num_tokens", h[:2]),
                 ("num_tokens", h.float())]:
        with pytest.raises((ValueError, SSDError)):
            reorder_pages(**{**ok, k: v})
    assert state(pm) == before
