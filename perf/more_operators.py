"""Cases that measure what several continuations of one prompt need in ssd_b200, beside their plain forms.

Rows (beams, branches, samples) that descend from one prompt hold forked page tables: the prompt's pages
are the same in all of them.  Three operators:

* ``attention``  each row's new tokens against its pages, the pages that a group of rows shares read once;
* ``select``     beam search's step: log-softmax of every beam's logits, the beams' scores added, the best
                 candidates over beams and vocabulary with their parents;
* ``reorder``    the rows' page tables follow the parents: whole pages shared, a partial page copied for every
                 child but the first, pages that nobody refers to back on the free list.

``own`` selects the framework's calls; otherwise ``run`` computes the operators with elementary torch
operations in 32 bits (64 where candidates are ranked).
"""

import math
import sys

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # four beams of a draft model (one KV head) shortly after a short prompt: latency
        dict(name="attention four beams", op="attention", dtype="bf16", groups=1, rows_lo=4, rows_hi=4, T=1, hq=8,
             hkv=1, D=256, bs=16, plo=137, phi=137, slo=3, shi=9),
        # the fp32 toy pair's beams, two prompts
        dict(name="attention toy fp32", op="attention", dtype="f32", groups=2, rows_lo=3, rows_hi=4, T=1, hq=4, hkv=1,
             D=64, bs=16, plo=60, phi=100, slo=1, shi=20),
        # the fan-out of a speculation tree: fifteen branches with their first two tokens
        dict(name="attention branches", op="attention", dtype="bf16", groups=1, rows_lo=15, rows_hi=15, T=2, hq=16,
             hkv=16, D=256, bs=16, plo=2003, phi=2003, slo=2, shi=6),
        # a serving batch under one long system prompt, verify steps of k = 6
        dict(name="attention system prompt", op="attention", dtype="bf16", groups=1, rows_lo=32, rows_hi=32, T=7,
             hq=16, hkv=16, D=256, bs=16, plo=8000, phi=8000, slo=60, shi=700),
        # eight prompts of unlike length, four to eight beams each, one KV head for eight query heads
        dict(name="attention many prompts", op="attention", dtype="bf16", groups=8, rows_lo=4, rows_hi=8, T=1, hq=8,
             hkv=1, D=256, bs=16, plo=1000, phi=8190, slo=5, shi=120),
        # the first step of one request with four beams: one live beam, no score yet (latency)
        dict(name="select one request", op="select", G=1, W=4, V=256000, first=True, done=0.0, alpha=0.0, masked=0.0),
        # eight requests of four beams in mid-flight, some beams finished, length-normalised
        dict(name="select eight requests", op="select", G=8, W=4, V=256000, first=False, done=0.2, alpha=0.6,
             masked=0.0),
        # the largest batch a forward takes, most of the vocabulary masked
        dict(name="select full batch", op="select", G=32, W=8, V=256000, first=False, done=0.05, alpha=1.0,
             masked=0.9),
        # a small vocabulary of odd size
        dict(name="select toy vocabulary", op="select", G=2, W=3, V=1021, first=False, done=0.0, alpha=0.0, masked=0.3),
        # the toy pair's beams (latency)
        dict(name="reorder toy", op="reorder", dtype="f32", G=1, W=4, L=2, hkv=1, D=64, bs=16, plo=45, phi=45, slo=4,
             shi=4),
        # four beams of a large model: pages of 7 MB over its layers
        dict(name="reorder four beams", op="reorder", dtype="bf16", G=1, W=4, L=28, hkv=16, D=256, bs=16, plo=500,
             phi=500, slo=27, shi=27),
        # thirty-two requests of eight beams on a draft-sized cache
        dict(name="reorder full batch", op="reorder", dtype="bf16", G=32, W=8, L=18, hkv=1, D=256, bs=16, plo=200,
             phi=4000, slo=1, shi=100),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "select", "reorder"])
    if op == "select":
        c = dict(op=op, G=_log(rng, 1, 32), W=rng.choice([1, 2, 3, 4, 5, 8, 10, 16]), V=_log(rng, 300, 256000),
                 first=rng.random() < 0.15, done=rng.choice([0.0, 0.1, 0.3]),
                 alpha=rng.choice([0.0, 0.0, 0.6, 1.0, 1.7]), masked=rng.choice([0.0, 0.0, 0.5, 0.95]))
        c["G"] = max(1, min(c["G"], 256 // c["W"]))
        return c
    dtype, hq, hkv, D = rng.choice([("bf16", 8, 1, 256), ("bf16", 16, 16, 256), ("bf16", 8, 8, 64),
                                    ("bf16", 16, 4, 128), ("f32", 4, 1, 64)])
    small = dtype == "f32"  # the fp32 pair is a toy: at most 16 rows a forward
    bs = rng.choice([16, 16, 16, 16, 4, 32])
    if op == "reorder":
        W = rng.choice([2, 3, 4, 5, 8])
        c = dict(op=op, dtype=dtype, G=max(1, min(_log(rng, 1, 32), (16 if small else 256) // W)), W=W,
                 L=2 if small else _log(rng, 2, 28), hkv=hkv, D=D, bs=bs, plo=_log(rng, 1, 300 if small else 2000), phi=0,
                 slo=rng.randint(1, 40), shi=0)
        c["phi"] = c["plo"] + _log(rng, 1, 100 if small else 2000) - 1
        c["shi"] = c["slo"] + rng.randint(0, 60)
        while _page_bytes(c) * _pool(c) > 6e9 or work(c)["bytes"] > work(listed()[3])["bytes"]:
            c["G"], c["L"], c["phi"] = max(1, c["G"] // 2), max(1, c["L"] // 2), c["plo"]
        return c
    groups = _log(rng, 1, 4 if small else 16)
    c = dict(op=op, dtype=dtype, groups=groups, rows_lo=rng.randint(1, 4), rows_hi=0, T=1, hq=hq, hkv=hkv, D=D, bs=bs,
             plo=_log(rng, 1, 300 if small else 4000), phi=0, slo=rng.randint(1, 60), shi=0)
    c["rows_hi"] = max(c["rows_lo"], min(_log(rng, 1, 32), (16 if small else 256) // groups))
    c["rows_lo"] = min(c["rows_lo"], c["rows_hi"])
    if rng.random() < 0.5:
        c["T"] = max(1, min(rng.randint(2, 8), (16 if small else 256) // (groups * c["rows_hi"])))
    c["phi"] = c["plo"] + _log(rng, 1, 100 if small else 4190) - 1
    c["slo"] = max(c["slo"], c["T"])
    c["shi"] = c["slo"] + _log(rng, 1, 20 if small else 640) - 1
    limit = work(listed()[3])
    while work(c)["bytes"] > limit["bytes"] or work(c)["flops"] > limit["flops"]:
        c["plo"], c["phi"], c["rows_hi"] = c["plo"] // 2 + 1, c["phi"] // 2 + 1, max(c["rows_lo"], c["rows_hi"] - 2)
        c["shi"] = max(c["slo"], c["shi"] // 2)
    return c


def _size(c):
    return 2 if c["dtype"] == "bf16" else 4


def _page_bytes(c):
    """Bytes of a page over all layers, K and V."""
    return 2 * c["L"] * c["bs"] * c["hkv"] * c["D"] * _size(c)


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _groups(c):
    """Rows of each group."""
    return _spread(c["rows_lo"], c["rows_hi"], c["groups"])


def _prefixes(c):
    return _spread(c["plo"], c["phi"], c["groups"])


def _tails(c):
    """Positions of each row behind its group's prefix, the new tokens among them."""
    n = sum(_groups(c))
    own_len = _spread(c["slo"], c["shi"], n)
    return [own_len[(i * 7) % n] if math.gcd(7, n) == 1 else own_len[i] for i in range(n)]


def _new(c):
    """New tokens of each row: all T in most, fewer in every fourth."""
    n = sum(_groups(c))
    return [max(1, c["T"] - c["T"] // 3) if i % 4 == 3 else c["T"] for i in range(n)]


def _tokens(c):
    """Tokens held by each request's beams (reorder)."""
    return [p + s for p, s in zip(_spread(c["plo"], c["phi"], c["G"]), _spread(c["slo"], c["shi"], c["G"]))]


def _pool(c):
    """Blocks of a reorder case's pool: the prompts' pages, the beams' own ones, and free ones."""
    bs = c["bs"]
    need = 0
    for p, n in zip(_spread(c["plo"], c["phi"], c["G"]), _tokens(c)):
        need += p // bs + c["W"] * (-(-n // bs) - p // bs)
    return need + 2 * c["G"] * c["W"] + 5


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 29)
    return {"attention": _prepare_attention, "select": _prepare_select, "reorder": _prepare_reorder}[c["op"]](c, g)


def _prepare_attention(c, g):
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    bs, hkv, D = c["bs"], c["hkv"], c["D"]
    sizes, prefixes, tails, news = _groups(c), _prefixes(c), _tails(c), _new(c)
    B = sum(sizes)
    group = [i for i, n in enumerate(sizes) for _ in range(n)]
    lens = [prefixes[group[b]] + tails[b] for b in range(B)]
    M = max(-(-n // bs) for n in lens)
    NB = sum(p // bs for p in prefixes) + sum(-(-n // bs) - prefixes[group[b]] // bs for b, n in enumerate(lens)) + 3
    ids = torch.randperm(NB, generator=g, device=DEV).to(torch.int32)
    pages = torch.empty((2, 1, NB, bs, hkv, D), dtype=dt, device=DEV)
    for p in range(2):
        pages[p] = torch.randn(pages.shape[1:], generator=g, device=DEV)
    tables = torch.full((B, M), -1, dtype=torch.int32, device=DEV)
    at, row = 0, 0
    for n, P in zip(sizes, prefixes):
        full, part = P // bs, P % bs
        shared = ids[at:at + full]
        at += full
        for i in range(n):
            rest = -(-lens[row] // bs) - full
            tables[row, :full] = shared
            tables[row, full:full + rest] = ids[at:at + rest]
            if part and i:  # the prompt's last, partial page was copied for each row
                pages[:, :, tables[row, full].long(), :part] = pages[:, :, tables[row - i, full].long(), :part]
            at += rest
            row += 1
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    starts = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    return {"case": c, "dtype": dt, "pages": pages, "tables": tables, "seq_lens": i32(lens), "q_lens": i32(news),
            "starts": i32(starts), "prefixes": i32(prefixes),
            "q": torch.randn((B, c["T"], c["hq"], D), generator=g, device=DEV).to(dt)}


def _prepare_select(c, g):
    G, W, V = c["G"], c["W"], c["V"]
    logits = 3.0 * torch.randn((G, W, V), generator=g, device=DEV)
    if c["masked"]:
        drop = torch.rand((G, W, V), generator=g, device=DEV) < c["masked"]
        logits.masked_fill_(drop, float("-inf"))
    s = {"case": c, "logits": logits}
    if c["first"]:
        s["scores"] = torch.full((G, W), float("-inf"), device=DEV)
        s["scores"][:, 0] = 0.0
        s["lengths"] = torch.zeros((G, W), dtype=torch.int32, device=DEV)
        s["finished"] = torch.zeros((G, W), dtype=torch.uint8, device=DEV)
    else:
        n = torch.randint(5, 60, (G, 1), generator=g, device=DEV)
        s["finished"] = (torch.rand((G, W), generator=g, device=DEV) < c["done"]).to(torch.uint8)
        # finished beams ended earlier
        back = torch.randint(0, 4, (G, W), generator=g, device=DEV) * s["finished"]
        s["lengths"] = (n - back).to(torch.int32)
        s["scores"] = -(1.5 * n + 4.0 * torch.rand((G, W), generator=g, device=DEV)).float()
    return s


def _prepare_reorder(c, g):
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    bs, G, W, NB = c["bs"], c["G"], c["W"], _pool(c)
    pages = torch.empty((2, c["L"], NB, bs, c["hkv"], c["D"]), dtype=dt, device=DEV)
    for p in range(2):
        for l in range(c["L"]):
            pages[p, l] = torch.randn(pages.shape[2:], generator=g, device=DEV)
    perm = torch.randperm(NB, generator=g, device=DEV).to(torch.int32)
    tokens, prefixes = _tokens(c), _spread(c["plo"], c["phi"], G)
    M = max(-(-n // bs) for n in tokens) + 1
    tables = torch.full((G * W, M), -1, dtype=torch.int32, device=DEV)
    ref = torch.zeros(NB, dtype=torch.int32, device=DEV)
    at = 0
    for i, (P, n) in enumerate(zip(prefixes, tokens)):
        full, need = P // bs, -(-n // bs)
        rows = tables[i * W:(i + 1) * W]
        rows[:, :full] = perm[at:at + full]
        ref[perm[at:at + full].long()] = W
        at += full
        mine = perm[at:at + W * (need - full)].view(W, need - full)
        rows[:, full:need] = mine
        ref[mine.long().flatten()] = 1
        at += W * (need - full)
    free = torch.full((NB,), -1, dtype=torch.int32, device=DEV)
    free[:NB - at] = perm[at:]
    # parents as beam search gives them: a few beams keep most of the children
    weight = torch.rand((G, W), generator=g, device=DEV) ** 3 + 1e-3
    parents = torch.multinomial(weight, W, replacement=True, generator=g).to(torch.int32)
    held = torch.tensor([n for n in tokens for _ in range(W)], dtype=torch.int32, device=DEV)
    return {"case": c, "dtype": dt, "pages": pages, "tables": tables, "lens": (held + bs - 1).div(bs, rounding_mode="floor")
            .to(torch.int32), "ref": ref, "free": free, "top": torch.tensor([NB - at], dtype=torch.int32, device=DEV),
            "parents": parents, "held": held}


# ---------------------------------------------------------------------------------------------- one pass
def _run_own(s):
    if "ssd-tpu-_b200" not in sys.path:
        sys.path.insert(0, "ssd-tpu-_b200")
    c, op = s["case"], s["case"]["op"]
    if op == "select":
        from ssd_b200.algorithm.beam import beam_select

        r = beam_select(s["logits"], s["scores"], s["lengths"], s["finished"], eos_token_id=_eos(c),
                        length_penalty=c["alpha"])
        return {"scores": r.scores, "parents": r.parents, "tokens": r.tokens, "lengths": r.lengths,
                "finished": r.finished}
    from ssd_b200.kernels.kv_cache import KVCacheState

    cache = KVCacheState(pages=s["pages"], block_size=c["bs"])
    if op == "attention":
        from ssd_b200.kernels.prefix_attention import shared_prefix_attention

        return shared_prefix_attention(s["q"], cache, 0, s["tables"], s["seq_lens"], s["starts"], s["prefixes"],
                                       q_lens=s["q_lens"])
    from ssd_b200.kernels.page_moves import reorder_pages

    ok = reorder_pages(cache, s["tables"], s["lens"], s["ref"], s["free"], s["top"], s["parents"], s["held"])
    return {"pages": s["pages"], "tables": s["tables"], "lens": s["lens"], "ref": s["ref"], "free": s["free"],
            "top": s["top"], "ok": ok}


def run(state):
    if own:
        return _run_own(state)
    return {"attention": _attention, "select": _select, "reorder": _reorder}[state["case"]["op"]](state)


def _eos(c):
    return 1


# ---------------------------------------------------------------------------------------------- plain forms
def _attention(s):
    c = s["case"]
    bs, hkv, D, T, hq = c["bs"], c["hkv"], c["D"], c["T"], c["hq"]
    scale = 1.0 / math.sqrt(D)
    outs, row = [], 0
    tails = _tails(c)
    for n, P in zip(_groups(c), _prefixes(c)):
        rows = slice(row, row + n)
        S = max(tails[rows])
        first = s["tables"][row].long()[: -(-P // bs)]
        k0, v0 = (s["pages"][p, 0, first].view(-1, hkv, D)[:P].float() for p in range(2))
        at = P + torch.arange(S, device=DEV)
        blk = s["tables"][rows].long().clamp(min=0)[:, (at.div(bs, rounding_mode="floor")).clamp(
            max=s["tables"].shape[1] - 1)]
        k1, v1 = (s["pages"][p, 0, blk, at % bs].float() for p in range(2))          # [n, S, Hkv, D]
        live = (at[None, :] < s["seq_lens"][rows, None])[:, :, None, None]
        k1, v1 = torch.where(live, k1, torch.zeros_like(k1)), torch.where(live, v1, torch.zeros_like(v1))
        q = s["q"][rows].float().view(n, T, hkv, hq // hkv, D)
        score = torch.cat([torch.einsum("bthgd,shd->bthgs", q, k0), torch.einsum("bthgd,bshd->bthgs", q, k1)], -1) * scale
        pos = (s["seq_lens"] - s["q_lens"])[rows, None] + torch.arange(T, device=DEV)  # [n, T]
        j = torch.arange(P + S, device=DEV)
        seen = (j[None, None, :] <= pos[:, :, None])[:, :, None, None]
        score = torch.where(seen, score, torch.full_like(score, float("-inf")))
        w = torch.exp(score - score.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        out = torch.einsum("bthgs,shd->bthgd", w[..., :P], v0) + torch.einsum("bthgs,bshd->bthgd", w[..., P:], v1)
        outs.append(out.reshape(n, T, hq, D))
        row += n
    out = torch.cat(outs)
    real = torch.arange(T, device=DEV)[None, :] < s["q_lens"][:, None]
    return torch.where(real[:, :, None, None], out, torch.zeros_like(out)).to(s["dtype"])


def _select(s):
    c = s["case"]
    G, W, V, eos, alpha = c["G"], c["W"], c["V"], _eos(c), c["alpha"]
    x = s["logits"].double()                             # 64 bits: neighbouring candidates are ranked by these
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    score = s["scores"].double()[:, :, None] + (x - lse)
    lens = s["lengths"].double()[:, :, None]
    rank = score / (lens + 1) ** alpha
    done = s["finished"].bool()[:, :, None]
    is_eos = torch.arange(V, device=DEV) == eos
    none = torch.full_like(rank, float("-inf"))
    rank = torch.where(done, torch.where(is_eos, s["scores"].double()[:, :, None] / lens.clamp(min=1) ** alpha, none),
                       rank)
    rank = torch.where(torch.isnan(rank), none, rank)
    best, order = torch.sort(rank.view(G, W * V), dim=1, descending=True, stable=True)
    best, order = best[:, :W], order[:, :W]
    live = best > float("-inf")
    parents, tokens = order // V, order % V
    was_done = s["finished"].bool().gather(1, parents)
    picked = torch.where(was_done, s["scores"].double().gather(1, parents), score.view(G, W * V).gather(1, order))
    lengths = s["lengths"].gather(1, parents) + (~was_done).int()
    no = torch.full_like(parents, -1)
    return {"scores": torch.where(live, picked, torch.full_like(picked, float("-inf"))).float(),
            "parents": torch.where(live, parents, no).int(), "tokens": torch.where(live, tokens, no).int(),
            "lengths": torch.where(live, lengths, torch.zeros_like(lengths)),
            "finished": (~live | was_done | (tokens == eos)).to(torch.uint8)}


def _reorder(s):
    c = s["case"]
    bs, W, NB = c["bs"], c["W"], s["ref"].shape[0]
    B, M = s["tables"].shape
    rows = torch.arange(B, device=DEV)
    parent = (rows // W) * W + s["parents"].view(-1).long()
    children = torch.zeros(B, dtype=torch.int64, device=DEV).index_add_(0, parent, torch.ones_like(parent))
    same = parent[:, None] == parent[None, :]
    first = ~(same & (rows[None, :] < rows[:, None])).any(1)
    held = s["held"].long()
    full, part = held // bs, held % bs != 0
    need = full + part
    # references: every row lets go of its pages, every child takes its parent's whole ones, the first child the partial one
    j = torch.arange(M, device=DEV)[None, :]
    old = s["tables"].long()
    change = torch.where(j < full[:, None], children[:, None] - 1,
                         torch.where(j < need[:, None], (children[:, None] > 0).long() - 1, torch.full_like(old, -1)))
    change = torch.where(j < s["lens"][:, None], change, torch.zeros_like(change))
    spare = torch.zeros(NB + 1, dtype=torch.int64, device=DEV)
    ids = torch.where(old >= 0, old, torch.full_like(old, NB)).view(-1)
    ref = torch.cat([s["ref"].long(), spare[:1]]).index_add_(0, ids, change.view(-1))[:NB]
    gone = (s["ref"] > 0) & (ref == 0)
    # freed pages in ascending order behind the others, then one popped for each further child of a partial page
    pos = s["top"] + torch.cumsum(gone.long(), 0) - 1
    stack = torch.cat([s["free"].long(), spare[:1]])
    blocks = torch.arange(NB, device=DEV)
    stack[torch.where(gone, pos, torch.full_like(pos, NB))] = blocks
    top = s["top"].long() + gone.sum()
    take = part[parent] & ~first
    slot = top - torch.cumsum(take.long(), 0)
    fresh = stack[torch.where(take, slot, torch.full_like(slot, NB))]
    stack[torch.where(take, slot, torch.full_like(slot, NB))] = -1
    tables = torch.where(j < need[parent][:, None], old[parent], torch.full_like(old, -1))
    src = old[parent, full[parent]]
    tables[rows, full[parent]] = torch.where(take, fresh, tables[rows, full[parent]])
    ref = torch.cat([ref, spare[:1]])
    ref[torch.where(take, fresh, torch.full_like(fresh, NB))] = 1
    moved = take.nonzero().squeeze(1)
    a, b = src[moved], fresh[moved]
    live = (torch.arange(bs, device=DEV)[None, :] < (held % bs)[parent][moved, None])[None, None, :, :, None, None]
    s["pages"][:, :, b] = torch.where(live, s["pages"][:, :, a], s["pages"][:, :, b])
    s["tables"].copy_(tables)
    s["lens"].copy_(need[parent])
    s["ref"].copy_(ref[:NB])
    s["free"].copy_(stack[:NB])
    s["top"].copy_((top - take.sum()).view(1))
    return {"pages": s["pages"], "tables": s["tables"], "lens": s["lens"], "ref": s["ref"], "free": s["free"],
            "top": s["top"], "ok": torch.ones(B, dtype=torch.uint8, device=DEV)}


# ---------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "select":
        rows = c["G"] * (1 if c["first"] else c["W"])
        return {"bytes": 4 * rows * c["V"] + 34 * c["G"] * c["W"], "flops": 4 * rows * c["V"]}
    if c["op"] == "reorder":
        # the rows' tables read and written; of a partial page's copies about two in five children are further ones
        B, bs = c["G"] * c["W"], c["bs"]
        entries = c["W"] * sum(-(-n // bs) for n in _tokens(c))
        rows = sum(0.4 * c["W"] * (n % bs) for n in _tokens(c))
        return {"bytes": int(2 * rows * _page_bytes(c) / bs) + 8 * entries + 16 * B, "flops": 0}
    row, R = c["hkv"] * c["D"], c["hq"] * c["D"]
    sizes, prefixes, tails, news = _groups(c), _prefixes(c), _tails(c), _new(c)
    seen = sum(prefixes) + sum(tails)
    group = [i for i, n in enumerate(sizes) for _ in range(n)]
    pairs = sum((prefixes[group[b]] + tails[b]) * news[b] for b in range(sum(sizes)))
    return {"bytes": 2 * seen * row * _size(c) + 2 * sum(sizes) * c["T"] * R * _size(c), "flops": 4 * pairs * R}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    c = case
    if c["op"] == "reorder":
        return None  # pages move and whole numbers change: nothing is computed
    s = prepare(case, seed)
    if c["op"] == "select":
        G, W, V = c["G"], c["W"], c["V"]
        scores = torch.full((G, W), float("-inf"), dtype=torch.float64, device=DEV)
        for g in range(G):
            cand = []  # (rank, score)
            for w in range(W):
                base, n = float(s["scores"][g, w]), int(s["lengths"][g, w])
                if base == float("-inf"):
                    continue
                if int(s["finished"][g, w]):
                    cand.append((base / max(n, 1) ** c["alpha"], base))
                    continue
                lp = torch.log_softmax(s["logits"][g, w].double(), 0)
                best = torch.topk(lp, min(W, V)).values
                cand += [((base + v) / (n + 1) ** c["alpha"], base + v) for v in best.tolist() if v > float("-inf")]
            cand.sort(key=lambda t: -t[0])
            for i, (_, v) in enumerate(cand[:W]):
                scores[g, i] = v
        return {"scores": scores, "parents": None, "tokens": None, "lengths": None, "finished": None}
    bs, G = c["bs"], c["hq"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lens, news = s["seq_lens"].tolist(), s["q_lens"].tolist()
    for b in range(len(lens)):
        n, t = lens[b], news[b]
        at = torch.arange(n, device=DEV)
        blk = s["tables"][b].long()[at // bs]
        k, v = (s["pages"][p, 0, blk, at % bs].double().transpose(0, 1) for p in range(2))  # [Hkv, n, D]
        for i in range(t):
            see = n - t + i + 1
            q = s["q"][b, i].double().view(c["hkv"], G, c["D"])
            w = torch.softmax(q @ k[:, :see].transpose(1, 2) / math.sqrt(c["D"]), -1)
            out[b, i] = (w @ v[:, :see]).reshape(c["hq"], c["D"])
    return out
