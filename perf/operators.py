"""Cases that measure the 8-bit paged KV cache and the page moves of ssd_b200, beside their plain forms.

The cache holds K and V as e4m3 with one power-of-two scale for each page (``block_size`` tokens) and KV
head: ``pages[2, L, NB, BS, Hkv, D]`` and ``scales[2, L, NB, Hkv]`` (fp32).  Four operators:

* ``append``       new K/V rows enter their sequences' pages, quantised; as ``rope_append`` from a QKV
                   projection's rows, with the rotary embedding of q and k;
* ``attention``    each sequence's new tokens against its pages;
* ``copy``         whole pages of every layer copied inside a cache;
* ``compact``      the used pages of a fragmented pool moved to its front, tables and free list rebuilt.

``own`` selects the framework's calls; otherwise ``run`` computes the operators with elementary torch
operations in 32 bits.
"""

import math
import sys

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one draft token of one sequence, one KV head: the append of a draft decode step (latency)
        dict(name="append one token", op="append", dtype="bf16", B=1, T=1, hkv=1, D=256, bs=16, lo=137, hi=137),
        # four whole prompts entering a 16-head cache (prefill)
        dict(name="append prompts", op="append", dtype="bf16", B=4, T=1500, hkv=16, D=256, bs=16, lo=1500, hi=1531),
        # a verify step of eight sequences, k = 4: five rows each, lengths anywhere in a page
        dict(name="rope append verify", op="rope_append", dtype="bf16", B=8, T=5, hq=16, hkv=16, D=256, bs=16,
             lo=500, hi=4096),
        # one draft token of one short sequence (latency)
        dict(name="attention one token", op="attention", dtype="bf16", B=1, T=1, hq=8, hkv=1, D=256, bs=16, lo=137,
             hi=137),
        # the fp32 toy pair's verify step
        dict(name="attention toy fp32", op="attention", dtype="f32", B=2, T=5, hq=4, hkv=1, D=64, bs=16, lo=77, hi=200),
        # the target's verify step over eight sequences, k = 4
        dict(name="attention verify", op="attention", dtype="bf16", B=8, T=5, hq=16, hkv=16, D=256, bs=16, lo=512,
             hi=4096),
        # a serving batch with long contexts, k = 6
        dict(name="attention long batch", op="attention", dtype="bf16", B=32, T=7, hq=16, hkv=16, D=256, bs=16,
             lo=2000, hi=8192),
        # prompt chunks against long contexts, one KV head for eight query heads
        dict(name="attention prompt chunk", op="attention", dtype="bf16", B=4, T=64, hq=8, hkv=1, D=256, bs=16,
             lo=1000, hi=8192),
        # copy-on-write of a few pages of a two-layer cache (a fork's partial pages)
        dict(name="copy few pages", op="copy", dtype="bf16", L=2, NB=64, bs=16, hkv=1, D=64, n=3),
        # the pages of long prefixes duplicated across an 18-layer cache
        dict(name="copy many pages", op="copy", dtype="bf16", L=18, NB=2500, bs=16, hkv=4, D=256, n=1100),
        # a serving pool with sequences finished in between: used pages scattered over the whole pool
        dict(name="compact pool", op="compact", dtype="bf16", L=18, NB=3000, bs=16, hkv=1, D=256, rows=32,
             fill=0.45),
        # the toy pair's small pool (latency)
        dict(name="compact small pool", op="compact", dtype="f32", L=2, NB=256, bs=16, hkv=1, D=64, rows=4, fill=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "rope_append", "attention", "attention", "copy", "compact"])
    if op in ("copy", "compact"):
        hkv, D = rng.choice([(1, 64), (1, 256), (4, 256), (16, 256), (8, 64), (2, 128)])
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), L=_log(rng, 1, 28), NB=_log(rng, 40, 3000),
                 bs=rng.choice([16, 16, 16, 4, 32]), hkv=hkv, D=D)
        while _page_bytes(c) * c["NB"] > 2e9:
            c["NB"] = max(40, c["NB"] // 2)
            c["L"] = max(1, c["L"] // 2)
        if op == "copy":
            c["n"] = _log(rng, 1, c["NB"] // 2 - 1)
        else:
            c.update(rows=rng.randint(1, 32), fill=round(rng.uniform(0.2, 0.9), 2))
        return c
    dtype, hq, hkv, D = rng.choice([("bf16", 8, 1, 256), ("bf16", 16, 16, 256), ("bf16", 8, 8, 64),
                                    ("bf16", 16, 4, 128), ("f32", 4, 1, 64)])
    small = dtype == "f32"  # the fp32 pair is a toy: at most 16 rows a forward
    c = dict(op=op, dtype=dtype, B=_log(rng, 1, 3 if small else 32), T=0, hkv=hkv, D=D,
             bs=rng.choice([16, 16, 16, 16, 4, 32]))
    if op != "append":
        c["hq"] = hq
    if op == "append":
        c["T"] = _log(rng, 1, 5 if small else 1500)
        while c["B"] * c["T"] * hkv * D > 2.4e7:
            c["B"] = max(1, c["B"] // 2)
    else:
        c["T"] = _log(rng, 1, 5 if small else 8 if rng.random() < 0.6 else 200)
        c["B"] = max(1, min(c["B"], (16 if small else 256) // c["T"]))
    c["lo"] = c["T"] + _log(rng, 1, 300 if small else 2000) - 1
    c["hi"] = c["lo"] + _log(rng, 1, 100 if small else 6000) - 1
    return c


def _page_bytes(c):
    return 2 * c["L"] * c["bs"] * c["hkv"] * c["D"] * _size(c)


def _size(c):
    return 2 if c["dtype"] == "bf16" else 4


def _lens(c):
    """The sequences' lengths, new tokens included: spread over [lo, hi] whatever the seed."""
    B = c["B"]
    return [c["lo"] + (c["hi"] - c["lo"]) * i // max(1, B - 1) for i in range(B)] if B > 1 else [c["hi"]]


def _new(c):
    """New tokens of each sequence: all T in most rows, fewer in every fourth."""
    return [max(1, c["T"] - c["T"] // 3) if i % 4 == 3 else c["T"] for i in range(c["B"])]


def _used(c):
    return max(c["rows"], int(c["NB"] * c["fill"]))


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 17)
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    if c["op"] in ("copy", "compact"):
        return _prepare_pool(c, g, dt)
    s = {"case": c, "dtype": dt}
    B, T, hkv, D, bs = c["B"], c["T"], c["hkv"], c["D"], c["bs"]
    lens = torch.tensor(_lens(c), device=DEV)[torch.randperm(B, generator=g, device=DEV)]
    M = -(-max(_lens(c)) // bs)
    s["q_lens"] = torch.tensor(_new(c), dtype=torch.int32, device=DEV)
    s["seq_lens"] = lens.to(torch.int32)
    # rows that attention reads are live; an append needs the sequences' last pages alone, so its pool holds those
    first = (lens - s["q_lens"]).div(bs, rounding_mode="floor") if c["op"] != "attention" else torch.zeros_like(lens)
    need = (lens + bs - 1).div(bs, rounding_mode="floor") - first
    NB = B * int(need.max()) + 3
    ids = torch.randperm(NB, generator=g, device=DEV)[: B * int(need.max())].view(B, -1)
    page = torch.arange(M, device=DEV)[None, :] - first[:, None]
    live = (page >= 0) & (page < need[:, None])
    s["tables"] = torch.where(live, ids.gather(1, page.clamp(0, ids.shape[1] - 1)), -1).to(torch.int32)
    s["pages"] = torch.empty((2, 1, NB, bs, hkv, D), dtype=torch.float8_e4m3fn, device=DEV)
    s["scales"] = torch.empty((2, 1, NB, hkv), dtype=torch.float32, device=DEV)
    s["layer"] = 0
    step = max(1, (1 << 28) // (bs * hkv * D))
    for p in range(2):
        for a in range(0, NB, step):
            n = min(step, NB - a)
            x = torch.randn((n, bs, hkv, D), generator=g, device=DEV)
            x *= torch.exp(0.4 * torch.randn((n, 1, hkv, 1), generator=g, device=DEV))  # pages of unlike magnitude
            x, sc = _quantise(x.to(torch.bfloat16).float(), None)
            s["pages"][p, 0, a:a + n] = x
            s["scales"][p, 0, a:a + n] = sc
    if c["op"] == "attention":
        s["q"] = torch.randn((B, T, c["hq"], D), generator=g, device=DEV).to(dt)
        s["scale"] = 1.0 / math.sqrt(D)
    else:
        N = T + 2 * bs
        at = first[:, None] * bs + torch.arange(N, device=DEV)[None, :]
        s["touched"] = torch.where(at < lens[:, None], at, -1).to(torch.int32)  # what the append changes
        if c["op"] == "append":
            s["k"] = (1.5 * torch.randn((B, T, hkv, D), generator=g, device=DEV)).to(dt)
            s["v"] = torch.randn((B, T, hkv, D), generator=g, device=DEV).to(dt)
        else:
            s["qkv"] = torch.randn((B * T, (c["hq"] + 2 * hkv) * D), generator=g, device=DEV).to(dt)
            ang = torch.arange(c["hi"] + 1, dtype=torch.float64, device=DEV)[:, None] / (
                10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D))[None, :]
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    return s


def _prepare_pool(c, g, dt):
    s = {"case": c, "dtype": dt}
    NB = c["NB"]
    s["pages"] = torch.empty((2, c["L"], NB, c["bs"], c["hkv"], c["D"]), dtype=dt, device=DEV)
    for p in range(2):
        for l in range(c["L"]):
            s["pages"][p, l] = torch.randn(s["pages"].shape[2:], generator=g, device=DEV)
    perm = torch.randperm(NB, generator=g, device=DEV).to(torch.int32)
    if c["op"] == "copy":
        s["src"], s["dst"] = perm[: c["n"]].contiguous(), perm[c["n"]: 2 * c["n"]].contiguous()
    else:
        # `used` scattered blocks over `rows` tables of unlike length; two rows share a prefix block
        used, rows = _used(c), c["rows"]
        cut = [used * i * (i + 1) // (rows * (rows + 1)) for i in range(rows + 1)]
        lens = [b - a for a, b in zip(cut, cut[1:])]
        M = max(lens) + 2
        tables = torch.full((rows, M), -1, dtype=torch.int32, device=DEV)
        start = torch.tensor(cut[:-1], device=DEV)[:, None] + torch.arange(M, device=DEV)[None, :]
        live = torch.arange(M, device=DEV)[None, :] < torch.tensor(lens, device=DEV)[:, None]
        tables[live] = perm[start[live]]
        ref = torch.zeros(NB, dtype=torch.int32, device=DEV)
        ref[perm[:used].long()] = 1
        if rows > 1 and lens[-2] > 0:
            gone = tables[-1, 0].long()
            tables[-1, 0] = tables[-2, 0]
            ref[tables[-2, 0].long()] += 1
            ref[gone] = 0
            free = torch.cat([perm[used:], gone[None].to(torch.int32)])
        else:
            free = perm[used:]
        s["tables"], s["lens"] = tables, torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["ref"] = ref
        s["free"] = torch.full((NB,), -1, dtype=torch.int32, device=DEV)
        s["free"][: free.numel()] = free
        s["top"] = torch.tensor([free.numel()], dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------- one pass
def _modules():
    if "ssd-tpu-_b200" not in sys.path:
        sys.path.insert(0, "ssd-tpu-_b200")
    from ssd_b200.kernels import kv8_cache, kv_cache, page_moves

    return kv8_cache, kv_cache, page_moves


def _run_own(s):
    c, op = s["case"], s["case"]["op"]
    k8, kv, moves = _modules()
    if op in ("copy", "compact"):
        cache = kv.KVCacheState(pages=s["pages"], block_size=c["bs"])
        if op == "copy":
            moves.copy_pages(cache, s["src"], s["dst"])
            return s["pages"]
        r = moves.compact_pages(cache, s["tables"], s["lens"], s["ref"], s["free"], s["top"])
        return {"pages": s["pages"], "tables": r.tables, "ref": r.ref_counts, "free": r.free_list, "top": r.free_top,
                "remap": r.remap}
    cache = k8.KV8CacheState(pages=s["pages"], scales=s["scales"], block_size=c["bs"])
    if op == "attention":
        return k8.paged_kv8_attention(s["q"], cache, s["layer"], s["tables"], s["seq_lens"], q_lens=s["q_lens"],
                                      scale=s["scale"])
    if op == "append":
        k8.append_kv8(cache, s["layer"], s["tables"], s["seq_lens"], s["k"], s["v"], q_lens=s["q_lens"])
        return k8.gather_kv8(cache, s["layer"], s["tables"], s["touched"])
    q = k8.rope_append_kv8(s["qkv"], cache, s["layer"], s["tables"], s["seq_lens"], c["hq"], s["cos"], s["sin"],
                           q_lens=s["q_lens"])
    return (q,) + k8.gather_kv8(cache, s["layer"], s["tables"], s["touched"])


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        return _run_own(s)
    if op == "append":
        _append(s, s["k"].float(), s["v"].float())
        return _gather(s, s["touched"], torch.bfloat16)
    if op == "rope_append":
        return _rope_append(s)
    if op == "attention":
        return _attention(s)
    if op == "copy":
        s["pages"][:, :, s["dst"].long()] = s["pages"][:, :, s["src"].long()]
        return s["pages"]
    return _compact(s)


# ---------------------------------------------------------------------------------------------- plain forms
def _quantise(x, floor):
    """x [..., BS, Hkv, D] as e4m3 under the smallest power of two that keeps each page and head within 448
    (and, where `floor` is given, is not below it); and that scale [..., Hkv]."""
    amax = x.abs().amax(dim=(-3, -1))
    m, e = torch.frexp(amax)                       # amax = m 2^e, m in [1/2, 1); 448 = (7/8) 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-118)
    e = torch.where(amax > 0, e, torch.full_like(e, -118))
    sc = torch.ldexp(torch.ones_like(amax), e)
    if floor is not None:
        sc = torch.maximum(sc, floor)
    return (x / sc[..., None, :, None]).to(torch.float8_e4m3fn), sc


def _append(s, k, v):
    """The pages that the new rows touch are read, joined with the rows, quantised again and written back."""
    c, bs = s["case"], s["case"]["bs"]
    B, T = k.shape[:2]
    start = (s["seq_lens"] - s["q_lens"]).long()
    P = (T + bs - 2) // bs + 1                                     # pages that T rows can touch
    logical = start[:, None].div(bs, rounding_mode="floor") + torch.arange(P, device=k.device)[None, :]
    at = logical[:, :, None] * bs + torch.arange(bs, device=k.device)   # [B, P, BS] positions
    end = s["seq_lens"].long()[:, None, None]
    new = (at >= start[:, None, None]) & (at < end)
    touched = new.any(-1)
    blk = s["tables"].long().gather(1, logical.clamp(max=s["tables"].shape[1] - 1))
    b, p = touched.nonzero(as_tuple=True)
    blk = blk[b, p]
    src = (at - start[:, None, None]).clamp(0, T - 1)[b, p]        # [n, BS] rows of k and v
    new = new[b, p]
    kept = (at < start[:, None, None])[b, p]
    for plane, x in ((0, k), (1, v)):
        rows = x[b[:, None], src]                                  # [n, BS, Hkv, D]
        old, osc = s["pages"][plane, s["layer"], blk], s["scales"][plane, s["layer"], blk]
        old_sc = torch.where(kept.any(-1)[:, None], osc, torch.zeros_like(osc))
        _, sc = _quantise(torch.where(new[..., None, None], rows, torch.zeros_like(rows)), old_sc)
        val = torch.where(new[..., None, None], rows, old.float() * osc[:, None, :, None])
        q = (val / sc[:, None, :, None]).to(torch.float8_e4m3fn)
        live = (new | kept)[..., None, None].expand_as(q)
        s["pages"][plane, s["layer"], blk] = torch.where(live, q.view(torch.uint8),
                                                         old.view(torch.uint8)).view(torch.float8_e4m3fn)
        s["scales"][plane, s["layer"], blk] = sc


def _gather(s, positions, dtype):
    bs = s["case"]["bs"]
    pos = positions.long()
    ok = pos >= 0
    p = pos.clamp(min=0)
    blk = s["tables"].long().gather(1, p.div(bs, rounding_mode="floor"))
    live = ok[..., None, None]
    x = s["pages"][:, s["layer"], blk, p % bs].float() * s["scales"][:, s["layer"], blk][..., None]
    x = torch.where(live, x, torch.zeros_like(x)).to(dtype)
    return x[0], x[1]


def _rope_append(s):
    c = s["case"]
    B, T, hq, hkv, D = c["B"], c["T"], c["hq"], c["hkv"], c["D"]
    x = s["qkv"].float().view(B, T, hq + 2 * hkv, D)
    at = (s["seq_lens"] - s["q_lens"]).long()[:, None] + torch.arange(T, device=x.device)
    real = (torch.arange(T, device=x.device)[None, :] < s["q_lens"][:, None])
    at = torch.where(real, at, torch.zeros_like(at))
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    a, b = x[:, :, :hq + hkv, :D // 2], x[:, :, :hq + hkv, D // 2:]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    _append(s, y[:, :, hq:], x[:, :, hq + hkv:])
    q = torch.where(real[:, :, None, None], y[:, :, :hq], torch.zeros_like(y[:, :, :hq]))
    return (q.to(s["dtype"]),) + _gather(s, s["touched"], torch.bfloat16)


def _attention(s):
    c = s["case"]
    B, T, hq, hkv, D, bs = c["B"], c["T"], c["hq"], c["hkv"], c["D"], c["bs"]
    S = s["tables"].shape[1] * bs
    blk = s["tables"].long().clamp(min=0)
    j = torch.arange(S, device=DEV)
    live = (j[None, :] < s["seq_lens"][:, None])                               # [B, S]
    x = s["pages"][:, s["layer"], blk].float() * s["scales"][:, s["layer"], blk][:, :, :, None, :, None]
    x = x.view(2, B, S, hkv, D)
    x = torch.where(live[None, :, :, None, None], x, torch.zeros_like(x))
    q = s["q"].float().view(B, T, hkv, hq // hkv, D)
    score = torch.einsum("bthgd,bshd->bhgts", q, x[0]) * s["scale"]
    pos = (s["seq_lens"] - s["q_lens"])[:, None] + torch.arange(T, device=DEV)  # [B, T]
    seen = (j[None, None, :] <= pos[:, :, None])[:, None, None]
    score = torch.where(seen, score, torch.full_like(score, float("-inf")))
    score = score - score.amax(-1, keepdim=True)
    w = torch.exp(score)
    w = w / w.sum(-1, keepdim=True)
    out = torch.einsum("bhgts,bshd->bthgd", w, x[1]).reshape(B, T, hq, D)
    real = torch.arange(T, device=DEV)[None, :] < s["q_lens"][:, None]
    return torch.where(real[:, :, None, None], out, torch.zeros_like(out)).to(s["dtype"])


def _compact(s):
    NB = s["case"]["NB"]
    ids = torch.arange(NB, device=DEV)
    free = s["free"].long()
    is_free = torch.zeros(NB + 1, dtype=torch.bool, device=DEV)
    is_free[torch.where(ids < s["top"], free, torch.full_like(free, NB))] = True
    is_free = is_free[:NB]
    used = (~is_free).sum()
    src = (~is_free & (ids >= used)).nonzero().squeeze(1)
    dst = (is_free & (ids < used)).nonzero().squeeze(1)
    s["pages"][:, :, dst] = s["pages"][:, :, src]
    remap = torch.where(is_free, torch.full_like(ids, -1), ids)
    remap[src] = dst
    ref = s["ref"].clone()
    ref[dst] = s["ref"][src]
    ref[src] = 0
    live = torch.arange(s["tables"].shape[1], device=DEV)[None, :] < s["lens"][:, None]
    tables = torch.where(live, remap[s["tables"].long().clamp(min=0)], torch.full_like(s["tables"], -1).long())
    n = NB - used
    lst = torch.where(ids < n, NB - 1 - ids, torch.full_like(ids, -1))
    return {"pages": s["pages"], "tables": tables.to(torch.int32), "ref": ref, "free": lst.to(torch.int32),
            "top": n.to(torch.int32)[None], "remap": remap.to(torch.int32)}


# ---------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "copy":
        return {"bytes": 2 * c["n"] * _page_bytes(c), "flops": 0}
    if c["op"] == "compact":
        used = _used(c)  # of scattered blocks, the share of the pool that is free lies in front of the used ones
        return {"bytes": 2 * used * (1 - used / c["NB"]) * _page_bytes(c) + 8 * c["NB"], "flops": 0}
    row = c["hkv"] * c["D"]
    if c["op"] == "attention":
        seen = sum(_lens(c))
        pairs = sum(n * t for n, t in zip(sorted(_lens(c)), _new(c)))
        return {"bytes": 2 * seen * row + 2 * c["B"] * c["T"] * c["hq"] * c["D"] * _size(c),
                "flops": 4 * pairs * c["hq"] * c["D"]}
    new = sum(_new(c))
    # K and V rows read, the pages written, and the touched rows handed out in 16 bits
    b = 2 * new * row * (_size(c) + 1 + 2)
    if c["op"] == "rope_append":
        b += 2 * c["B"] * c["T"] * c["hq"] * c["D"] * _size(c) + new * c["D"] * 4
    return {"bytes": b, "flops": 6 * new * row}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "copy":
        out = s["pages"].double()
        out.index_copy_(2, s["dst"].long(), out.index_select(2, s["src"].long()))
        return out
    if c["op"] == "compact":
        return None  # pages move and whole numbers change: nothing is computed
    bs = c["bs"]
    lens, news = s["seq_lens"].tolist(), s["q_lens"].tolist()
    if c["op"] == "attention":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        G = c["hq"] // c["hkv"]
        for b in range(c["B"]):
            n, t = lens[b], news[b]
            at = torch.arange(n, device=DEV)
            blk = s["tables"][b].long()[at // bs]
            for h in range(c["hkv"]):
                kk = s["pages"][0, 0, blk, at % bs, h].double() * s["scales"][0, 0, blk, h].double()[:, None]
                vv = s["pages"][1, 0, blk, at % bs, h].double() * s["scales"][1, 0, blk, h].double()[:, None]
                for i in range(t):
                    see = n - t + i + 1
                    q = s["q"][b, i, h * G:(h + 1) * G].double()
                    w = torch.softmax(q @ kk[:see].T * s["scale"], -1)
                    out[b, i, h * G:(h + 1) * G] = w @ vv[:see]
        return out
    hkv, D, T = c["hkv"], c["D"], c["T"]
    if c["op"] == "append":
        k, v, q = s["k"].double(), s["v"].double(), None
    else:
        hq = c["hq"]
        x = s["qkv"].double().view(c["B"], T, hq + 2 * hkv, D)
        z = torch.complex(x[..., :D // 2], x[..., D // 2:])[:, :, :hq + hkv]
        r = torch.zeros((c["B"], T, D // 2), dtype=torch.complex128, device=DEV)
        for b in range(c["B"]):
            at = torch.arange(lens[b] - news[b], lens[b], device=DEV)
            r[b, :news[b]] = torch.complex(s["cos"][at].double(), s["sin"][at].double())
        z = z * r[:, :, None]
        y = torch.cat([z.real, z.imag], -1)
        q, k, v = y[:, :, :hq], y[:, :, hq:], x[:, :, hq + hkv:]
    N = s["touched"].shape[1]
    outs = [torch.zeros((c["B"], N, hkv, D), dtype=torch.float64, device=DEV) for _ in range(2)]
    for b in range(c["B"]):
        n0 = lens[b] - news[b]
        base = n0 // bs * bs
        for plane, x in ((0, k), (1, v)):
            for p in range(base // bs, -(-lens[b] // bs)):
                a, e = max(n0, p * bs), min(lens[b], (p + 1) * bs)
                blk = int(s["tables"][b, p])
                rows = x[b, a - n0:e - n0]
                need = rows.abs().amax(dim=(0, 2)) / 448
                sc = torch.exp2(torch.ceil(torch.log2(need.clamp(min=2.0 ** -118))))
                sc = torch.where(sc * 0.5 >= need, sc * 0.5, sc).clamp(min=2.0 ** -118)
                if a > p * bs:
                    osc = s["scales"][plane, 0, blk].double()
                    sc = torch.maximum(sc, osc)
                    rows = torch.cat([s["pages"][plane, 0, blk, :a - p * bs].double() * osc[None, :, None], rows])
                outs[plane][b, p * bs - base:e - base] = _e4m3(rows / sc[None, :, None]) * sc[None, :, None]
    return tuple(outs) if q is None else (q, outs[0], outs[1])


def _e4m3(x):
    """x at the nearest value with four significant bits, steps of 2^-9 at least, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step
