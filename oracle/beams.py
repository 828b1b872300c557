"""Numpy restatement, in 64 bits, of what several continuations of one prompt need: attention over shared prefixes,
beam search's selection, and the re-ordering of paged rows.

Test infrastructure only.
"""

from __future__ import annotations

import numpy as np


def prefix_attention(q, pages, tables, seq_lens, q_lens, starts, prefixes, scale):
    """q [B, T, Hq, D], pages [2, NB, BS, Hkv, D] of one layer; returns (out, size, slack).

    ``size`` is sum_j w_j |v_j| / sum_j w_j over the finite seen V, what a relative error of the weights scales with;
    ``slack`` [B, T, Hq] the largest sum_d |q_d k_d| |scale| over the seen positions, what the scores' error scales
    with.  Rows that see nothing are zeros.
    """
    B, T, Hq, D = q.shape
    _, NB, BS, Hkv, _ = pages.shape
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    slack = np.zeros((B, T, Hq))
    for g in range(len(prefixes)):
        for b in range(starts[g], starts[g + 1]):
            ql = T if q_lens is None else int(np.clip(q_lens[b], 0, T))
            for t in range(ql):
                p = int(seq_lens[b]) - ql + t
                j = np.arange(p + 1)
                row = np.where(j < prefixes[g], starts[g], b)
                ok = j // BS < tables.shape[1]
                blk = np.where(ok, tables[row, np.minimum(j // BS, tables.shape[1] - 1)], -1)
                ok &= (blk >= 0) & (blk < NB)
                j, blk = j[ok], blk[ok]
                if len(j) == 0:
                    continue
                for h in range(Hq):
                    kv = h // (Hq // Hkv)
                    k = pages[0, blk, j % BS, kv].astype(np.float64)
                    v = pages[1, blk, j % BS, kv].astype(np.float64)
                    x = q[b, t, h].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = k @ x * scale
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        out[b, t, h] = w @ v
                        size[b, t, h] = w @ np.where(np.isfinite(v), np.abs(v), 0)
                        slack[b, t, h] = (np.abs(k) @ np.abs(x)).max() * abs(scale)
    return out, size, slack


def beam_select(logits, scores, lengths, finished, eos, alpha):
    """[G, W, V] fp32, [G, W]; (scores, parents, tokens, lengths, finished), see ``ssd_beam_select``."""
    G, W, V = logits.shape
    o_s = np.full((G, W), -np.inf)
    o_p, o_t = np.full((G, W), -1), np.full((G, W), -1)
    o_l, o_f = np.zeros((G, W), int), np.ones((G, W), int)
    for g in range(G):
        cand = []
        for w in range(W):
            base = float(scores[g, w])
            n = 0 if lengths is None else int(lengths[g, w])
            if not base > -np.inf:
                continue
            if finished is not None and finished[g, w]:
                cand.append((-(base / max(n, 1) ** alpha), w * V + eos, base, n, 1))
                continue
            x = logits[g, w].astype(np.float64)
            if np.isnan(x).any() or x.max() in (np.inf, -np.inf):
                continue
            lse = x.max() + np.log(np.exp(x - x.max()).sum())
            best = np.lexsort((np.arange(V), -x))[:W]  # equal logits: the lower token first
            for v in best:
                if x[v] > -np.inf:
                    s = base + (x[v] - lse)
                    cand.append((-(s / (n + 1) ** alpha), w * V + int(v), s, n + 1, int(v == eos)))
        cand.sort(key=lambda c: c[:2])
        for i, (_, flat, s, n, f) in enumerate(cand[:W]):
            o_s[g, i], o_p[g, i], o_t[g, i], o_l[g, i], o_f[g, i] = s, flat // V, flat % V, n, f
    return o_s, o_p, o_t, o_l, o_f


def reorder(tables, lens, refs, free, parents, held, block_size):
    """Lists of blocks a row; returns (tables, refs, free, ok, copies [(row, src, dst, rows)])."""
    W = parents.shape[1]
    B = len(tables)
    refs, free = dict(refs), list(free)
    par = [b // W * W + int(parents.flat[b]) if 0 <= parents.flat[b] < W else -1 for b in range(B)]
    new, want = [], []
    for b in range(B):
        p = par[b]
        if p < 0:
            new.append([])
            want.append(None)
            continue
        full = min(held[p] // block_size, lens[p])
        part = full < lens[p] and held[p] % block_size
        row = list(tables[p][:full])
        if part:
            if par.index(p) == b:
                row.append(tables[p][full])
                want.append(None)
            else:
                want.append((tables[p][full], int(held[p] % block_size)))
        else:
            want.append(None)
        new.append(row)
    for row in new:
        for blk in row:
            refs[blk] = refs.get(blk, 0) + 1
    gone = set()
    for b in range(B):
        for blk in tables[b][:lens[b]]:
            refs[blk] -= 1
            if refs[blk] == 0:
                gone.add(blk)
    free += sorted(gone)
    ok, copies = [1] * B, []
    for b in range(B):
        if want[b] is None:
            continue
        if not free:
            ok[b] = 0
            for blk in new[b]:
                refs[blk] -= 1
            new[b] = []
            continue
        dst = free.pop()
        refs[dst] = 1
        new[b].append(dst)
        copies.append((b, want[b][0], dst, want[b][1]))
    return new, {k: v for k, v in refs.items() if v}, free, ok, copies
