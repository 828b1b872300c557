"""Attention of a batch whose rows share long prefixes: beams, branches or samples of one prompt, or requests under
one system prompt.

After ``PageManager.fork_rows`` the rows' tables name the same pages for the shared tokens, and
``paged_verify_attention`` reads those pages once for each row.  ``shared_prefix_attention`` takes the groups of rows
and the lengths of their prefixes, reads a prefix once for all the query rows of a group that fit a tile, and
each row's own positions with them.

bf16 and fp32 caches, head_dim 64, 128 or 256.  Every call runs on the current stream of the cache's device and keeps
nothing of its arguments.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from .._lib import dtype_code, lib
from .kv8_cache import _current_device, _rows, _tables, ints, launch
from .kv_cache import KVCacheState


@lru_cache(maxsize=1024)  # a function of these sizes alone
def _workspace_size(*sizes: int) -> int:
    return lib().ssd_shared_prefix_attention_workspace_size(*sizes)


def shared_prefix_attention(q: torch.Tensor, cache: KVCacheState, layer: int, block_tables: torch.Tensor,
                            seq_lens: torch.Tensor, group_starts: torch.Tensor, prefix_lens: torch.Tensor,
                            q_lens: torch.Tensor | None = None, scale: float | None = None,
                            max_seq_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [B,T,Hq,D] against each row's pages, shared prefixes read once (``ssd_shared_prefix_attention``).

    ``group_starts`` int32 [groups + 1], ascending from 0 to B: rows group_starts[g] .. group_starts[g+1]-1 are group g;
    rows before the first group or behind the last come back as zeros, and a start below one before it counts as that one.
    ``prefix_lens`` int32 [groups]: leading positions in which the group's rows agree, read through the table of its
    first row (0: nothing is shared).  The other arguments and the result are those of ``paged_verify_attention``:
    seq_lens [B] counts cached tokens INCLUDING the new ones, new token t of row b sits at position seq_lens[b] -
    q_lens[b] + t and sees the positions up to it, rows past q_lens[b] come back as zeros.  ``out`` may not be q.
    """
    p = cache.pages
    if len(p.shape) != 6 or p.shape[0] != 2 or not p.is_contiguous():
        raise ValueError("a cache's pages are a contiguous tensor [2, L, NB, BS, Hkv, D]")
    dev = p.get_device()
    _, nl, nb, bs, hkv, hd = p.shape
    shape = q.shape
    if len(shape) != 4 or shape[3] != hd or q.dtype is not p.dtype:
        raise ValueError(f"q must be {p.dtype} [B, T, Hq, {hd}], got {q.dtype} {list(shape)}")
    b, t, hq, _ = shape
    groups = prefix_lens.shape[0] if prefix_lens.dim() == 1 else -1
    q, at = _rows(q, "q", dev)
    tab, cols = _tables(block_tables, b, dev)
    max_seq_len = cols * bs if max_seq_len is None else int(max_seq_len)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {q.dtype} tensor {list(q.shape)} on cuda:{dev}")
    dtype = dtype_code(q.dtype)
    # a workspace of its own for every call: calls on other streams or in captured graphs share nothing
    need = _workspace_size(dtype, b, t, hq, hkv, hd, bs, groups, max_seq_len)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    launch("ssd_shared_prefix_attention", dev, at, p.data_ptr(), dtype, nl, nb, bs, hkv, hd, layer, tab, cols,
           ints(seq_lens, (b,), "seq_lens", dev), ints(q_lens, (b,), "q_lens", dev),
           ints(group_starts, (groups + 1,), "group_starts", dev), ints(prefix_lens, (groups,), "prefix_lens", dev),
           groups, out.data_ptr(), hd ** -0.5 if scale is None else float(scale), b, t, hq, max_seq_len,
           None if ws is None else ws.data_ptr(), need)
    return out


def check_shared_prefix_attention(device=None) -> None:
    """Wait for the current stream of the GPU (None: the current one) and raise if a ``shared_prefix_attention`` there gave
    up a device-side wait since the last check (``ssd_shared_prefix_attention_status``); its unfinished rows are NaN."""
    dev = torch.device("cuda" if device is None else device)
    launch("ssd_shared_prefix_attention_status", _current_device() if dev.index is None else dev.index)
