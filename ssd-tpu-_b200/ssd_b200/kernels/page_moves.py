"""Moves of whole pages: copies inside a cache or between two, and compaction of a fragmented pool.

Both work on ``KVCacheState`` (bf16, fp32) and ``KV8CacheState`` (pages and scales).  Nothing
synchronises: the ids, the plan and its length stay on the device.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .._lib import check, lib, ptr
from .kv8_cache import _ints, _stream, on_device


def _pool(cache):
    """(pages, scales or None, bytes of a page in one plane, scales of a page, planes)."""
    p = cache.pages
    s = getattr(cache, "scales", None)
    if p.dim() != 6 or not p.is_contiguous() or not p.is_cuda:
        raise ValueError("a cache's pages are a contiguous CUDA tensor [2, L, NB, BS, Hkv, D]")
    if s is not None and (s.dtype != torch.float32 or s.shape != (*p.shape[:3], p.shape[4]) or s.device != p.device
                          or not s.is_contiguous()):
        raise ValueError(f"scales do not fit pages {tuple(p.shape)}")
    return p, s, p.shape[3] * p.shape[4] * p.shape[5] * p.element_size(), 0 if s is None else p.shape[4]


def _copy(cache, dst_cache, src: int, src_step: int, dst: int, dst_step: int, n: int, count: int | None) -> None:
    p, s, nbytes, nscales = _pool(cache)
    dp, ds, dbytes, dscales = _pool(dst_cache)
    if (dp.dtype != p.dtype or dp.shape[:2] != p.shape[:2] or dp.shape[3:] != p.shape[3:] or dscales != nscales
            or dp.device != p.device):
        raise ValueError(f"pages {tuple(dp.shape)} {dp.dtype} cannot take copies of pages {tuple(p.shape)} {p.dtype}")
    check(lib().ssd_page_copy(_stream(p.device), ptr(p), ptr(s), p.shape[2], ptr(dp), ptr(ds), dp.shape[2],
                              2 * p.shape[1], nbytes, nscales, src, src_step, dst, dst_step, n, count),
          "ssd_page_copy")


def copy_pages(cache, src: torch.Tensor, dst: torch.Tensor, dst_cache=None):
    """Copy page ``src[i]`` to page ``dst[i]`` in every layer, K and V (``ssd_page_copy``).

    ``src`` and ``dst``: int32 [n] on the cache's device (any stride; an expanded ``src`` copies one
    page to many); pairs with an id out of range (-1) are skipped.  ``dst_cache``: another cache of
    the same page shape to copy into.  Within one cache a page may not be both source and
    destination, nor a destination twice.  Returns the cache written to.
    """
    dev = cache.pages.device
    for t, name in ((src, "src"), (dst, "dst")):
        if t.dtype != torch.int32 or t.dim() != 1 or t.device != dev or t.shape != src.shape:
            raise ValueError(f"{name} must be an int32 tensor [n] on {dev}")
    out = cache if dst_cache is None else dst_cache
    with on_device(dev):
        _copy(cache, out, src.data_ptr(), src.stride(0), dst.data_ptr(), dst.stride(0), src.shape[0], None)
    return out


@dataclass
class Compaction:
    """State of a pool after ``compact_pages``: what the arguments became, and the blocks' new ids."""

    tables: torch.Tensor
    ref_counts: torch.Tensor
    free_list: torch.Tensor
    free_top: torch.Tensor
    remap: torch.Tensor                       # [num_blocks]: new id of a block in use, -1 of a free one
    draft_tables: torch.Tensor | None = None


def compact_pages(cache, tables: torch.Tensor, lens: torch.Tensor, ref_counts: torch.Tensor,
                  free_list: torch.Tensor, free_top: torch.Tensor, draft_tables: torch.Tensor | None = None,
                  draft_lens: torch.Tensor | None = None, *, inplace: bool = False) -> Compaction:
    """Move the blocks in use to the front of the pool: blocks 0 .. U-1 hold what the U used blocks held.

    ``cache`` (one cache, or a sequence of caches that share the pool's block ids) is changed in
    place; ``tables`` [rows, max_blocks] with ``lens`` [rows], ``ref_counts`` [num_blocks],
    ``free_list`` [num_blocks] and ``free_top`` [1] (the arrays of ``PageManager``) come back as new
    tensors, or are changed too with ``inplace``.  Every block that is not on the free list counts as
    in use.  The fewest pages move: the k-th used block at U or above to the k-th free one below U.
    ``ssd_page_compact``, ``ssd_page_remap`` and ``ssd_page_copy``.
    """
    caches = list(cache) if isinstance(cache, (list, tuple)) else [cache]
    if not caches:
        raise ValueError("compact_pages wants a cache")
    dev = caches[0].pages.device
    nb = caches[0].pages.shape[2]
    for c in caches:
        if c.pages.shape[2] != nb or c.pages.device != dev:
            raise ValueError("the caches of one pool have the same blocks and device")
    if (draft_tables is None) != (draft_lens is None):
        raise ValueError("draft_tables and draft_lens go together")
    fl, ft = _ints(free_list, (nb,), "free_list", dev), _ints(free_top, (1,), "free_top", dev)
    rc = _ints(ref_counts, (nb,), "ref_counts", dev)
    pairs = [(tables, lens, "tables")] + ([] if draft_tables is None else [(draft_tables, draft_lens, "draft_tables")])
    for t, n, name in pairs:
        _ints(t, (n.shape[0], -1), name, dev)
        _ints(n, (t.shape[0],), "lens of " + name, dev)
    half = max(1, nb // 2)
    buf = torch.empty(nb + 2 * half + 1, dtype=torch.int32, device=dev)
    remap, src, dst, count = buf[:nb], buf[nb:nb + half], buf[nb + half:nb + 2 * half], buf[nb + 2 * half:]
    new = (lambda t: t) if inplace else torch.empty_like
    free_list_out, free_top_out, ref_out = new(free_list), new(free_top), new(ref_counts)
    outs = [new(t) for t, _, _ in pairs]
    with on_device(dev):
        st = _stream(dev)
        check(lib().ssd_page_compact(st, fl, ft, rc, nb, ptr(free_list_out), ptr(free_top_out), ptr(ref_out),
                                     ptr(remap), ptr(src), ptr(dst), ptr(count)), "ssd_page_compact")
        for (t, n, _), o in zip(pairs, outs):
            check(lib().ssd_page_remap(st, ptr(t), ptr(o), ptr(n), t.shape[1], t.shape[0], ptr(remap), nb),
                  "ssd_page_remap")
        for c in caches:
            _copy(c, c, ptr(src), 1, ptr(dst), 1, nb // 2, ptr(count))
    return Compaction(outs[0], ref_out, free_list_out, free_top_out, remap, outs[1] if len(outs) > 1 else None)
