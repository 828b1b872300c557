"""Moves of whole pages: copies inside a cache or between two, and compaction of a fragmented pool.

Both work on ``KVCacheState`` (bf16, fp32) and ``KV8CacheState`` (pages and scales).  Nothing
synchronises: the ids, the plan and its length stay on the device.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .kv8_cache import KV8CacheState, ints, launch

_MAX_PAGE = 1 << 31  # bytes of a page in one plane (``ssd_page_copy``)


def _pool(cache) -> tuple:
    """(device, pages, scales or None: pointers, blocks, planes, bytes of a page in one plane, scales of a page, rest)."""
    p = cache.pages
    shape = p.shape
    if len(shape) != 6 or shape[0] != 2 or not p.is_contiguous():
        raise ValueError("a cache's pages are a contiguous tensor [2, L, NB, BS, Hkv, D]")
    _, nl, nb, bs, hkv, hd = shape
    kv8 = isinstance(cache, KV8CacheState)  # its scales fit: it has looked
    if not kv8 and p.dtype is torch.float8_e4m3fn:
        raise ValueError("8-bit pages move as a KV8CacheState: they mean nothing without the scales")
    return (p.get_device(), p.data_ptr(), cache.scales.data_ptr() if kv8 else None, nb, 2 * nl,
            bs * hkv * hd * p.element_size(), hkv if kv8 else 0, (p.dtype, bs, hkv, hd))


def _copy(src: tuple, dst: tuple, src_ids: int, src_step: int, dst_ids: int, dst_step: int, n: int,
          count: int | None) -> None:
    if dst is not src and (dst[0] != src[0] or dst[4:] != src[4:]):
        raise ValueError("the caches' devices, layers or page shapes differ")
    dev, p, s, nb, planes, nbytes, nscales, _ = src
    launch("ssd_page_copy", dev, p, s, nb, dst[1], dst[2], dst[3], planes, nbytes, nscales, src_ids, src_step, dst_ids,
           dst_step, n, count)


def copy_pages(cache, src: torch.Tensor, dst: torch.Tensor, dst_cache=None):
    """Copy page ``src[i]`` to page ``dst[i]`` in every layer, K and V (``ssd_page_copy``).

    ``src`` and ``dst``: int32 [n] on the cache's device (any stride; an expanded ``src`` copies one
    page to many); pairs with an id out of range (-1) are skipped.  ``dst_cache``: another cache of
    the same page shape to copy into.  Within one cache a page may not be both source and
    destination, nor a destination twice.  Returns the cache written to.
    """
    pool = _pool(cache)
    n = src.shape[0] if src.dim() == 1 else -1
    for t, name in ((src, "src"), (dst, "dst")):
        if t.dtype is not torch.int32 or t.get_device() != pool[0] or t.shape != (n,):
            raise ValueError(f"{name} must be an int32 tensor [n] on cuda:{pool[0]}, got {t.dtype} {list(t.shape)} on {t.device}")
    out = cache if dst_cache is None else dst_cache
    _copy(pool, pool if out is cache else _pool(out), src.data_ptr(), src.stride(0), dst.data_ptr(), dst.stride(0), n,
          None)
    return out


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (a, b))
    return max(a0, b0) < min(a1, b1)


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
    ``ssd_page_compact`` and ``ssd_page_copy``.
    """
    pools = [_pool(c) for c in cache] if isinstance(cache, (list, tuple)) else [_pool(cache)]
    if not pools:
        raise ValueError("compact_pages wants a cache")
    dev, nb = pools[0][0], pools[0][3]
    if any(p[0] != dev or p[3] != nb for p in pools):
        raise ValueError("the caches of one pool have the same blocks and device")
    if any(p[5] > _MAX_PAGE for p in pools):  # before the tables change: the copies would be refused
        raise ValueError(f"a page of one plane may hold {_MAX_PAGE} bytes at most")
    if (draft_tables is None) != (draft_lens is None):
        raise ValueError("draft_tables and draft_lens go together")
    if free_list.dtype is not torch.int32:
        raise ValueError(f"free_list must be int32, got {free_list.dtype}")
    if tables.dim() != 2 or (draft_tables is not None and draft_tables.dim() != 2):
        raise ValueError("tables are [rows, max_blocks]")
    if inplace and draft_tables is not None and _overlap(tables, draft_tables):
        raise ValueError("tables and draft_tables share memory: in place, entries would be mapped twice")
    half = max(1, nb // 2)
    work = free_list.new_empty((nb + 2 * half + 1,))  # new ids; the moves' sources, targets, number
    remap = work[:nb]
    src = work.data_ptr() + 4 * nb
    dst, count = src + 4 * half, src + 8 * half
    if inplace:
        out = Compaction(tables, ref_counts, free_list, free_top, remap, draft_tables)
    else:
        new = torch.empty_like
        out = Compaction(new(tables), new(ref_counts), new(free_list), new(free_top), remap,
                         None if draft_tables is None else new(draft_tables))
    drafts = (None, None, None, 0, 0)
    if draft_tables is not None:
        rows, cols = draft_tables.shape
        drafts = (ints(draft_tables, (rows, cols), "draft_tables", dev), out.draft_tables.data_ptr(),
                  ints(draft_lens, (rows,), "draft_lens", dev), cols, rows)
    rows, cols = tables.shape
    launch("ssd_page_compact", dev, ints(free_list, (nb,), "free_list", dev), ints(free_top, (1,), "free_top", dev),
           ints(ref_counts, (nb,), "ref_counts", dev), nb, out.free_list.data_ptr(), out.free_top.data_ptr(),
           out.ref_counts.data_ptr(), remap.data_ptr(), src, dst, count, ints(tables, (rows, cols), "tables", dev),
           out.tables.data_ptr(), ints(lens, (rows,), "lens", dev), cols, rows, *drafts)
    for p in pools:
        _copy(p, p, src, 1, dst, 1, nb // 2, count)
    return out
