"""Paged KV cache held in 8 bits: half the bytes of the bf16 cache to store and to read.

Layout: ``pages[2, num_layers, num_blocks, block_size, num_kv_heads, head_dim]`` e4m3 (as
``kv_cache.KVCacheState``, plane 0 = K, plane 1 = V) and ``scales[2, num_layers, num_blocks,
num_kv_heads]`` fp32: an element is its e4m3 value times the scale of its page and KV head.  Scales
are powers of two, so a page whose scale grows as rows are appended is rewritten without a second
rounding (values below 2^-14 of the page's largest aside).

Rows enter by ``append_kv8`` / ``rope_append_kv8`` at the end of each sequence, in the order of its
positions: a block's scale follows what has been appended to it, so there is no write at arbitrary
slots.  ``paged_kv8_attention`` takes the arguments of ``paged_verify_attention``.

head_dim 64, 128 or 256; queries and rows in bf16 or fp32.  Every call runs on the current stream of
the cache's device and keeps nothing of its arguments.
"""

from __future__ import annotations

import contextlib
from dataclasses import dataclass

import torch

from .._lib import check, dtype_code, lib, ptr


@dataclass
class KV8CacheState:
    """Paged e4m3 cache and its scales, [2, L, num_blocks, block_size, Hkv, D] and [2, L, num_blocks, Hkv]."""

    pages: torch.Tensor
    scales: torch.Tensor
    block_size: int

    @classmethod
    def allocate(cls, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 device="cuda") -> "KV8CacheState":
        pages = torch.zeros((2, num_layers, num_blocks, block_size, num_kv_heads, head_dim),
                            dtype=torch.float8_e4m3fn, device=device)
        scales = torch.ones((2, num_layers, num_blocks, num_kv_heads), dtype=torch.float32, device=device)
        return cls(pages=pages, scales=scales, block_size=block_size)

    @property
    def num_blocks(self) -> int:
        return self.pages.shape[2]

    @property
    def num_layers(self) -> int:
        return self.pages.shape[1]


_NO_GUARD = contextlib.nullcontext()


def on_device(dev: torch.device):
    """A context with ``dev`` current (nothing to do when it already is, the usual case)."""
    return _NO_GUARD if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _cache_dims(cache: KV8CacheState):
    p, s = cache.pages, cache.scales
    if (p.dtype != torch.float8_e4m3fn or s.dtype != torch.float32 or p.dim() != 6 or not p.is_contiguous()
            or not s.is_contiguous() or not p.is_cuda or s.device != p.device):
        raise ValueError("an 8-bit cache is contiguous e4m3 pages [2, L, NB, BS, Hkv, D] and fp32 scales on one GPU")
    two, nl, nb, bs, hkv, hd = p.shape
    if two != 2 or bs != cache.block_size or s.shape != (2, nl, nb, hkv):
        raise ValueError(f"scales {tuple(s.shape)} and block_size {cache.block_size} do not fit pages {tuple(p.shape)}")
    return nl, nb, bs, hkv, hd


def _ints(t: torch.Tensor | None, shape: tuple, what: str, dev: torch.device) -> int | None:
    """Pointer of an int32 device array of the shape (-1: any size)."""
    if t is None:
        return None
    if (t.dtype != torch.int32 or t.device != dev or t.dim() != len(shape)
            or any(n >= 0 and n != m for n, m in zip(shape, t.shape)) or not t.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous int32 tensor {list(shape)} on {dev}, got "
                         f"{t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, what: str, dev: torch.device) -> torch.Tensor:
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, the cache on {dev}")
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t  # the kernels move 16 bytes at a time


def append_kv8(cache: KV8CacheState, layer: int, block_tables: torch.Tensor, seq_lens: torch.Tensor,
               k: torch.Tensor, v: torch.Tensor, q_lens: torch.Tensor | None = None) -> KV8CacheState:
    """Quantise k/v [B,T,Hkv,D] into each sequence's pages (``ssd_kv8_append``).

    Token t < q_lens[b] (None: T) of row b goes to position seq_lens[b] - q_lens[b] + t; ``seq_lens``
    counts the new tokens, as for ``paged_kv8_attention``.  A page whose first row is among the new
    ones starts over; in any other page the earlier rows keep their values.
    """
    nl, nb, bs, hkv, hd = _cache_dims(cache)
    dev = cache.pages.device
    if k.dim() != 4 or k.shape[2:] != (hkv, hd) or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"k and v must be [B, T, {hkv}, {hd}] of one dtype, got {list(k.shape)} and {list(v.shape)}")
    b, t = k.shape[:2]
    k, v = _rows(k, "k", dev), _rows(v, "v", dev)
    with on_device(dev):
        check(lib().ssd_kv8_append(_stream(dev), ptr(cache.pages), ptr(cache.scales), nl, nb, bs, hkv, hd, layer,
                                   _ints(block_tables, (b, -1), "block_tables", dev), block_tables.shape[1],
                                   _ints(seq_lens, (b,), "seq_lens", dev), _ints(q_lens, (b,), "q_lens", dev),
                                   ptr(k), ptr(v), dtype_code(k.dtype), b, t), "ssd_kv8_append")
    return cache


def rope_append_kv8(qkv: torch.Tensor, cache: KV8CacheState, layer: int, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, num_heads: int, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                    q_lens: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """RoPE on the q and k parts of qkv [B*T, (Hq+2Hkv)*D], k and v appended to the cache
    (``ssd_kv8_rope_append``); returns the rotated q [B, T, Hq, D] (zeros for t >= q_lens[b])."""
    nl, nb, bs, hkv, hd = _cache_dims(cache)
    dev = cache.pages.device
    b = block_tables.shape[0]
    if qkv.dim() != 2 or qkv.shape[1] != (num_heads + 2 * hkv) * hd or (b == 0) != (qkv.shape[0] == 0) or (
            b and qkv.shape[0] % b):
        raise ValueError(f"qkv must be [B*T, {(num_heads + 2 * hkv) * hd}] for {b} sequences, got {list(qkv.shape)}")
    t = qkv.shape[0] // b if b else 0
    for tab, name in ((rope_cos, "rope_cos"), (rope_sin, "rope_sin")):
        if (tab.dtype != torch.float32 or tab.device != dev or tab.shape != (rope_cos.shape[0], hd // 2)
                or not tab.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 tensor [positions, {hd // 2}] on {dev}")
    qkv = _rows(qkv, "qkv", dev)
    if out is None:
        out = torch.empty((b, t, num_heads, hd), dtype=qkv.dtype, device=dev)
    elif (out.shape != (b, t, num_heads, hd) or out.dtype != qkv.dtype or out.device != dev
          or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {qkv.dtype} tensor [{b}, {t}, {num_heads}, {hd}] on {dev}")
    with on_device(dev):
        check(lib().ssd_kv8_rope_append(_stream(dev), ptr(qkv), ptr(out), ptr(cache.pages), ptr(cache.scales),
                                        dtype_code(qkv.dtype), nl, nb, bs, num_heads, hkv, hd, layer,
                                        _ints(block_tables, (b, -1), "block_tables", dev), block_tables.shape[1],
                                        _ints(seq_lens, (b,), "seq_lens", dev), _ints(q_lens, (b,), "q_lens", dev),
                                        ptr(rope_cos), ptr(rope_sin), rope_cos.shape[0], b, t), "ssd_kv8_rope_append")
    return out


def gather_kv8(cache: KV8CacheState, layer: int, block_tables: torch.Tensor, positions: torch.Tensor,
               dtype=torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V rows [B, N, Hkv, D] of positions [B, N] (-1: zeros), as the values the cache holds (``ssd_kv8_gather``)."""
    nl, nb, bs, hkv, hd = _cache_dims(cache)
    dev = cache.pages.device
    b, n = positions.shape
    k = torch.empty((b, n, hkv, hd), dtype=dtype, device=dev)
    v = torch.empty((b, n, hkv, hd), dtype=dtype, device=dev)
    with on_device(dev):
        check(lib().ssd_kv8_gather(_stream(dev), ptr(cache.pages), ptr(cache.scales), nl, nb, bs, hkv, hd, layer,
                                   _ints(block_tables, (b, -1), "block_tables", dev), block_tables.shape[1],
                                   _ints(positions, (b, n), "positions", dev), ptr(k), ptr(v), dtype_code(dtype), b,
                                   n), "ssd_kv8_gather")
    return k, v


def paged_kv8_attention(q: torch.Tensor, cache: KV8CacheState, layer: int, block_tables: torch.Tensor,
                        seq_lens: torch.Tensor, q_lens: torch.Tensor | None = None, scale: float | None = None,
                        max_seq_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [B,T,Hq,D] against each sequence's pages (``ssd_kv8_attention``).

    Arguments as ``paged_verify_attention``: seq_lens [B] counts cached tokens INCLUDING the new
    ones; new token t of sequence b sits at position seq_lens[b] - q_lens[b] + t.  Rows past
    q_lens[b] come back as zeros.
    """
    nl, nb, bs, hkv, hd = _cache_dims(cache)
    dev = cache.pages.device
    if q.dim() != 4 or q.shape[3] != hd:
        raise ValueError(f"q must be [B, T, Hq, {hd}], got {list(q.shape)}")
    b, t, hq, _ = q.shape
    if max_seq_len is None:
        max_seq_len = block_tables.shape[1] * bs
    if scale is None:
        scale = 1.0 / float(hd) ** 0.5
    q = _rows(q, "q", dev)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {q.dtype} tensor {list(q.shape)} on {dev}")
    with on_device(dev):
        # a workspace of its own for every call: calls on other streams or in captured graphs share nothing
        ws = torch.empty(lib().ssd_kv8_attention_workspace_size(b, t, hq, hkv, hd, int(max_seq_len)),
                         dtype=torch.uint8, device=dev)
        check(lib().ssd_kv8_attention(_stream(dev), ptr(q), ptr(cache.pages), ptr(cache.scales), dtype_code(q.dtype),
                                      nl, nb, bs, hkv, hd, layer, _ints(block_tables, (b, -1), "block_tables", dev),
                                      block_tables.shape[1], _ints(seq_lens, (b,), "seq_lens", dev),
                                      _ints(q_lens, (b,), "q_lens", dev), ptr(out), float(scale), b, t, hq,
                                      int(max_seq_len), ptr(ws), ws.numel()), "ssd_kv8_attention")
    return out

