"""Paged KV cache held in 8 bits: half the bytes of the bf16 cache to store and to read.

Layout: ``pages[2, num_layers, num_blocks, block_size, num_kv_heads, head_dim]`` e4m3 (as
``kv_cache.KVCacheState``, plane 0 = K, plane 1 = V) and ``scales[2, num_layers, num_blocks,
num_kv_heads]`` fp32: an element is its e4m3 value times the scale of its page and KV head.  Scales
are powers of two, 2^-118 to 2^120 (any other value counts as the one at its exponent), so a page whose
scale 2^e grows as rows are appended is rewritten without a second rounding (values below 2^-6 2^e
aside).  A scale keeps to the largest row its page has held since its first row was appended, a rejected
draft's included: a value x is off by at most 2^-4 |x| + 2^-9 2^e.

Rows enter by ``append_kv8`` / ``rope_append_kv8`` at the end of each sequence, in the order of its
positions: a block's scale follows what has been appended to it, so there is no write at arbitrary
slots.  ``paged_kv8_attention`` takes the arguments of ``paged_verify_attention``.

head_dim 64, 128 or 256; queries and rows in bf16 or fp32.  Every call runs on the current stream of
the cache's device and keeps nothing of its arguments.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from functools import lru_cache

import torch

from .._lib import check, dtype_code, lib


@dataclass(frozen=True)
class KV8CacheState:
    """Paged e4m3 cache and its scales, [2, L, num_blocks, block_size, Hkv, D] and [2, L, num_blocks, Hkv]."""

    pages: torch.Tensor
    scales: torch.Tensor
    block_size: int
    # layers, blocks, block size, KV heads, head dim
    dims: tuple = field(init=False, repr=False, compare=False)

    def __post_init__(self) -> None:
        p, s = self.pages, self.scales
        shape = p.shape
        if (p.dtype is not torch.float8_e4m3fn or s.dtype is not torch.float32 or len(shape) != 6
                or not p.is_contiguous() or not s.is_contiguous() or s.get_device() != p.get_device()):
            raise ValueError("an 8-bit cache is contiguous e4m3 pages [2, L, NB, BS, Hkv, D] and fp32 scales on one GPU")
        two, nl, nb, bs, hkv, hd = shape
        if two != 2 or bs != self.block_size or s.shape != (2, nl, nb, hkv):
            raise ValueError(f"scales {tuple(s.shape)} and block_size {self.block_size} do not fit pages {tuple(p.shape)}")
        object.__setattr__(self, "dims", (nl, nb, bs, hkv, hd))

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


# the current stream's handle without the Stream object around it, and the current device without the module's lazy
# initialisation (a tensor on a GPU has seen to that): a microsecond of each call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_int32 = torch.int32


def launch(name: str, dev: int, *args) -> None:
    """Call a C entry point on the current stream of GPU ``dev``; raise for its status."""
    if dev < 0:
        raise ValueError(f"{name}: the tensors must be on a GPU")
    fn = getattr(lib(), name)
    if dev == _current_device():
        rc = fn(_raw_stream(dev), *args)
    else:
        with torch.cuda.device(dev):
            rc = fn(_raw_stream(dev), *args)
    if rc:
        check(rc, name)


def ints(t: torch.Tensor | None, shape: tuple, what: str, dev: int) -> int | None:
    """Pointer of a contiguous int32 array of the shape on GPU ``dev`` (None for None)."""
    if t is None:
        return None
    if t.dtype is _int32 and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{what} must be a contiguous int32 tensor {list(shape)} on cuda:{dev}, got "
                     f"{t.dtype} {list(t.shape)} on {t.device}")


def _cache(cache: KV8CacheState) -> tuple:
    """(device index, pages and scales: pointers, layers, blocks, block size, KV heads, head dim)."""
    p = cache.pages
    return (p.get_device(), p.data_ptr(), cache.scales.data_ptr(), *cache.dims)


def _rows(t: torch.Tensor, what: str, dev: int) -> tuple[torch.Tensor, int]:
    """The rows as the kernels read them (contiguous, 16 bytes at a time), and their pointer."""
    if t.get_device() != dev:
        raise ValueError(f"{what} is on {t.device}, the cache on cuda:{dev}")
    if not t.is_contiguous():
        t = t.contiguous()
    at = t.data_ptr()
    if at & 15:
        t = t.clone()
        at = t.data_ptr()
    return t, at


def _tables(t: torch.Tensor, b: int, dev: int) -> tuple[int, int]:
    """(pointer, columns) of block tables [b, max_blocks]."""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"block_tables must be [{b}, max_blocks], got {list(shape)}")
    m = shape[1]
    return ints(t, (b, m), "block_tables", dev), m


def append_kv8(cache: KV8CacheState, layer: int, block_tables: torch.Tensor, seq_lens: torch.Tensor,
               k: torch.Tensor, v: torch.Tensor, q_lens: torch.Tensor | None = None) -> KV8CacheState:
    """Quantise k/v [B,T,Hkv,D] into each sequence's pages (``ssd_kv8_append``).

    Token t < q_lens[b] (None: T) of row b goes to position seq_lens[b] - q_lens[b] + t; ``seq_lens``
    counts the new tokens, as for ``paged_kv8_attention``.  A page whose first row is among the new
    ones starts over; in any other page the earlier rows keep their values.  A page that is written
    belongs to one sequence (fork a shared one first, ``PageManager.fork_rows``).
    """
    dev, pages, scales, nl, nb, bs, hkv, hd = _cache(cache)
    shape = k.shape
    if len(shape) != 4 or shape[2] != hkv or shape[3] != hd or v.shape != shape or v.dtype != k.dtype:
        raise ValueError(f"k and v must be [B, T, {hkv}, {hd}] of one dtype, got {list(shape)} and {list(v.shape)}")
    b, t = shape[0], shape[1]
    k, k_at = _rows(k, "k", dev)
    v, v_at = _rows(v, "v", dev)
    tab, cols = _tables(block_tables, b, dev)
    launch("ssd_kv8_append", dev, pages, scales, nl, nb, bs, hkv, hd, layer, tab, cols,
           ints(seq_lens, (b,), "seq_lens", dev), ints(q_lens, (b,), "q_lens", dev), k_at, v_at,
           dtype_code(k.dtype), b, t)
    return cache


def rope_append_kv8(qkv: torch.Tensor, cache: KV8CacheState, layer: int, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, num_heads: int, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                    q_lens: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """RoPE on the q and k parts of qkv [B*T, (Hq+2Hkv)*D], k and v appended to the cache
    (``ssd_kv8_rope_append``); returns the rotated q [B, T, Hq, D] (zeros for t >= q_lens[b])."""
    dev, pages, scales, nl, nb, bs, hkv, hd = _cache(cache)
    b = block_tables.shape[0]
    width = (num_heads + 2 * hkv) * hd
    if qkv.dim() != 2 or qkv.shape[1] != width or (qkv.shape[0] % b if b else qkv.shape[0]):
        raise ValueError(f"qkv must be [B*T, {width}] for {b} sequences, got {list(qkv.shape)}")
    t = qkv.shape[0] // b if b else 0
    max_pos = rope_cos.shape[0]
    for tab, name in ((rope_cos, "rope_cos"), (rope_sin, "rope_sin")):
        if (tab.dtype is not torch.float32 or tab.get_device() != dev or tab.shape != (max_pos, hd // 2)
                or not tab.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 tensor [positions, {hd // 2}] on cuda:{dev}")
    qkv, at = _rows(qkv, "qkv", dev)
    if out is None:
        out = qkv.new_empty((b, t, num_heads, hd))
    elif (out.shape != (b, t, num_heads, hd) or out.dtype != qkv.dtype or out.get_device() != dev
          or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {qkv.dtype} tensor [{b}, {t}, {num_heads}, {hd}] on cuda:{dev}")
    tab, cols = _tables(block_tables, b, dev)
    launch("ssd_kv8_rope_append", dev, at, out.data_ptr(), pages, scales, dtype_code(qkv.dtype), nl, nb,
           bs, num_heads, hkv, hd, layer, tab, cols, ints(seq_lens, (b,), "seq_lens", dev),
           ints(q_lens, (b,), "q_lens", dev), rope_cos.data_ptr(), rope_sin.data_ptr(), max_pos, b, t)
    return out


def gather_kv8(cache: KV8CacheState, layer: int, block_tables: torch.Tensor, positions: torch.Tensor,
               dtype=torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V rows [B, N, Hkv, D] of positions [B, N] (-1: zeros), as the values the cache holds (``ssd_kv8_gather``)."""
    dev, pages, scales, nl, nb, bs, hkv, hd = _cache(cache)
    if positions.dim() != 2:
        raise ValueError(f"positions must be [B, N], got {list(positions.shape)}")
    b, n = positions.shape
    k, v = cache.scales.new_empty((2, b, n, hkv, hd), dtype=dtype).unbind(0)
    tab, cols = _tables(block_tables, b, dev)
    launch("ssd_kv8_gather", dev, pages, scales, nl, nb, bs, hkv, hd, layer, tab, cols,
           ints(positions, (b, n), "positions", dev), k.data_ptr(), v.data_ptr(), dtype_code(dtype), b, n)
    return k, v


@lru_cache(maxsize=1024)  # a function of these sizes alone
def _workspace_size(dtype: int, b: int, t: int, hq: int, hkv: int, hd: int, max_seq_len: int) -> int:
    return lib().ssd_kv8_attention_workspace_size_for(dtype, b, t, hq, hkv, hd, max_seq_len)


def paged_kv8_attention(q: torch.Tensor, cache: KV8CacheState, layer: int, block_tables: torch.Tensor,
                        seq_lens: torch.Tensor, q_lens: torch.Tensor | None = None, scale: float | None = None,
                        max_seq_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [B,T,Hq,D] against each sequence's pages (``ssd_kv8_attention``).

    Arguments as ``paged_verify_attention``: seq_lens [B] counts cached tokens INCLUDING the new
    ones; new token t of sequence b sits at position seq_lens[b] - q_lens[b] + t.  Rows past
    q_lens[b] come back as zeros.  For T up to 8 a query's bits do not depend on how many new tokens
    stand beside it; they may differ between batch sizes and values of ``max_seq_len``, by which the
    context is split.
    """
    dev, pages, scales, nl, nb, bs, hkv, hd = _cache(cache)
    shape = q.shape
    if len(shape) != 4 or shape[3] != hd:
        raise ValueError(f"q must be [B, T, Hq, {hd}], got {list(shape)}")
    b, t, hq, _ = shape
    q, at = _rows(q, "q", dev)
    tab, cols = _tables(block_tables, b, dev)
    max_seq_len = cols * bs if max_seq_len is None else int(max_seq_len)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {q.dtype} tensor {list(q.shape)} on cuda:{dev}")
    # a workspace of its own for every call: calls on other streams or in captured graphs share nothing
    dtype = dtype_code(q.dtype)
    need = _workspace_size(dtype, b, t, hq, hkv, hd, max_seq_len)
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    launch("ssd_kv8_attention", dev, at, pages, scales, dtype, nl, nb, bs, hkv, hd, layer, tab,
           cols, ints(seq_lens, (b,), "seq_lens", dev), ints(q_lens, (b,), "q_lens", dev), out.data_ptr(),
           hd ** -0.5 if scale is None else float(scale), b, t, hq, max_seq_len, None if ws is None else ws.data_ptr(), need)
    return out


def check_kv8_attention(device=None) -> None:
    """Wait for the current stream of the GPU (None: the current one) and raise if a ``paged_kv8_attention`` there gave
    up a device-side wait since the last check (``ssd_kv8_attention_status``); its unfinished rows are NaN."""
    dev = torch.device("cuda" if device is None else device)
    launch("ssd_kv8_attention_status", _current_device() if dev.index is None else dev.index)
