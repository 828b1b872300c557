"""CPU: the 8-bit cache's and the page moves' argument checks, and the oracle they are tested against."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8 as o


def test_e4m3_rounding_matches_the_cast():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-448, 448, 4000), rng.standard_normal(4000), 2.0 ** rng.uniform(-14, 8, 4000),
                        o.e4m3_values()[~np.isnan(o.e4m3_values())], [0.0, 2.0 ** -10, 3 * 2.0 ** -10, 448, 17.0]])
    x = x.astype(np.float32)
    cast = torch.tensor(x).to(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(o.e4m3_round(x), cast)
    byte = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(o.e4m3_values(), byte)


def test_scale_is_the_smallest_power_of_two():
    for amax in (448.0, 448.0001, 1.0, 0.875, 0.876, 1e-30, 3e38, 0.0):
        e = o.scale_exponent(np.array([[[amax, -amax / 3, np.inf, np.nan]]]))[0]
        assert amax <= 448 * 2.0 ** float(e)
        assert e == o.MIN_EXP or amax > 448 * 2.0 ** float(e - 1)


def test_appending_in_pieces_holds_the_same_values():
    """Powers of two: rows appended one by one under a growing scale end as rows appended at once (values that
    stay above e4m3's subnormals)."""
    rng = np.random.default_rng(1)
    k = (1 + rng.random((16, 2, 64))) * np.exp2(rng.integers(-3, 4, (16, 1, 1)))
    one, exp1 = np.zeros((2, 1, 16, 2, 64)), np.zeros((2, 1, 2), np.int64)
    many, exp2 = one.copy(), exp1.copy()
    o.append(one, exp1, [0], 16, k, -k)
    for i in range(16):
        o.append(many, exp2, [0], i + 1, k[i:i + 1], -k[i:i + 1])
    np.testing.assert_array_equal(exp1, exp2)
    np.testing.assert_array_equal(one, many)


def test_c_abi_refusals():
    from ssd_b200 import _lib

    so = _lib.lib()
    P = 4096  # an aligned stand-in pointer: every call below is refused on the host

    def append(pages=P, scales=P, nl=2, nb=8, bs=16, hkv=2, d=64, layer=0, tab=P, mb=4, sl=P, k=P, v=P, dt=0, b=1, t=1):
        return so.ssd_kv8_append(None, pages, scales, nl, nb, bs, hkv, d, layer, tab, mb, sl, None, k, v, dt, b, t)

    assert append(b=0) == 0 and append(t=0) == 0
    for bad in (dict(pages=None), dict(scales=None), dict(k=None), dict(v=None), dict(tab=None), dict(sl=None),
                dict(layer=2), dict(layer=-1), dict(bs=0), dict(nb=0), dict(hkv=0), dict(mb=0), dict(dt=2),
                dict(b=-1), dict(t=-1)):
        assert append(**bad) == 1, bad
    for bad in (dict(d=96), dict(d=512), dict(k=P + 2), dict(pages=P + 8), dict(nb=1 << 28), dict(b=1 << 20, t=1 << 20)):
        assert append(**bad) == 4, bad

    def rope(qkv=P, q=P, d=64, cos=P, hq=4, mp=64, b=1, t=1):
        return so.ssd_kv8_rope_append(None, qkv, q, P, P, 0, 2, 8, 16, hq, 2, d, 0, P, 4, P, None, cos, P, mp, b, t)

    assert rope(b=0) == 0
    assert rope(qkv=None) == rope(q=None) == rope(cos=None) == rope(hq=0) == rope(mp=0) == 1
    assert rope(d=32) == rope(qkv=P + 4) == 4

    def gather(pos=P, k=P, n=1, d=64, dt=0):
        return so.ssd_kv8_gather(None, P, P, 2, 8, 16, 2, d, 0, P, 4, pos, k, P, dt, 1, n)

    assert gather(n=0) == 0
    assert gather(pos=None) == gather(k=None) == gather(dt=7) == gather(n=-1) == 1
    assert gather(d=48) == gather(k=P + 2) == 4

    def attn(q=P, out=P, hq=4, hkv=2, d=64, sl=P, b=1, t=1, mx=64, ws=P, nbytes=1 << 40, dt=0, mb=4):
        return so.ssd_kv8_attention(None, q, P, P, dt, 2, 8, 16, hkv, d, 0, P, mb, sl, None, out, 0.1, b, t, hq, mx, ws,
                                    nbytes)

    assert attn(b=0) == 0
    for bad in (dict(hq=3), dict(q=None), dict(out=None), dict(sl=None), dict(mx=0), dict(mx=65), dict(dt=3),
                dict(t=-1)):
        assert attn(**bad) == 1, bad
    assert attn(d=80) == attn(q=P + 2) == attn(b=70000) == 4
    assert attn(mb=63, mx=1000, ws=None) == attn(mb=63, mx=1000, nbytes=0) == 5  # split contexts
    assert so.ssd_kv8_attention_workspace_size(1, 5, 4, 3, 64, 1000) == 0
    assert so.ssd_kv8_attention_workspace_size(1, 5, 4, 2, 64, 1000) > 0
    assert so.ssd_kv8_attention_workspace_size(1, 5, 4, 2, 64, 64) == 0  # one split: nothing to join

    def copy(src=P, ss=None, dst=P, ds=None, planes=4, nbytes=64, sc=0, sid=P, st=1, did=P, n=1):
        return so.ssd_page_copy(None, src, ss, 8, dst, ds, 8, planes, nbytes, sc, sid, st, did, 1, n, None)

    assert copy(n=0) == 0
    for bad in (dict(src=None), dict(dst=None), dict(planes=0), dict(nbytes=0), dict(sc=2), dict(sid=None),
                dict(did=None), dict(st=-1), dict(n=-1)):
        assert copy(**bad) == 1, bad
    assert copy(nbytes=(1 << 31) + 16) == 4

    def compact(nb=8, out=P, tab=P, tab_out=P, lens=P, mb=4, rows=1, draft=None, drows=0):
        return so.ssd_page_compact(None, P, P, P, nb, out, P, P, P, P, P, P, tab, tab_out, lens, mb, rows, draft, P, P,
                                   4, drows)

    for bad in (dict(nb=0), dict(out=None), dict(tab=None), dict(tab_out=None), dict(lens=None), dict(mb=0),
                dict(rows=-1), dict(drows=1), dict(drows=-1)):
        assert compact(**bad) == 1, bad


def test_python_refusals():
    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, paged_kv8_attention
    from ssd_b200.kernels.page_moves import compact_pages, copy_pages

    cache = KV8CacheState.allocate(1, 4, 16, 2, 64, device="cpu")
    assert cache.num_blocks == 4 and cache.num_layers == 1
    tab, lens = torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    k = torch.zeros((1, 1, 2, 64))
    with pytest.raises(ValueError):  # no CPU implementation
        append_kv8(cache, 0, tab, lens, k, k)
    with pytest.raises(ValueError):
        paged_kv8_attention(k, cache, 0, tab, lens)
    with pytest.raises(ValueError):
        copy_pages(cache, torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        compact_pages([], tab, lens, lens, lens, lens)


def test_sizes_past_the_kernels_integers_are_refused():
    """Limits that keep 32-bit positions, rows and pieces in range: 4 (unsupported), before anything is launched."""
    from ssd_b200._lib import lib

    so, P, big = lib(), 4096, 1 << 30

    def attn(nb=8, bs=16, hkv=2, b=1, t=1, hq=4, mb=4, mx=64, ws=P):
        return so.ssd_kv8_attention(None, P, P, P, 0, 1, nb, bs, hkv, 64, 0, P, mb, P, None, P, 0.1, b, t, hq, mx, ws,
                                    1 << 62)

    assert attn(t=big, hq=1 << 20, hkv=1) == 4          # more row groups than a grid has
    assert attn(mb=(1 << 31) - 1, bs=1, mx=big + 1) == 4
    assert attn(mb=63, mx=1000, ws=P + 8) == 4
    assert attn(nb=1, bs=(1 << 20) + 1) == 4
    assert so.ssd_kv8_attention_workspace_size(1, 1, 4, 2, 64, big + 1) == 0
    assert so.ssd_kv8_append(None, P, P, 1, 1, (1 << 20) + 1, 2, 64, 0, P, 4, P, None, P, P, 0, 1, 1) == 4


def test_pages_in_8_bits_do_not_move_without_their_scales():
    from types import SimpleNamespace

    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.kernels.page_moves import copy_pages

    cache = KV8CacheState.allocate(1, 4, 16, 2, 64, device="cpu")
    ids = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="scales"):
        copy_pages(SimpleNamespace(pages=cache.pages, block_size=16), ids, ids)
