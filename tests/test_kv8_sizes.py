"""CPU: what calls over the 8-bit cache ask for."""

from __future__ import annotations


def test_workspace_goes_by_the_type():
    """Prompts of thousands of bf16 rows are not split and need no workspace, whatever fp32 would take."""
    from ssd_b200._lib import SSD_DTYPE_BF16, SSD_DTYPE_F32, lib

    so = lib()
    size, either = so.ssd_kv8_attention_workspace_size_for, so.ssd_kv8_attention_workspace_size
    for shape in ((4, 2048, 16, 16, 256, 8192), (1, 1500, 16, 16, 256, 8192)):
        assert size(SSD_DTYPE_BF16, *shape) == 0
        assert size(SSD_DTYPE_F32, *shape) > 1 << 29
    for shape in ((1, 5, 4, 2, 64, 1000), (8, 5, 16, 16, 256, 4096), (4, 64, 8, 1, 256, 8192), (1, 1, 8, 1, 256, 137)):
        assert either(*shape) == max(size(d, *shape) for d in (SSD_DTYPE_BF16, SSD_DTYPE_F32))
    assert size(2, 1, 5, 4, 2, 64, 1000) == size(0, 1, 5, 4, 3, 64, 1000) == size(0, 1, 5, 4, 2, 64, (1 << 30) + 1) == 0


def test_batches_of_nothing_have_no_addresses():
    """An empty tensor's pointer is NULL: B = 0 and T = 0 do nothing all the same."""
    from ssd_b200._lib import lib

    so, P = lib(), 4096
    for b, t, table, rows in ((0, 3, None, None), (0, 0, None, None), (2, 0, P, None)):
        assert so.ssd_kv8_append(None, P, P, 2, 8, 16, 2, 64, 0, table, 4, table, None, rows, rows, 0, b, t) == 0
        assert so.ssd_kv8_rope_append(None, rows, rows, P, P, 0, 2, 8, 16, 4, 2, 64, 0, table, 4, table, None, P, P, 64, b,
                                      t) == 0
        assert so.ssd_kv8_gather(None, P, P, 2, 8, 16, 2, 64, 0, table, 4, rows, rows, rows, 0, b, t) == 0
        assert so.ssd_kv8_attention(None, rows, P, P, 0, 2, 8, 16, 2, 64, 0, table, 4, table, None, rows, 0.1, b, t, 4, 64,
                                    None, 0) == 0
    # with sequences, their arrays have to be there
    assert so.ssd_kv8_append(None, P, P, 2, 8, 16, 2, 64, 0, None, 4, P, None, None, None, 0, 2, 0) == 1
    assert so.ssd_kv8_attention(None, P, P, P, 0, 2, 8, 16, 2, 64, 0, P, 4, None, None, P, 0.1, 1, 1, 4, 64, None, 0) == 1


def test_compaction_in_place_refuses_tables_that_share_entries():
    """Also where only some rows are the same memory; views side by side are fine (and refused for want of a GPU)."""
    import pytest
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.kernels.page_moves import compact_pages

    cache = KV8CacheState.allocate(1, 8, 16, 1, 64, device="cpu")
    z = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    base = z(6, 4)
    for a, b, why in ((base[:3], base[2:], "share"), (base[1:5], base[2:3], "share"), (base[:3], base[3:], "on a GPU")):
        with pytest.raises(ValueError, match=why):
            compact_pages(cache, a, z(a.shape[0]), z(8), z(8), z(1), b, z(b.shape[0]), inplace=True)
