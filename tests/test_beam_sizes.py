"""CPU: sizes of the shared-prefix attention at their limits."""

from __future__ import annotations


def test_attention_workspace_of_very_long_contexts():
    """A tile's positions are counted in 32 bits: of contexts of 2^28 positions and more a tile takes fewer sequences, so that
    there are more tiles, and more partial sums."""
    from ssd_b200 import _lib

    size = lambda rows, s: _lib.lib().ssd_shared_prefix_attention_workspace_size(  # noqa: E731
        1, rows, 1, 1, 1, 64, 1 << 16, 1, s)
    # 32 parts of 8 rows of 64 sums, their two numbers, and where they are: 2 tiles may stand in one group of 8 rows
    per_tile = 32 * 8 * (64 * 4 + 8)
    assert size(8, 1 << 20) == 2 * per_tile + 256 and size(8, (1 << 28) - (1 << 16)) == 2 * per_tile + 256
    assert size(8, 1 << 28) == 2 * per_tile + 256     # 7 sequences a tile
    assert size(8, 1 << 29) == 3 * per_tile + 256     # 3
    assert size(8, 1 << 30) == 8 * per_tile + 256     # 1


def test_reorder_refuses_more_columns_than_it_counts():
    """G * max_blocks columns are counted in 32 bits; refused before any address is looked at."""
    from ssd_b200 import _lib

    p = 1 << 20  # an address that no refused call touches

    def call(g, max_blocks):
        return _lib.lib().ssd_page_reorder(None, p, p, max_blocks, p, p, p, 64, p, p, 16, None, p, p, p, g, 1)

    for g, cols in ((1024, (1 << 20) + 1), (2, (1 << 29) + 1), (1, (1 << 30) + 1), (3, 0x7fffffff)):
        assert call(g, cols) == 4
