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


def _peak(num_beams, prompt, max_new, block_size, rng, apart):
    """Blocks in use at most while beams follow random parents, or (``apart``) each goes on for itself, which shares least:
    tables as page lists, as ``PageManager`` keeps them."""
    import numpy as np

    from oracle import beams

    W, pages = num_beams, -(-prompt // block_size)
    supply = iter(range(pages, 1 << 30))
    tables = [list(range(pages))] + [[] for _ in range(W - 1)]
    refs = {b: 1 for b in range(pages)}
    free, peak, held = [], pages, [prompt] + [0] * (W - 1)
    for step in range(max_new - 1):
        # blocks that nobody holds are taken first; new ones only where the list is empty
        free = free + [next(supply) for _ in range(2 * W)]
        parents = rng.integers(0, W, (1, W)) if step else np.zeros((1, W), int)
        if step and (apart or rng.random() < 0.3):
            parents[:] = rng.permutation(W)
        tables, refs, free, ok, _ = beams.reorder(tables, [len(t) for t in tables], refs, free, parents, held, block_size)
        assert all(ok)
        held = [prompt + step] * W
        for t in tables:
            for _ in range(-(-(held[0] + 1) // block_size) - len(t)):
                b = free.pop()
                t.append(b)
                refs[b] = 1
        held = [h + 1 for h in held]
        peak = max(peak, len(refs))
    return peak


def test_a_requests_blocks_suffice():
    """No search holds more blocks than its share of the pool, and the worst prompts hold about as many."""
    import numpy as np

    from ssd_b200.runtime.beam import blocks_per_request

    rng = np.random.default_rng(0)
    for W, bs, max_seq_len, max_new in [(4, 16, 64, 20), (3, 1, 12, 5), (1, 4, 30, 9), (8, 4, 40, 40), (2, 16, 50, 1),
                                        (5, 3, 31, 2), (4, 5, 60, 17)]:
        most = 0
        for prompt in range(1, max_seq_len + 1):
            new = min(max_new, max_seq_len - prompt + 1)
            most = max(most, _peak(W, prompt, new, bs, rng, True))
            if prompt % 3 == 0:
                most = max(most, _peak(W, prompt, new, bs, rng, False),
                           _peak(W, prompt, int(rng.integers(1, new + 1)), bs, rng, True))
        bound = blocks_per_request(W, max_seq_len, max_new, bs)
        assert most <= bound <= most + W + 1, (W, bs, max_seq_len, max_new, most, bound)


def test_the_prompts_blocks_are_held_once():
    from ssd_b200.runtime.beam import blocks_per_request

    # 4 beams of 64 new tokens behind up to 1437 prompt tokens: 4 times 5 blocks, and the prompt's
    assert blocks_per_request(4, 1500, 64, 16) == 94 - 5 + 4 * 5
    assert blocks_per_request(4, 1500, 1500, 16) == 4 * 94
    assert blocks_per_request(1, 1500, 64, 16) == 94
    assert blocks_per_request(4, 10, 0, 1) == 10 and blocks_per_request(4, 10, 1, 1) == 10


def test_requests_go_by_the_memory_that_is_there():
    from ssd_b200.models.gemma import PRESETS
    from ssd_b200.runtime.beam import blocks_per_request, requests_that_fit

    s = PRESETS["gemma-7b"]
    fit = lambda free, elem=2: requests_that_fit(s, elem, 4, 64, 1500, 64, 16, free)  # noqa: E731
    each = blocks_per_request(4, 1500, 64, 16) * 16 * 2 * 2 * 28 * 16 * 256 + 4 * 4 * 256000
    assert fit(180 << 30) == 64
    assert fit(10 * each) == 10 and fit(10 * each - 1) == 9 and fit(10 * each, 1) in (19, 20)
    assert fit(0) == 1 and fit(each // 2) == 1


def test_attention_refuses_its_queries_as_output():
    """Rows that V's infinities reach are worked out again from q, after others of the row's warps have written theirs."""
    from ssd_b200 import _lib

    p = 1 << 20  # an aligned address that no refused call touches

    def call(out, ws):
        return _lib.lib().ssd_shared_prefix_attention(None, p, p, 0, 2, 64, 16, 2, 64, 1, p, 8, p, None, p, p, 2, out, 0.1, 4,
                                                      2, 8, 128, ws, 0 if ws is None else 1 << 40)

    assert call(p, 4 * p) == 1 and call(2 * p, None) == 5
