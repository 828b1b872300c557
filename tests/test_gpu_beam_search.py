"""GPU: beam searches whole: in a cache of just the blocks that they need."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_beam_path import weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("W,G,bs,max_seq_len,max_new", [(4, 4, 16, 128, 40), (8, 2, 4, 70, 33), (3, 5, 1, 40, 9), (2, 1, 16, 100, 1),
                                                        (5, 3, 16, 64, 17)])
def test_a_search_in_its_own_share_of_blocks(cuda, W, G, bs, max_seq_len, max_new):
    """The cache for ``max_new`` tokens holds the prompts once; the search is the one in a cache for any number."""
    from ssd_b200.runtime.beam import BeamSearchDecoder, blocks_per_request

    w = weights("toy-target")
    rng = np.random.default_rng(W)
    longest = max_seq_len - max_new + 1
    prompts = [[int(t) for t in rng.integers(0, w.shape.vocab, n)]
               for n in [longest, max(1, longest // bs * bs - 1), max(1, longest // bs * bs), 1, 2][:G]]
    roomy = BeamSearchDecoder(w, W, G, max_seq_len=max_seq_len, block_size=bs)
    tight = BeamSearchDecoder(w, W, G, max_seq_len=max_seq_len, block_size=bs, max_new=max_new)
    assert tight.pm.num_blocks == G * blocks_per_request(W, max_seq_len, max_new, bs) + 2 <= roomy.pm.num_blocks
    assert W == 1 or max_new > max_seq_len // 2 or tight.pm.num_blocks < roomy.pm.num_blocks
    for new in (max_new, max(1, max_new // 2)):
        assert tight.generate(prompts, new) == roomy.generate(prompts, new)
    # a longer prompt, fewer new tokens
    long = [p + [1] * (max_new - 1) for p in prompts]
    assert tight.generate(long, 1) == roomy.generate(long, 1)
    for dec in (tight, roomy):
        dec.pm.free_rows(0, dec.B)
        assert sorted(dec.pm.free_blocks) == list(range(dec.pm.num_blocks)) and dec.pm.ref_counts == {}
    with pytest.raises(ValueError):
        tight.generate([[1]], max_new + 1)
    for bad in (-1, max_seq_len + 1):
        with pytest.raises(ValueError):
            BeamSearchDecoder(w, W, G, max_seq_len=max_seq_len, block_size=bs, max_new=bad)
