"""GPU: the shared-prefix attention over lists of more positions than 32 bits count."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_prefix_attention import bound, check, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_eight_rows_of_a_quarter_of_a_thousand_million_positions(cuda, dtype):
    """Rows of 2^28 positions and some more, of which a page or two are there: each row is what it is over these alone."""
    import torch

    from ssd_b200.kernels.kv_cache import KVCacheState
    from ssd_b200.kernels.prefix_attention import shared_prefix_attention

    bs, cols, B, D = 1 << 16, (1 << 12) + 1, 8, 64
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    cache = KVCacheState(pages=torch.randn((2, 1, B, bs, 1, D), generator=g, device="cuda").to(dt), block_size=bs)
    q = torch.randn((B, 1, 1, D), generator=g, device="cuda").to(dt)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ends = [7 + 13 * b for b in range(B)]  # positions of the last page that a row sees
    tables = np.full((B, cols), -1, np.int32)
    for b in range(B):
        tables[b, -1] = b
    got = shared_prefix_attention(q, cache, 0, i32(tables), i32([bs * (cols - 1) + n for n in ends]), i32([0, B]), i32([0]))
    small = dict(q=q, cache=cache, layer=0, block_tables=i32([[b] for b in range(B)]), seq_lens=i32(ends),
                 group_starts=i32([0, B]), prefix_lens=i32([0]), q_lens=None)
    want, size, slack = oracle(small)
    check(small)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound(small, want, size, slack)).all()
