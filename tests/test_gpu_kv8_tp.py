"""GPU: the 8-bit cache on a tensor-parallel shard, with a group of one on one GPU."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def comm(cuda):
    from ssd_b200.runtime.tensor_parallel import TPComm

    c = TPComm(heap_bytes=64 << 20, max_m=256, max_n=4096, device=cuda)
    yield c
    c.close()


@pytest.mark.parametrize("t", [21, 5, 1])
def test_forward_with_group_of_one_equals_plain(comm, cuda, t):
    from ssd_b200.models.gemma import PRESETS, GemmaRunner, GemmaWeights, allocate_kv_cache

    s = PRESETS["tp-target"]
    w = GemmaWeights.random(s, seed=11, device=cuda, max_pos=512)
    toks = torch.randint(0, s.vocab, (1, t), device=cuda, dtype=torch.int32)
    outs, caches = [], []
    top = comm._top
    for use in (False, True):
        cache = allocate_kv_cache(w, 8, 16, "fp8")
        table = torch.arange(8, dtype=torch.int32, device=cuda)[None]
        r = GemmaRunner(w, 1, 64, 128, comm=comm if use else None)
        lg = comm.alloc((1, t, s.vocab)) if use else torch.empty((1, t, s.vocab), device=cuda)
        for before in (0, t):  # a second call reads what the first has appended
            r.forward(toks, torch.full((1,), before, dtype=torch.int32, device=cuda), cache, table, lg)
        torch.cuda.synchronize()
        outs.append(lg.clone())
        caches.append(cache)
    comm._top = top
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(caches[0].pages.view(torch.uint8), caches[1].pages.view(torch.uint8))
    assert torch.equal(caches[0].scales, caches[1].scales)
    assert comm.status() == 0


def test_decoders_with_group_of_one(comm, cuda):
    from ssd_b200.models.gemma import PRESETS, GemmaWeights
    from ssd_b200.runtime.batched import BatchedSpeculativeDecoder
    from ssd_b200.runtime.speculative import GreedyDecoder, SpeculativeDecoder

    t = GemmaWeights.random(PRESETS["tp-target"], seed=21, device=cuda, max_pos=512)
    prompt = list(range(100, 140))
    top = comm._top
    for make in (lambda c: GreedyDecoder(t, max_seq_len=256, comm=c, kv_cache_dtype="fp8").generate(prompt, 24),
                 lambda c: SpeculativeDecoder(t, t, k=4, max_seq_len=256, comm=c,
                                              kv_cache_dtype="fp8").generate(prompt, 24)[0],
                 lambda c: _batched(BatchedSpeculativeDecoder(t, t, batch=2, k=3, max_seq_len=256, comm=c,
                                                              kv_cache_dtype="fp8"), [prompt, prompt[:9]])):
        plain, group = make(None), make(comm)
        comm._top = top
        assert plain == group
    assert comm.status() == 0


def _batched(dec, prompts):
    first = [dec.admit(i, p) for i, p in enumerate(prompts)]
    return first, [dec.step() for _ in range(4)]


def test_a_rank_reports_waits_that_ran_out(cuda):
    """The status that ends a generate call holds the 8-bit attention's, once."""
    from ssd_b200._lib import lib
    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, paged_kv8_attention
    from ssd_b200.runtime.rank_group import LocalRank

    rank = LocalRank({"target_model_path": None, "draft_model_path": None, "use_toy_model": True, "seed": 0,
                      "draft_seed": 1, "max_model_len": 64, "kv_cache_dtype": "fp8", "local_draft": False,
                      "target_adapter": False}, 0)
    try:
        cache = KV8CacheState.allocate(1, 4, 16, 1, 64)
        table = torch.arange(4, dtype=torch.int32, device=cuda)[None]
        n = torch.full((1,), 40, dtype=torch.int32, device=cuda)
        q = torch.randn((1, 40, 2, 64), device=cuda).bfloat16()
        append_kv8(cache, 0, table, n, q[:, :, :1], q[:, :, :1])
        rank.call("begin")
        lib().ssd_kv8_attention_set_polls(0)
        try:
            paged_kv8_attention(q, cache, 0, table, n)
        finally:
            lib().ssd_kv8_attention_set_polls(-1)
        assert rank.call("end") == [3]
        rank.call("begin")
        assert paged_kv8_attention(q, cache, 0, table, n).isfinite().all()
        assert rank.call("end") == [0]
    finally:
        rank.close()
