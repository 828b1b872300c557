"""GPU: the 8-bit cache in the model's forward, the decoders, the engine and the page manager."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _model(dtype, shape, seed=3, max_pos=512):
    from ssd_b200.models.gemma import GemmaWeights

    return GemmaWeights.random(shape, seed=seed, dtype=dtype, max_pos=max_pos)


def _i32(v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_forward_is_the_operators_one_after_another(cuda, kind):
    """One layer: ssd_gemma_forward with an 8-bit cache gives the bits of the operators called in its order --
    embedding, QKV, RoPE + append, attention, O, gate/up, down, norm, head -- over a prompt, a ragged verify step and
    a single token, and leaves the same cache."""
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState, paged_kv8_attention, rope_append_kv8
    from ssd_b200.kernels.ops import embed, linear, rmsnorm
    from ssd_b200.models.gemma import GemmaRunner, GemmaShape

    dt = torch.float32 if kind == "f32" else torch.bfloat16
    s = GemmaShape(1, 256, 8, 2, 64, 1024, 2048)
    w = _model(dt, s)
    b, cols = 2, 8
    table = torch.arange(b * cols, dtype=torch.int32, device="cuda").view(b, cols)
    caches = [KV8CacheState.allocate(1, b * cols, 16, 2, 64) for _ in range(2)]
    run = GemmaRunner(w, b, 8, cols * 16)
    rng = np.random.default_rng(0)
    before = [0, 0]
    for t, ql in ((8, [8, 8]), (8, [8, 5]), (5, [5, 3]), (1, [1, 1])):
        tok = _i32(rng.integers(0, s.vocab, (b, t)))
        logits = torch.empty((b, t, s.vocab), dtype=torch.float32, device="cuda")
        run.forward(tok, _i32(before), caches[0], table, logits, q_lens=_i32(ql))
        after = [x + y for x, y in zip(before, ql)]
        x = embed(tok, w.embed)
        qkv = linear(x, w.w_qkv[0], rownorm_eps=s.eps)
        q = rope_append_kv8(qkv, caches[1], 0, table, _i32(after), 8, w.rope_cos, w.rope_sin, q_lens=_i32(ql))
        a = paged_kv8_attention(q, caches[1], 0, table, _i32(after), q_lens=_i32(ql))
        linear(a.view(b * t, -1), w.w_o[0], "residual", out=x)
        act = linear(x, w.w_gate_up[0], "geglu", rownorm_eps=s.eps)
        linear(act, w.w_down[0], "residual", out=x)
        ref = linear(rmsnorm(x, w.final_norm, s.eps), w.embed, "store_f32").view(b, t, -1)
        for i in range(b):
            assert torch.equal(logits[i, :ql[i]], ref[i, :ql[i]])
        assert torch.equal(caches[0].pages.view(torch.uint8), caches[1].pages.view(torch.uint8))
        assert torch.equal(caches[0].scales, caches[1].scales)
        before = after


def test_forward_stays_near_the_unquantised_cache(cuda):
    """e4m3 rounds K and V by at most 2^-4 of each value: attention outputs, weighted means of V, move by at most
    2^-4 |V| and by the scores' shift; over the toy pair's two layers the logits keep their shape."""
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.kernels.kv_cache import KVCacheState
    from ssd_b200.models.gemma import PRESETS, GemmaRunner

    s = PRESETS["toy-target"]
    w = _model(torch.float32, s)
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    tok = _i32(np.random.default_rng(1).integers(0, s.vocab, (1, 16)))
    out = []
    for cache in (KVCacheState.allocate(2, 4, 16, 1, 64, dtype=torch.float32), KV8CacheState.allocate(2, 4, 16, 1, 64)):
        lg = torch.empty((1, 16, s.vocab), dtype=torch.float32, device="cuda")
        GemmaRunner(w, 1, 16, 64).forward(tok, _i32([0]), cache, table, lg)
        out.append(lg.double())
    # two layers, each rounding K and V by 2^-4: 4 * 2^-4 of the logits' norm is far above what that can do to them
    assert (out[1] - out[0]).norm() <= 4 * 2.0 ** -4 * out[0].norm()
    assert (out[1] - out[0]).norm() > 0


def test_verify_matches_decoding_one_by_one(cuda):
    """k + 1 tokens at once or one after the other: a page's scale may grow at another moment, which only moves values
    among e4m3's subnormals (2^-18 of the page's largest)."""
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.models.gemma import PRESETS, GemmaRunner

    for name, dt in (("toy-target", torch.float32), ("tp-target", torch.bfloat16)):
        s = PRESETS[name]
        w = _model(dt, s)
        table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
        toks = np.random.default_rng(2).integers(0, s.vocab, 21)
        run = GemmaRunner(w, 1, 16, 128)
        outs = []
        for steps in ([5], [1] * 5):
            cache = KV8CacheState.allocate(s.num_layers, 8, 16, s.num_kv_heads, s.head_dim)
            run.forward(_i32(toks[None, :16]), _i32([0]), cache, table, None)
            rows, at = [], 16
            for n in steps:
                lg = torch.empty((1, n, s.vocab), dtype=torch.float32, device="cuda")
                run.forward(_i32(toks[None, at:at + n]), _i32([at]), cache, table, lg)
                rows.append(lg[0])
                at += n
            outs.append(torch.cat(rows).double())
        assert (outs[0] - outs[1]).abs().max() <= 2.0 ** -10 * outs[0].abs().max()


@pytest.mark.parametrize("mode", ["ar", "sd", "ssd"])
def test_engine_runs_on_an_fp8_cache(cuda, mode):
    from ssd_b200 import LLM, SamplingParams

    llm = LLM.from_mode(mode, use_toy_model=True, kv_cache_dtype="fp8", max_model_len=256)
    try:
        prompts = [[5, 6, 7, 8, 9], [100, 101, 102]]
        outs = [llm.generate(prompts, SamplingParams(max_new_tokens=20))[0] for _ in range(2)]
        assert outs[0] == outs[1]
        assert [len(o) for o in outs[0]] == [20, 20]
        assert all(0 <= t < 1024 for o in outs[0] for t in o)
        if mode == "sd":
            one = llm.generate(prompts[:1], SamplingParams(max_new_tokens=20))[0]
            assert len(one[0]) == 20
            hot = llm.generate(prompts, SamplingParams(max_new_tokens=9, temperature=1.0, top_p=0.9))[0]
            assert [len(o) for o in hot] == [9, 9]
    finally:
        llm.shutdown()


def test_engine_refuses_an_unknown_cache_dtype(cuda):
    import torch

    from ssd_b200 import LLM
    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.models.gemma import PRESETS, GemmaRunner, allocate_kv_cache

    with pytest.raises(ValueError):
        LLM.from_mode("ar", use_toy_model=True, kv_cache_dtype="int3")
    w = _model(torch.float32, PRESETS["toy-target"])
    with pytest.raises(ValueError):
        allocate_kv_cache(w, 4, 16, "fp4")
    cache = KV8CacheState.allocate(2, 4, 16, 1, 64)
    with pytest.raises(ValueError):  # pages without their scales
        GemmaRunner(w, 1, 16, 64).forward(_i32([[1]]), _i32([0]), cache.pages, _i32([[0, 1, 2, 3]]), None)


def _filled(pm, cache, lens, rng, hkv, d):
    import torch

    from ssd_b200.kernels.kv8_cache import append_kv8

    b = len(lens)
    pm.allocate_rows(0, b, _i32([0] * b), _i32(lens), None)
    k = torch.tensor(rng.standard_normal((b, max(lens), hkv, d)).astype(np.float32), device="cuda").bfloat16()
    for layer in range(cache.num_layers):
        append_kv8(cache, layer, pm.tables[:b], _i32(lens), k * (layer + 1), k + layer, q_lens=_i32(lens))


@pytest.mark.parametrize("num_tokens", [37, 32, 5])
def test_fork_and_go_on_with_an_8_bit_cache(cuda, num_tokens):
    """Forked rows read as their source does, and appends to one leave the others alone."""
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, gather_kv8
    from ssd_b200.runtime.page_manager import PageManager

    rng = np.random.default_rng(7)
    pm = PageManager(16, 12, max_seqs=4, max_blocks_per_seq=5)
    cache = KV8CacheState.allocate(2, 12, 16, 2, 64)
    _filled(pm, cache, [40], rng, 2, 64)
    ok = pm.fork_rows(0, 1, 3, num_tokens, cache)
    assert ok.tolist() == [1, 1, 1]
    pos = torch.arange(num_tokens, dtype=torch.int32, device="cuda")[None]
    want = [gather_kv8(cache, layer, pm.tables[:1], pos) for layer in range(2)]
    for layer in range(2):
        for row in (1, 2, 3):
            got = gather_kv8(cache, layer, pm.tables[row:row + 1], pos)
            assert torch.equal(got[0], want[layer][0]) and torch.equal(got[1], want[layer][1])
    pm.allocate_rows(1, 1, _i32([num_tokens]), _i32([3]), None)
    big = torch.full((1, 3, 2, 64), 1000.0, device="cuda")
    append_kv8(cache, 1, pm.tables[1:2], _i32([num_tokens + 3]), big, big)  # needs a larger scale than the trunk's
    for row in (0, 2, 3):
        got = gather_kv8(cache, 1, pm.tables[row:row + 1], pos)
        assert torch.equal(got[0], want[1][0]) and torch.equal(got[1], want[1][1])
    new = gather_kv8(cache, 1, pm.tables[1:2], _i32([list(range(num_tokens, num_tokens + 3))]))[0]
    assert ((new.float() - 1000).abs() <= 1000 * 2.0 ** -4).all()


def test_fork_without_a_free_block(cuda):
    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.runtime.page_manager import PageManager

    rng = np.random.default_rng(8)
    pm = PageManager(16, 4, max_seqs=4, max_blocks_per_seq=4)
    cache = KV8CacheState.allocate(1, 4, 16, 1, 64)
    _filled(pm, cache, [40], rng, 1, 64)
    assert pm.fork_rows(0, 1, 3, 40, cache).tolist() == [1, 0, 0]  # three blocks held, one left


def test_compact_then_decode_on(cuda):
    """Sequences finish, the pool is compacted, a smaller cache takes its used blocks: attention reads the same, and
    allocation, append and attention go on."""
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState, append_kv8, paged_kv8_attention
    from ssd_b200.kernels.page_moves import copy_pages
    from ssd_b200.runtime.page_manager import PageManager

    rng = np.random.default_rng(9)
    lens = [60, 33, 90, 16, 47, 5]
    nb, hkv, d = 40, 2, 64
    pm = PageManager(16, nb, max_seqs=6, max_blocks_per_seq=8)
    cache = KV8CacheState.allocate(2, nb, 16, hkv, d)
    _filled(pm, cache, lens, rng, hkv, d)
    pm.free_rows(0, 2)
    pm.free_rows(3, 1)
    live = [2, 4, 5]
    q = torch.randn((6, 2, 4, d), device="cuda").bfloat16()
    sl = torch.zeros(6, dtype=torch.int32, device="cuda")
    sl[live] = _i32([lens[i] for i in live])
    want = [paged_kv8_attention(q, cache, layer, pm.tables, sl) for layer in range(2)]
    remap = pm.compact(cache)
    used = sum(-(-lens[i] // 16) for i in live)
    tabs = pm.tables.cpu().numpy()
    held = sorted(int(x) for i in live for x in tabs[i, : -(-lens[i] // 16)])
    assert held == list(range(used)) and len(pm.free_blocks) == nb - used
    assert sorted(x for x in remap.tolist() if x >= 0) == list(range(used))
    assert pm.free_blocks[-1] == used and pm.ref_counts == {i: 1 for i in range(used)}
    for layer in range(2):
        assert torch.equal(paged_kv8_attention(q, cache, layer, pm.tables, sl), want[layer])
    small = KV8CacheState.allocate(2, used + 4, 16, hkv, d)
    ids = torch.arange(used, dtype=torch.int32, device="cuda")
    copy_pages(cache, ids, ids, dst_cache=small)
    assert torch.equal(paged_kv8_attention(q, small, 1, pm.tables, sl), want[1])
    before = sl[2:3].clone()
    pm.allocate_rows(2, 1, before, _i32([20]), None)
    k = torch.randn((1, 20, hkv, d), device="cuda").bfloat16()
    append_kv8(cache, 0, pm.tables[2:3], before + 20, k, k)
    assert paged_kv8_attention(q[2:3], cache, 0, pm.tables[2:3], before + 20).isfinite().all()


def test_adapter_branches_on_an_8_bit_cache(cuda):
    import torch

    from ssd_b200.models.gemma import PRESETS
    from ssd_b200.models.gemma_adapter import GemmaAdapter

    w = _model(torch.float32, PRESETS["toy-draft"])
    ad = GemmaAdapter(w, max_model_len=128, max_branches=3, kv_cache_dtype="fp8")
    out = ad.draft_branches([3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3, 2, 3], [[7], [8, 9], [10]], 4)
    assert [len(o) for o in out] == [4, 4, 4] and all(0 <= t < 1024 for o in out for t in o)
    spec, logits = ad.draft_speculate([3, 1, 4, 1, 5], 3)
    assert len(spec) == 3 and logits.shape == (3, 1024)


def test_forward_refuses_another_models_cache(cuda):
    import torch

    from ssd_b200.kernels.kv8_cache import KV8CacheState
    from ssd_b200.kernels.kv_cache import KVCacheState
    from ssd_b200.models.gemma import GemmaRunner, GemmaShape

    s = GemmaShape(2, 256, 8, 2, 64, 1024, 2048)
    run = GemmaRunner(_model(torch.bfloat16, s), 1, 4, 64)
    table, tok = _i32([[0, 1, 2, 3]]), _i32([[1, 2]])
    good = KV8CacheState.allocate(2, 4, 16, 2, 64)
    run.forward(tok, _i32([0]), good, table, None)
    for bad in (KV8CacheState.allocate(1, 4, 16, 2, 64), KV8CacheState.allocate(2, 4, 16, 1, 64),
                KV8CacheState.allocate(2, 4, 16, 2, 128), KVCacheState.allocate(1, 4, 16, 2, 64), good.pages):
        with pytest.raises(ValueError):
            run.forward(tok, _i32([0]), bad, table, None)
