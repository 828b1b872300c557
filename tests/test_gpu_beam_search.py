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


def test_the_engine_takes_as_many_requests_as_fit(cuda, monkeypatch):
    """Bounded by batch_buckets and by the free memory: more prompts go through one after another."""
    import torch

    from ssd_b200 import LLM, DecodeMode, SamplingParams
    from ssd_b200.runtime import beam

    llm = LLM.from_mode(DecodeMode.AR)
    try:
        seen = []
        make = beam.BeamSearchDecoder.__init__

        def spy(self, target, num_beams, requests=1, *args, **kw):
            seen.append(requests)
            make(self, target, num_beams, requests, *args, **kw)

        monkeypatch.setattr(beam.BeamSearchDecoder, "__init__", spy)
        prompts = [[1, 2, 3, 4, 5], [9, 8, 7], [5] * 20, [6, 6], [30, 31, 32], [7]]
        sampling = SamplingParams(max_new_tokens=6, num_beams=4)
        out, metrics = llm.generate(prompts, sampling)
        assert seen == [4] and metrics.total_tokens == 36  # 16 rows a forward
        llm._engine.config.batch_buckets = (1, 3)
        few, _ = llm.generate(prompts, sampling)
        assert seen == [4, 3] and [len(t) for t in few] == [6] * 6
        state = llm._engine.ranks.state
        shape, max_len = state.target_w.shape, 20 + 6 + 2 * 5 + 16
        each = beam.blocks_per_request(4, max_len, 6, 16) * 16 * shape.kv_bytes_per_token(4) + 4 * 4 * shape.vocab
        monkeypatch.setattr(torch.cuda, "memory_reserved", lambda d=None: 0)
        monkeypatch.setattr(torch.cuda, "memory_allocated", lambda d=None: 0)
        for free, want in ((each * 10 // 9 * 2 + 100, 2), (each, 1), (0, 1)):
            monkeypatch.setattr(torch.cuda, "mem_get_info", lambda d=None, f=free: (f, 1 << 37))
            one, _ = llm.generate(prompts, sampling)
            assert seen[-1] == want and [len(t) for t in one] == [6] * 6
    finally:
        llm.shutdown()


@pytest.mark.parametrize("mode,prompts,temperature", [("ar", 2, 0.0), ("sd", 1, 0.0), ("sd", 3, 0.0), ("sd", 2, 0.8), ("ssd", 1, 0.0)])
def test_eos_ends_an_output_in_every_mode(cuda, mode, prompts, temperature):
    from ssd_b200 import LLM, DecodeMode, SamplingParams

    llm = LLM.from_mode(DecodeMode(mode))
    try:
        given = [[1, 2, 3, 4, 5], [9, 8, 7], [5] * 20][:prompts]
        make = lambda **kw: SamplingParams(max_new_tokens=12, temperature=temperature, **kw)  # noqa: E731
        full, _ = llm.generate(given, make())
        assert [len(t) for t in full] == [12] * prompts
        for stop in {full[0][0], full[0][5], full[-1][11]}:
            got, _ = llm.generate(given, make(eos_token_id=stop))
            if temperature == 0:
                assert got == [t[:t.index(stop) + 1] if stop in t else t for t in full]
            for t in got:
                assert stop not in t[:-1] and (len(t) == 12 or t[-1] == stop)
            assert [len(t) for t in llm.generate(given, make(eos_token_id=stop, ignore_eos=True))[0]] == [12] * prompts
        for bad in (dict(eos_token_id=llm._engine.vocab_size), dict(eos_token_id=-1)):
            with pytest.raises(ValueError):
                llm.generate(given, make(**bad))
    finally:
        llm.shutdown()


@pytest.mark.parametrize("mode", ["ar", "sd", "ssd"])
def test_fewer_than_one_beam_is_refused(cuda, mode):
    from ssd_b200 import LLM, DecodeMode, SamplingParams

    llm = LLM.from_mode(DecodeMode(mode))
    try:
        for n in (0, -3):
            with pytest.raises(ValueError):
                llm.generate([[1, 2]], SamplingParams(max_new_tokens=4, num_beams=n))
    finally:
        llm.shutdown()
