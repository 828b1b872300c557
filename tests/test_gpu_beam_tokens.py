"""GPU: the tokens of whole beam searches, against a search over plain forwards, and on a tensor-parallel shard."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_beam_path import Plain, plain_search, weights

pytestmark = pytest.mark.gpu

# toy logits agree within 1e-4 whichever way they are computed, so a log-probability does within 2e-4
PER_TOKEN = 2e-4


@pytest.mark.parametrize("W,alpha,ends", [(2, 0.0, False), (4, 0.0, False), (4, 0.7, True), (8, 1.0, True), (3, 0.0, True)])
def test_tokens_equal_the_plain_search(cuda, W, alpha, ends):
    """As far as no two candidates near the border come closer than their scores' error, the tokens have to be the same: each
    prompt's search is compared at the longest length at which that holds.  A score over n tokens is off by PER_TOKEN n, its
    rank by PER_TOKEN n / n^alpha, so two ranks by twice the largest of these."""
    from ssd_b200.runtime.beam import BeamSearchDecoder

    w = weights("toy-target")
    rng = np.random.default_rng(100 + W)
    plain, most, compared, ended = Plain(w), 6, [], 0
    for n in [int(x) for x in rng.integers(1, 50, 24)]:
        prompt = [int(t) for t in rng.integers(0, w.shape.vocab, n)]
        eos = None
        if ends:  # a token that the second beam has in its middle, so that beams do finish
            eos = plain_search(plain, prompt, W, most, -1, alpha)[0][1][0][2]
        for steps in range(most, 0, -1):
            want, gap = plain_search(plain, prompt, W, steps, -1 if eos is None else eos, alpha)
            if gap > 2 * PER_TOKEN * steps ** (1 - alpha):  # (alpha is 1 at most: the longest has the largest)
                break
        else:
            continue
        got, = BeamSearchDecoder(w, W, max_seq_len=64, length_penalty=alpha, eos_token_id=eos).generate([prompt], steps)
        assert [t for t, _ in got] == [t for t, _ in want]
        assert np.allclose([s for _, s in got], [s for _, s in want], atol=PER_TOKEN * steps, rtol=0)
        compared.append(steps)
        ended += any(t[-1] == eos for t, _ in got)
    # (how many are compared is the plain search's doing alone: the toy's candidates lie close, those of many beams closest)
    assert len(compared) >= 8 and max(compared) >= 2 and (not ends or ended >= 1), (compared, ended)
    assert W > 4 or (sum(compared) >= 24 and max(compared) >= 3), compared


@pytest.mark.parametrize("W,G", [(8, 2), (5, 3), (16, 1)])
def test_every_beams_score_is_its_tokens_log_probability(cuda, W, G):
    from ssd_b200.runtime.beam import BeamSearchDecoder

    w = weights("toy-target")
    rng = np.random.default_rng(W)
    prompts = [[int(t) for t in rng.integers(0, w.shape.vocab, n)] for n in (33, 7, 48)[:G]]
    steps, plain = 19, Plain(w)
    for prompt, found in zip(prompts, BeamSearchDecoder(w, W, G, max_seq_len=80, max_new=steps).generate(prompts, steps)):
        assert len(found) == W and len({tuple(t) for t, _ in found}) == W
        for tokens, score in found:
            assert len(tokens) == steps
            total = 0.0
            for i, t in enumerate(tokens):
                x = plain(prompt + tokens[:i]).astype(np.float64)
                total += x[t] - x.max() - np.log(np.exp(x - x.max()).sum())
            assert abs(total - score) <= PER_TOKEN * steps


@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_search_with_a_tensor_parallel_group_of_one(cuda, kv):
    """The logits gathered by the group's LM head, in its buffers: the same beams and scores as without a group."""
    from ssd_b200.models.gemma import PRESETS, GemmaWeights
    from ssd_b200.runtime.beam import BeamSearchDecoder
    from ssd_b200.runtime.tensor_parallel import TPComm

    t = GemmaWeights.random(PRESETS["tp-target"], seed=21, device=cuda, max_pos=512)
    prompts = [list(range(100, 140)), [7, 8, 9]]
    comm = TPComm(heap_bytes=64 << 20, max_m=256, max_n=4096, device=cuda)
    try:
        top = comm._top
        make = lambda c: BeamSearchDecoder(t, 4, 2, max_seq_len=128, comm=c, kv_cache_dtype=kv, length_penalty=0.6,  # noqa: E731
                                           eos_token_id=5, max_new=20).generate(prompts, 20)
        want, got = make(None), make(comm)
        comm._top = top
        assert got == want
        assert comm.status() == 0
    finally:
        comm.close()
