"""GPU: beam search as a user runs it: forward over shared prefixes, selection and re-ordered pages together."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import beams

pytestmark = pytest.mark.gpu


def weights(preset, seed=3):
    import torch

    from ssd_b200.models.gemma import PRESETS, GemmaWeights

    dtype = torch.float32 if preset.startswith("toy") else torch.bfloat16
    return GemmaWeights.random(PRESETS[preset], seed=seed, dtype=dtype)


class Plain:
    """Last-token logits of whole sequences, each prefilled alone: no shared pages, no beams."""

    def __init__(self, w, max_len=256):
        import torch

        from ssd_b200.kernels.ops import max_tokens_per_forward
        from ssd_b200.models.gemma import GemmaRunner, allocate_kv_cache

        self.w, self.torch = w, torch
        self.chunk = min(16, max_tokens_per_forward(w.dtype))
        self.cache = allocate_kv_cache(w, max_len // 16 + 1, 16)
        self.table = torch.arange(max_len // 16 + 1, dtype=torch.int32, device="cuda")[None]
        self.runner = GemmaRunner(w, 1, 16, max_len)
        self.lg = torch.empty((1, w.shape.vocab), device="cuda")

    def __call__(self, seq):
        t = self.torch
        for c in range(0, len(seq), self.chunk):
            part = t.tensor([seq[c:c + self.chunk]], dtype=t.int32, device="cuda")
            self.runner.forward(part, t.tensor([c], dtype=t.int32, device="cuda"), self.cache, self.table, self.lg,
                                last_only=True)
        return self.lg[0].cpu().numpy().copy()


def plain_search(logits_of, prompt, W, steps, eos, alpha):
    """(beams as (tokens, score, length), smallest gap of ranks among the best W + 1 of any step)."""
    V = None
    seqs, scores, lengths, done = [[]] * W, np.full((1, W), -np.inf), np.zeros((1, W), int), np.zeros((1, W), int)
    scores[0, 0] = 0
    gap = np.inf
    for _ in range(steps):
        x = None
        for w in range(W):
            if scores[0, w] > -np.inf and not done[0, w]:
                row = logits_of(prompt + seqs[w])
                if x is None:
                    V = len(row)
                    x = np.full((1, W, V), 0.0, np.float32)
                x[0, w] = row
        if x is None:
            break
        # one place more, for the gap behind the last beam
        pad = np.concatenate([x, np.zeros((1, 1, V), np.float32)], 1)
        more = beams.beam_select(pad, np.append(scores, [[-np.inf]], 1), np.append(lengths, [[0]], 1),
                                 np.append(done, [[0]], 1), eos, alpha)
        rank = more[0][0] / np.maximum(more[3][0], 1) ** alpha
        rank = rank[np.isfinite(rank)]
        if len(rank) > 1:
            gap = min(gap, np.min(-np.diff(rank)))
        s, p, t, n, f = (a[:, :W] for a in more)
        seqs = [seqs[p[0, w]] + ([int(t[0, w])] if not done[0, p[0, w]] else []) if p[0, w] >= 0 else [] for w in range(W)]
        scores, lengths, done = s, n, f
    return [(seqs[w], scores[0, w]) for w in range(W) if scores[0, w] > -np.inf], gap


@pytest.mark.parametrize("W,eos,alpha,lens", [(4, None, 0.0, [5, 37, 16]), (3, 7, 0.6, [20, 33]), (8, None, 1.0, [48, 3]),
                                              (1, None, 0.0, [12]), (5, 11, 0.0, [9])])
def test_toy_equals_plain_search(cuda, W, eos, alpha, lens):
    from ssd_b200.runtime.beam import BeamSearchDecoder

    w = weights("toy-target")
    rng = np.random.default_rng(W)
    prompts = [[int(t) for t in rng.integers(0, w.shape.vocab, n)] for n in lens]
    steps = 12
    dec = BeamSearchDecoder(w, W, requests=min(len(prompts) + 1, 16 // W), max_seq_len=128, length_penalty=alpha, eos_token_id=eos)
    got = []
    for i in range(0, len(prompts), dec.G):
        got += dec.generate(prompts[i:i + dec.G], steps)
    plain = Plain(w)
    for prompt, found in zip(prompts, got):
        want, gap = plain_search(plain, prompt, W, steps, -1 if eos is None else eos, alpha)
        # toy logits agree within 1e-4 whichever way they are computed, so scores do within 2e-4 a token
        assert np.allclose([s for _, s in found], [s for _, s in want], atol=2e-4 * steps)
        if gap > 4e-4 * steps:
            assert [t for t, _ in found] == [t for t, _ in want]
    dec.pm.free_rows(0, dec.B)
    assert len(dec.pm.free_blocks) == dec.pm.num_blocks and dec.pm.ref_counts == {}


def test_one_beam_is_the_greedy_stream(cuda):
    from ssd_b200.runtime.beam import BeamSearchDecoder
    from ssd_b200.runtime.speculative import GreedyDecoder

    w = weights("toy-target")
    prompt = [3, 1, 4, 1, 5, 9, 2, 6]
    want = GreedyDecoder(w, max_seq_len=128).generate(prompt, 20)
    (tokens, _), = BeamSearchDecoder(w, 1, max_seq_len=128).generate([prompt], 20)[0]
    assert tokens == want


@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_bf16_scores_are_the_tokens_log_probabilities(cuda, kv):
    """A bf16 model (tensor-core attention over shared pages, or an 8-bit cache): every beam's score is the sum of its
    tokens' log-probabilities under plain forwards, to the models' rounding: bf16 logits move by 2e-2 at this depth
    (5e-2 with 8-bit keys and values), a log-probability by twice that."""
    from ssd_b200.models.gemma import PRESETS
    from ssd_b200.runtime.beam import BeamSearchDecoder

    preset = next(p for p in PRESETS if not p.startswith("toy") and PRESETS[p].num_layers <= 4)
    w = weights(preset)
    rng = np.random.default_rng(1)
    prompts = [[int(t) for t in rng.integers(0, w.shape.vocab, n)] for n in (70, 33)]
    steps = 9
    dec = BeamSearchDecoder(w, 4, requests=2, max_seq_len=160, kv_cache_dtype=kv)
    got = dec.generate(prompts, steps)
    plain = Plain(w)
    for prompt, found in zip(prompts, got):
        assert len(found) == 4 and len({tuple(t) for t, _ in found}) == 4
        assert [s for _, s in found] == sorted((s for _, s in found), reverse=True)
        for tokens, score in found[:2]:
            total = 0.0
            for i, t in enumerate(tokens):
                x = plain(prompt + tokens[:i]).astype(np.float64)
                total += x[t] - x.max() - np.log(np.exp(x - x.max()).sum())
            assert abs(total - score) <= (4e-2 if kv == "auto" else 1e-1) * steps
    again = dec.generate(prompts, steps)
    assert again == got


def test_engine(cuda):
    from ssd_b200 import LLM, DecodeMode, SamplingParams
    from ssd_b200.runtime.beam import BeamSearchDecoder

    llm = LLM.from_mode(DecodeMode.AR)
    try:
        prompts = [[1, 2, 3, 4, 5], [9, 8, 7], [5] * 20, [6, 6], [30, 31, 32]]
        out, metrics = llm.generate(prompts, SamplingParams(max_new_tokens=10, num_beams=4, length_penalty=0.7))
        assert metrics.total_tokens == sum(len(o) for o in out) == 50
        dec = BeamSearchDecoder(llm._engine.ranks.state.target_w, 4, 4, max_seq_len=128, length_penalty=0.7)
        best = [b[0][0] for b in dec.generate(prompts[:4], 10) + dec.generate(prompts[4:], 10)]
        assert out == best
        stop = out[0][3]
        short, _ = llm.generate(prompts[:1], SamplingParams(max_new_tokens=10, num_beams=4, eos_token_id=stop))
        assert len(short[0]) <= 10 and stop not in short[0][:-1]
        long, _ = llm.generate(prompts[:1], SamplingParams(max_new_tokens=10, num_beams=4, eos_token_id=stop, ignore_eos=True))
        assert len(long[0]) == 10
        assert llm.generate([], SamplingParams(num_beams=4))[0] == []
        with pytest.raises(ValueError):
            llm.generate(prompts, SamplingParams(num_beams=4, temperature=0.5))
        with pytest.raises(ValueError):
            llm.generate(prompts, SamplingParams(num_beams=17))     # 17 rows: more than an fp32 forward takes
        with pytest.raises(ValueError):
            llm.generate(prompts, SamplingParams(num_beams=2, max_new_tokens=100000))
    finally:
        llm.shutdown()
    sd = LLM.from_mode(DecodeMode.SD)
    try:
        with pytest.raises(ValueError):
            sd.generate([[1, 2]], SamplingParams(num_beams=2))
    finally:
        sd.shutdown()


def test_decoder_refusals(cuda):
    from ssd_b200.runtime.beam import BeamSearchDecoder

    w = weights("toy-target")
    for kw in (dict(num_beams=0), dict(num_beams=33), dict(num_beams=4, requests=5), dict(num_beams=2, requests=0),
               dict(num_beams=2, eos_token_id=w.shape.vocab)):
        with pytest.raises(ValueError):
            BeamSearchDecoder(w, **kw)
    dec = BeamSearchDecoder(w, 2, requests=2, max_seq_len=32)
    for prompts, n in (([], 4), ([[1]] * 3, 4), ([[1], []], 4), ([[1] * 30], 10)):
        with pytest.raises(ValueError):
            dec.generate(prompts, n)
    assert dec.generate([[1, 2]], 0) == [[([], 0.0)]]
    assert len(dec.generate([[1] * 30], 3)[0]) == 2


def test_forward_refuses_half_given_groups(cuda):
    """The C struct's own checks: groups without prefixes, or without their workspace."""
    import ctypes as C

    import torch

    from ssd_b200._lib import GemmaBatchC, lib, ptr, stream_ptr
    from ssd_b200.models.gemma import GemmaRunner, allocate_kv_cache

    w = weights("toy-target")
    cache = allocate_kv_cache(w, 4, 16)
    runner = GemmaRunner(w, 1, 1, 32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tok, slb, tab, starts, pre = i32([[1]]), i32([0]), i32([[0, 1]]), i32([0, 1]), i32([0])
    lg = torch.empty((1, w.shape.vocab), device="cuda")
    sc = runner.scratch(1, 1)

    def batch(**kw):
        bt = GemmaBatchC()
        bt.B = bt.T = 1
        bt.tokens, bt.seq_lens_before, bt.kv_pages = ptr(tok), ptr(slb), ptr(cache.pages)
        bt.num_blocks, bt.block_size, bt.block_tables, bt.max_blocks, bt.max_seq_len = 4, 16, ptr(tab), 2, 32
        bt.logits, bt.logits_last_only, bt.scratch, bt.scratch_bytes = ptr(lg), 1, ptr(sc), sc.numel()
        for k, v in kw.items():
            setattr(bt, k, v)
        return lib().ssd_gemma_forward(stream_ptr(), C.byref(w.cstruct()), C.byref(bt))

    assert batch(group_starts=ptr(starts), num_groups=1) == 1
    assert batch(group_starts=ptr(starts), prefix_lens=ptr(pre)) == 1
    assert batch(group_starts=ptr(starts), prefix_lens=ptr(pre), num_groups=1) == 5
    assert batch() == 0
