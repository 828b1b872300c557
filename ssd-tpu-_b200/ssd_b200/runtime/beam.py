"""Beam search over paged rows (the reference decodes greedily, jax_ssd/runtime/engine.py:162-211).

G requests of W beams are G*W rows of one forward.  Per step, all on the device:

1. the rows follow their parents (``PageManager.reorder_rows``: the prompt's whole pages are shared by a request's
   beams, a partial page is copied for each further child);
2. one forward over the beams' last tokens; its attention reads what a request's beams share once
   (``ssd_shared_prefix_attention``; an 8-bit cache is read row by row);
3. ``beam_select`` picks the W best continuations of each request.

The tokens and parents of every step stay on the device; the beams are read back through their parents at the end.
"""

from __future__ import annotations

import torch

from ..algorithm.beam import MAX_BEAMS, beam_select
from ..kernels.ops import max_tokens_per_forward
from ..models.gemma import GemmaRunner, GemmaWeights, allocate_kv_cache
from .page_manager import PageManager

_CHECK_EVERY = 16  # steps between looks at whether every beam has finished


def blocks_per_request(num_beams: int, max_seq_len: int, max_new: int, block_size: int) -> int:
    """Blocks that one request's beams hold at most, whatever its prompt (prompt + max_new - 1 tokens within max_seq_len).

    The n // block_size whole blocks of a prompt of n tokens are shared by all beams; from the block of the prompt's end on
    each beam may have its own, at most (max_new + 2 block_size - 3) // block_size of them.
    """
    every = -(-max_seq_len // block_size)
    own = min((max(max_new, 1) + 2 * block_size - 3) // block_size, every)
    return every - own + num_beams * own


def requests_that_fit(shape, elem: int, num_beams: int, requests: int, max_seq_len: int, max_new: int, block_size: int,
                      free_bytes: int) -> int:
    """How many of ``requests`` searches fit side by side in ``free_bytes``, one at least (which may be refused its memory
    then): their blocks of ``elem`` bytes an element, and their logits."""
    blocks = blocks_per_request(num_beams, max_seq_len, max_new, block_size)
    each = blocks * block_size * shape.kv_bytes_per_token(elem) + 4 * num_beams * shape.vocab
    return max(1, min(requests, free_bytes // each))


class BeamSearchDecoder:
    """Beam search with ``num_beams`` beams for up to ``requests`` prompts at a time.

    ``length_penalty``: beams are ranked by score / length ** length_penalty.  ``eos_token_id``: a beam that emits it
    has finished and keeps its place and score (None: none ever does).  ``max_new``: the most tokens that ``generate`` will
    be asked for (None: up to max_seq_len); the cache holds a prompt's blocks once and the beams' own blocks for so many.
    """

    def __init__(self, target: GemmaWeights, num_beams: int, requests: int = 1, max_seq_len: int = 1024,
                 block_size: int = 16, comm=None, kv_cache_dtype: str = "auto", length_penalty: float = 0.0,
                 eos_token_id: int | None = None, max_new: int | None = None):
        G, W = self.G, self.W = int(requests), int(num_beams)
        if not 1 <= W <= MAX_BEAMS or G < 1:
            raise ValueError(f"1 to {MAX_BEAMS} beams and at least one request are needed, got {W} and {G}")
        B = self.B = G * W
        if B > max_tokens_per_forward(target.dtype):
            raise ValueError(f"requests*num_beams = {B} exceeds one forward ({max_tokens_per_forward(target.dtype)})")
        if eos_token_id is not None and not 0 <= eos_token_id < target.shape.vocab:
            raise ValueError(f"eos_token_id {eos_token_id} is outside the vocabulary of {target.shape.vocab}")
        self.dev = dev = target.device
        self.max_seq_len = int(max_seq_len)
        self.max_new = self.max_seq_len if max_new is None else int(max_new)
        if not 0 <= self.max_new <= self.max_seq_len:
            raise ValueError(f"max_new must be 0 to {self.max_seq_len}, got {max_new}")
        self.length_penalty, self.eos = float(length_penalty), eos_token_id
        blocks = (self.max_seq_len + block_size - 1) // block_size + 1
        num_blocks = G * blocks_per_request(W, self.max_seq_len, self.max_new, block_size) + 2
        self.cache = allocate_kv_cache(target, num_blocks, block_size, kv_cache_dtype)
        self.pm = PageManager(block_size, num_blocks, max_seqs=B, max_blocks_per_seq=blocks, device=dev)
        self.runner = GemmaRunner(target, B, 64, self.max_seq_len, comm=comm)
        self.chunk = min(64, max_tokens_per_forward(target.dtype))
        V = self.V = target.shape.vocab
        buf = comm.alloc if comm is not None else (lambda shape, dtype: torch.empty(shape, dtype=dtype, device=dev))
        self.logits = buf((B, V), torch.float32)
        self.starts = torch.arange(0, B + 1, W, dtype=torch.int32, device=dev)

    def _i32(self, v) -> torch.Tensor:
        return torch.tensor(v, dtype=torch.int32, device=self.dev)

    def _prefill(self, row: int, prompt: list[int]) -> None:
        n = len(prompt)
        p = torch.tensor([prompt], dtype=torch.int32, device=self.dev)
        self.pm.allocate_rows(row, 1, self._i32([0]), self._i32([n]), None)
        for c0 in range(0, n, self.chunk):
            c1 = min(n, c0 + self.chunk)
            self.runner.forward(p[:, c0:c1].contiguous(), self._i32([c0]), self.cache, self.pm.tables[row:row + 1],
                                self.logits[row:row + 1] if c1 == n else None, last_only=True)

    def generate(self, prompts: list[list[int]], max_new: int) -> list[list[tuple[list[int], float]]]:
        """For each prompt its beams, best first: (tokens, sum of their log-probabilities).  A finished beam's tokens end
        with ``eos_token_id``.  Fewer beams than ``num_beams`` where there are not as many continuations."""
        G, W, B, dev = self.G, self.W, self.B, self.dev
        prompts = [[int(t) for t in p] for p in prompts]
        n = len(prompts)
        if not 1 <= n <= G:
            raise ValueError(f"expected 1 to {G} prompts, got {n}")
        if any(not p for p in prompts):
            raise ValueError("empty prompt")
        if max_new < 1:
            return [[([], 0.0)] for _ in prompts]
        if max_new > self.max_new:
            raise ValueError(f"{max_new} new tokens were asked for, the decoder's cache was made for {self.max_new}")
        if max(len(p) for p in prompts) + max_new - 1 > self.max_seq_len:
            raise ValueError("prompt + max_new exceeds max_seq_len")
        self.pm.free_rows(0, B)
        scores = torch.full((G, W), float("-inf"), device=dev)
        for g, p in enumerate(prompts):
            self._prefill(g * W, p)
        scores[:n, 0] = 0.0
        prefix = self._i32([len(p) for p in prompts] + [0] * (G - n))
        held = torch.zeros((G, W), dtype=torch.int32, device=dev)
        held[:, 0] = prefix
        ones = torch.ones(B, dtype=torch.int32, device=dev)
        lengths = torch.zeros((G, W), dtype=torch.int32, device=dev)
        finished = None if self.eos is None else torch.zeros((G, W), dtype=torch.uint8, device=dev)
        logits = self.logits.view(G, W, self.V)
        history = []
        for t in range(max_new):
            step = beam_select(logits, scores, lengths, finished, eos_token_id=self.eos,
                               length_penalty=self.length_penalty)
            scores, lengths = step.scores, step.lengths
            finished = None if self.eos is None else step.finished
            history.append((step.parents, step.tokens))
            if t + 1 == max_new or (self.eos is not None and t % _CHECK_EVERY == _CHECK_EVERY - 1
                                    and bool(step.finished.all())):
                break
            ok = self.pm.reorder_rows(0, step.parents, held.view(B), self.cache)  # noqa: F841  (every beam has its blocks)
            # the rows of a request hold one number of tokens, but for places without a beam, which are empty
            held = torch.where(step.parents >= 0, held[:, :1] if t == 0 else held.amax(1, keepdim=True), 0).to(torch.int32)
            self.pm.allocate_rows(0, B, held.view(B), ones, None)
            self.runner.forward(step.tokens.clamp(min=0).view(B, 1), held.view(B), self.cache, self.pm.tables, self.logits,
                                last_only=True, groups=(self.starts, prefix))
            held = held + 1
        return self._read_back(history, scores, lengths, n)

    def _read_back(self, history, scores, lengths, n: int) -> list[list[tuple[list[int], float]]]:
        parents = torch.stack([p for p, _ in history]).cpu().tolist()
        tokens = torch.stack([t for _, t in history]).cpu().tolist()
        scores, lengths = scores.cpu().tolist(), lengths.cpu().tolist()
        out = []
        for g in range(n):
            beams = []
            for w in range(self.W):
                if scores[g][w] == float("-inf"):
                    continue
                seq, at = [], w
                for p, t in zip(reversed(parents), reversed(tokens)):
                    seq.append(t[g][at])
                    at = p[g][at]
                beams.append((seq[::-1][:lengths[g][w]], scores[g][w]))  # past its length a finished beam repeats eos
            out.append(beams)
        return out
