"""Beam search's selection over beams and vocabulary on the GPU (``ssd_beam_select``).

The reference decodes greedily (jax_ssd/runtime/engine.py:224) and has no counterpart.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from .._lib import lib
from ..kernels.kv8_cache import ints, launch

MAX_BEAMS = 32


class BeamStep(NamedTuple):
    scores: torch.Tensor    # [G, W] fp32 sums of log-probabilities, best rank first; -inf: no beam
    parents: torch.Tensor   # [G, W] int32 beam that each one continues (-1: none)
    tokens: torch.Tensor    # [G, W] int32 its new token; eos for a beam that had finished (-1: none)
    lengths: torch.Tensor   # [G, W] int32 tokens generated, the new one included
    finished: torch.Tensor  # [G, W] uint8


@lru_cache(maxsize=1024)  # a function of these sizes alone
def _workspace_size(g: int, w: int, v: int) -> int:
    return lib().ssd_beam_select_workspace_size(g, w, v)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, lengths: torch.Tensor | None = None,
                finished: torch.Tensor | None = None, *, eos_token_id: int | None = None,
                length_penalty: float = 0.0) -> BeamStep:
    """The W best continuations of each request's W beams (``ssd_beam_select``).

    ``logits`` fp32 [G, W, V] (rows contiguous, at one stride) and ``scores`` fp32 [G, W], the beams' sums of
    log-probabilities: -inf for beams that do not exist yet, all but the first before the first step.
    ``lengths`` int32 [G, W] tokens generated so far (None: 0), ``finished`` uint8 or bool [G, W] (None: none;
    needs ``eos_token_id``).  A live beam's candidates have the log-softmax of its logits added to its score and are
    ranked by score / length ** ``length_penalty``; a finished beam stands for itself.  Ranks are compared in
    64 bits, ties go to the lowest beam, then token.  Places without a candidate: score -inf, parent and token -1.
    """
    if logits.dim() != 3 or logits.dtype is not torch.float32 or not logits.is_cuda:
        raise ValueError(f"logits must be an fp32 CUDA tensor [G, W, V], got {logits.dtype} {list(logits.shape)}")
    g, w, v = logits.shape
    dev = logits.get_device()
    s0, ld, s2 = logits.stride()
    if w == 1:
        ld = s0
    if g * w == 1:
        ld = v
    if (s2 != 1 and v > 1) or (g > 1 and w > 1 and s0 != w * ld) or ld < v:
        logits = logits.contiguous()
        ld = v
    if not 1 <= w <= MAX_BEAMS or v < 1:
        raise ValueError(f"1 to {MAX_BEAMS} beams and a vocabulary are needed, got {list(logits.shape)}")
    if scores.dtype is not torch.float32 or scores.shape != (g, w) or scores.get_device() != dev or not scores.is_contiguous():
        raise ValueError(f"scores must be a contiguous fp32 tensor [{g}, {w}] on cuda:{dev}")
    if finished is not None:
        if eos_token_id is None:
            raise ValueError("finished beams need eos_token_id")
        if (finished.dtype not in (torch.uint8, torch.bool) or finished.shape != (g, w) or finished.get_device() != dev
                or not finished.is_contiguous()):
            raise ValueError(f"finished must be a contiguous uint8 or bool tensor [{g}, {w}] on cuda:{dev}")
    eos = -1 if eos_token_id is None else int(eos_token_id)
    if eos_token_id is not None and not 0 <= eos < v:
        raise ValueError(f"eos_token_id {eos} is outside the vocabulary of {v}")
    if length_penalty != 0.0 and lengths is None:
        raise ValueError("a length penalty needs lengths")
    like = torch.empty_like  # (the cheapest allocation: they are half of a small call's time on the host)
    i = like(scores, dtype=torch.int32) if lengths is None else like(lengths)
    out = BeamStep(like(scores), i, like(i), like(i),
                   like(finished) if finished is not None and finished.dtype is torch.uint8 else like(scores, dtype=torch.uint8))
    need = _workspace_size(g, w, v)
    # a workspace of its own for every call: calls on other streams or in captured graphs share nothing
    ws = scores.new_empty(need, dtype=torch.uint8) if need else None
    launch("ssd_beam_select", dev, logits.data_ptr(), ld, scores.data_ptr(), ints(lengths, (g, w), "lengths", dev),
           None if finished is None else finished.data_ptr(), eos, float(length_penalty), *[t.data_ptr() for t in out],
           None if ws is None else ws.data_ptr(), need, g, w, v)
    return out
