"""Generation controls (jax_ssd/sampling_params.py:8-13, plus ``top_p``)."""

from __future__ import annotations

from dataclasses import dataclass


@dataclass
class SamplingParams:
    temperature: float = 0.0
    draft_temperature: float = 0.0
    max_new_tokens: int = 128
    ignore_eos: bool = False
    # not in the reference: nucleus filtering of the target and draft distributions when temperature > 0
    top_p: float = 1.0
    # not in the reference: beam search (ar mode, temperature 0) when num_beams > 1; beams are ranked by
    # score / length ** length_penalty (with one beam there is nothing to rank).  Outputs, of every mode, end with
    # eos_token_id (None, or with ignore_eos: at max_new_tokens)
    num_beams: int = 1
    length_penalty: float = 0.0
    eos_token_id: int | None = None
