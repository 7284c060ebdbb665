"""Sampling parameters and the per-sequence random keys.

The reference draws with one torch generator shared by everything
(cpmcu/llm.py:55-59, 282-285): ``temperature == 0`` is greedy, otherwise
``multinomial(softmax(logits / temperature))``.  Here a sequence's draw number n uses
the counter-based random value of (seed, sequence key, n), so what a sequence draws
does not depend on which other sequences share its batch.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional


@dataclass(frozen=True)
class SamplingParams:
    """temperature 0 = greedy (lowest index among equal logits); top_p < 1 keeps the
    smallest set of most likely tokens whose mass reaches top_p.  top_k > 0 keeps the
    likeliest top_k first (and top_p counts in their mass); min_p > 0 keeps of the rest
    what is at least min_p times as likely as the likeliest.  With either of these a sequence
    is drawn by ``Ops.sample_filtered``, without by ``Ops.sample``, whatever the others of its
    batch are drawn by (a greedy one by either: they agree)."""

    temperature: float = 0.0
    top_p: float = 1.0
    top_k: int = 0
    min_p: float = 0.0

    def __post_init__(self):
        if self.temperature < 0:
            raise ValueError(f"temperature must be >= 0, got {self.temperature}")
        if not 0 < self.top_p <= 1:
            raise ValueError(f"top_p must be in (0, 1], got {self.top_p}")
        if self.top_k < 0:
            raise ValueError(f"top_k must be >= 0, got {self.top_k}")
        if not 0 <= self.min_p <= 1:
            raise ValueError(f"min_p must be in [0, 1], got {self.min_p}")

    @property
    def filtered(self) -> bool:
        return self.temperature > 0 and (self.top_k > 0 or self.min_p > 0)

    @property
    def unfiltered(self) -> bool:
        return self.temperature > 0 and not self.filtered

    @property
    def greedy(self) -> bool:
        return self.temperature == 0.0
