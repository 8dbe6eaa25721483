"""Sampling options under the reference's names, defaults and meanings.

Field for field the reference's ``SamplingConfig`` (app/runtime/generation_request.py:8-19):
``temperature`` (<= 0 means greedy argmax and nothing else runs, app/runtime/sampler.py:30-38),
``top_p``, ``top_k`` (0 disables), ``repeat_penalty`` (1.0 disables; applies to generated ids
only, sampler.py:12-26), ``num_ctx`` (the most tokens a request may hold), ``num_predict``
(-1: until EOS or ``num_ctx``) and ``seed`` (None: fresh entropy on every call).

The reference has no more. Beside them, in the meanings that serving interfaces give them: ``presence_penalty`` and
``frequency_penalty`` (taken off the score of a generated id, once and for each time it came), ``logit_bias`` (a mapping or
pairs of token id and what its score gains) and ``allowed_token_ids`` (None: all; the others are never drawn). They
are applied in that order after the repeat penalty and before everything else, greedy choice included.
"""

from __future__ import annotations

from collections.abc import Mapping
from dataclasses import dataclass


LARGEST_FLOAT32 = (2.0 - 2.0 ** -23) * 2.0 ** 127


@dataclass(frozen=True)
class SamplingConfig:
    temperature: float = 0.8
    top_p: float = 0.9
    top_k: int = 40
    repeat_penalty: float = 1.1
    num_ctx: int = 2048
    num_predict: int = -1
    seed: int | None = None
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: tuple[tuple[int, float], ...] = ()
    allowed_token_ids: tuple[int, ...] | None = None

    def __post_init__(self) -> None:
        pairs = self.logit_bias.items() if isinstance(self.logit_bias, Mapping) else (self.logit_bias or ())
        # a token named twice keeps its later bias
        bias = tuple({int(token): float(value) for token, value in pairs}.items())
        # scores are 32-bit numbers: what is beyond their range would become infinite there (nan fails the comparisons too)
        if not all(abs(value) <= LARGEST_FLOAT32 for _, value in bias):
            raise ValueError("a logit_bias must be finite as a 32-bit number; allowed_token_ids rules tokens out")
        if not (abs(self.presence_penalty) <= LARGEST_FLOAT32 and abs(self.frequency_penalty) <= LARGEST_FLOAT32):
            raise ValueError("presence_penalty and frequency_penalty must be finite as 32-bit numbers")
        allowed = self.allowed_token_ids
        if allowed is not None:
            allowed = tuple(sorted({int(token) for token in allowed}))
            if not allowed:
                raise ValueError("allowed_token_ids must name at least one token")
        for token in (*(token for token, _ in bias), *(allowed or ())):
            if token < 0:
                raise ValueError(f"{token} is no token id")
        object.__setattr__(self, "logit_bias", bias)
        object.__setattr__(self, "allowed_token_ids", allowed)

    @property
    def is_greedy(self) -> bool:
        return self.temperature <= 0.0

    @property
    def adjusts_scores(self) -> bool:
        """Whether scores change by more than the repeat penalty before a token is chosen."""
        return bool(self.presence_penalty or self.frequency_penalty or self.logit_bias) or self.allowed_token_ids is not None

    @property
    def largest_token_id(self) -> int:
        """The largest token id that the options name, -1 if they name none."""
        return max((*(token for token, _ in self.logit_bias), *(self.allowed_token_ids or ())), default=-1)
