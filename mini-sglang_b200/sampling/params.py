from __future__ import annotations

import dataclasses
import operator
from typing import Any, Dict, Optional

MAX_LOGPROBS = 32          # alternatives a token (what the kernel keeps)


@dataclasses.dataclass
class SamplingParams:
    """Names, meanings and defaults of mini_sglang/managers/sampling_params.py:4-19.
    temperature 0 is greedy; eos_token_id -1 means "the model's own end tokens"; `seed` (ours)
    fixes the noise of temperature sampling for the request; `logprobs` (ours): with every token its log probability
    under the model (before the temperature), the entropy of its distribution and that many most probable tokens."""

    temperature: float = 0.0
    max_new_tokens: int = 64
    ignore_eos: bool = False
    eos_token_id: int = -1
    seed: Optional[int] = None
    logprobs: Optional[int] = None

    def check_logprobs(self) -> None:
        """Anything but a whole number in range is refused (inside a step it would stop every other request of the batch as well)."""
        if self.logprobs is None:
            return
        try:
            n = -1 if isinstance(self.logprobs, bool) else operator.index(self.logprobs)
        except TypeError:
            n = -1
        if not 0 <= n <= MAX_LOGPROBS:
            raise ValueError(f"logprobs must be a whole number between 0 and {MAX_LOGPROBS}; got {self.logprobs!r}")
        self.logprobs = n

    @classmethod
    def init_from_dict(cls, d: Optional[Dict[str, Any]]) -> "SamplingParams":
        d = dict(d or {})
        known = {f.name for f in dataclasses.fields(cls)}
        extra = set(d) - known
        if extra:
            raise ValueError(f"unknown sampling parameters {sorted(extra)}; known: {sorted(known)}")
        p = cls(**d)
        if p.temperature < 0:
            raise ValueError("temperature must be >= 0")
        if p.max_new_tokens < 1:
            raise ValueError("max_new_tokens must be >= 1")
        p.check_logprobs()
        return p
