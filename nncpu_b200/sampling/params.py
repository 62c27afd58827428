"""How the next token is chosen and how a reply is generated: the reference's
``SamplerParams``, ``GenerateParams``, ``StopReason`` and ``GenerateResult``
(crates/nncpu/src/session/mod.rs:86-177) with the same names, meanings and
defaults."""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from enum import Enum
from typing import List, Optional, Tuple

from ..errors import InvalidArgument


@dataclass(frozen=True)
class SamplerParams:
    """top-k, then top-p, then min-p on the model's own distribution, then
    temperature over what survives.  ``temperature`` 0 = greedy; ``top_k`` 0 =
    all; ``top_p`` 1 = off; ``min_p`` 0 = off."""
    temperature: float = 0.7
    top_k: int = 40
    top_p: float = 0.95
    min_p: float = 0.05

    @staticmethod
    def greedy() -> "SamplerParams":
        return SamplerParams(temperature=0.0)

    def check(self, function: str = "sample") -> None:
        """crates/nncpu/src/session/mod.rs:122-131."""
        def unit(v):
            return isinstance(v, (int, float)) and math.isfinite(v) and 0.0 <= v <= 1.0
        ok = (isinstance(self.temperature, (int, float)) and math.isfinite(self.temperature)
              and self.temperature >= 0 and unit(self.top_p) and unit(self.min_p)
              and isinstance(self.top_k, int) and self.top_k >= 0)
        if not ok:
            raise InvalidArgument(f"{function}: temperature must be >= 0, top_k >= 0, and top_p/min_p in [0, 1]")

    @property
    def is_greedy(self) -> bool:
        return self.temperature <= 0.0

    def truncates(self, vocab: int) -> bool:
        """Whether any of top-k, top-p, min-p removes candidates."""
        return (0 < self.top_k < vocab) or (0.0 < self.top_p < 1.0) or self.min_p > 0.0


MAX_ALTERNATIVES = 32      # tokens beside the given one whose log probabilities can be asked for


@dataclass(frozen=True)
class GenerateParams:
    """``max_tokens`` 0 = until a stop token or a full context.  ``logprobs`` k: the result tells every generated token's log
    probability, the entropy of what it was drawn from and the k likeliest tokens (0: none of those; None: nothing of it)."""
    max_tokens: int = 0
    sampler: SamplerParams = field(default_factory=SamplerParams)
    logprobs: Optional[int] = None

    def check(self, function: str = "generate") -> None:
        self.sampler.check(function)
        if self.max_tokens < 0:
            raise InvalidArgument(f"{function}: max_tokens {self.max_tokens}")
        check_alternatives(self.logprobs, function)


def check_alternatives(k: Optional[int], function: str) -> None:
    if k is not None and not (isinstance(k, int) and 0 <= k <= MAX_ALTERNATIVES):
        raise InvalidArgument(f"{function}: the {k} likeliest tokens (0 to {MAX_ALTERNATIVES})")


@dataclass(frozen=True)
class TokenLogprob:
    """How likely a token was under the model's own distribution (temperature 1, nothing cut), in nats: its log probability, the
    distribution's entropy, and the likeliest tokens as (id, log probability), the likeliest first."""
    token: int
    logprob: float
    entropy: float
    top: Tuple[Tuple[int, float], ...] = ()


@dataclass
class ScoreResult:
    """A text's tokens from the second on, each given those before it."""
    tokens: List[TokenLogprob] = field(default_factory=list)

    @property
    def logprob(self) -> float:
        """The text's log probability given its first token."""
        return math.fsum(t.logprob for t in self.tokens)

    @property
    def perplexity(self) -> float:
        """e to the mean of the tokens' negative log probabilities (NaN of a text of one token)."""
        if not self.tokens:
            return math.nan
        mean = -self.logprob / len(self.tokens)
        return math.inf if mean >= 700 else math.exp(mean)


class StopReason(Enum):
    END_OF_TURN = "EndOfTurn"      # the model produced a stop token
    MAX_TOKENS = "MaxTokens"       # max_tokens were generated
    CONTEXT_FULL = "ContextFull"   # the sequence reached the context size
    CALLBACK = "Callback"          # the callback returned False
    CANCELLED = "Cancelled"        # cancel() was called


@dataclass
class GenerateResult:
    """What one sequence's generation did.  ``tokens`` are the generated
    tokens, the stop token not among them; ``n_generated == len(tokens)``.  ``logprobs``: one for each of them, if asked for."""
    stop: StopReason = StopReason.END_OF_TURN
    n_prompt: int = 0
    n_generated: int = 0
    prefill: float = 0.0   # seconds spent on the prompt (shared by a batch)
    decode: float = 0.0    # seconds spent generating (shared by a batch)
    tokens: List[int] = field(default_factory=list)
    logprobs: Optional[List[TokenLogprob]] = None
