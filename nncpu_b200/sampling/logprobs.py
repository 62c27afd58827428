"""The log probabilities of the tokens that a generation chose, or that a text holds.

What a step's logits say about its tokens is launched right after the choice, before the next step may overwrite the logits, into
tensors of its own; nothing waits for it until a result is asked for.
"""
from __future__ import annotations

from typing import List

import torch

from .. import perf
from ..kernels import ops
from .params import TokenLogprob


class Logprobs:
    """Collects rows of (logits, token) and reads them all at once.  ``k``: how many of the likeliest tokens come with each."""

    def __init__(self, k: int, vocab_size: int):
        self.k = min(k, vocab_size)
        self._steps: List[tuple] = []
        self._rows = 0

    def add(self, logits: torch.Tensor, tokens) -> int:
        """``logits`` [n, vocab] on the device, ``tokens`` int32 [n] there or a list: n rows more.  Returns the first one's number."""
        n = logits.shape[0]
        if not isinstance(tokens, torch.Tensor):
            tokens = torch.tensor(list(tokens), dtype=torch.int32, device=logits.device)
        lp, entropy = (torch.empty(n, dtype=torch.float32, device=logits.device) for _ in range(2))
        top = ids = None
        if self.k:
            top = torch.empty(n, self.k, dtype=torch.float32, device=logits.device)
            ids = torch.empty(n, self.k, dtype=torch.int32, device=logits.device)
        tokens = tokens[:n].clone()          # (a choice buffer is written again by the next step)
        with perf.scope("logprobs"):
            ops.token_logprobs(logits, tokens, lp, entropy, top, ids)
        self._steps.append((tokens, lp, entropy, top, ids))
        first, self._rows = self._rows, self._rows + n
        return first

    def read(self) -> List[TokenLogprob]:
        """All rows in the order in which they came; waits for the device."""
        if not self._steps:
            return []
        tokens, lp, entropy = (torch.cat([s[i] for s in self._steps]).tolist() for i in range(3))
        top = torch.cat([s[3] for s in self._steps]).tolist() if self.k else [()] * self._rows
        ids = torch.cat([s[4] for s in self._steps]).tolist() if self.k else [()] * self._rows
        return [TokenLogprob(t, a, e, tuple(zip(i, p))) for t, a, e, p, i in zip(tokens, lp, entropy, top, ids)]
