"""Rules on the logits of a verification step (K12).

The reference verifies greedily on the target's bare logits
(src/specfit/runtime/eagle3_tree.py:1241-1290).  ``LogitRules`` holds what a
request adds to that: penalties for repeated tokens, a bias, and, per call,
the set a grammar allows.  In a draft tree every row has a history of its
own, the committed sequence plus the row's path; the sequence's part is a
histogram on the device that ``count`` keeps, the paths come with the call.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import ops


@dataclass
class LogitRules:
    """counts      int32 [vocab] occurrences so far (None: only the paths)
    repetition  x / repetition, or x * repetition where x < 0, for every token
                that occurred
    presence    taken off every token that occurred
    frequency   taken off for each occurrence
    bias        fp32 [vocab] or [rows, vocab], added to every token

    All penalties go by the same occurrences; for others, ``adjust`` with two
    rules in turn (on fp32 logits, so that nothing is rounded in between)."""

    counts: torch.Tensor | None = None
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: torch.Tensor | None = None

    @classmethod
    def for_vocab(cls, vocab_size: int, device, **kwargs) -> "LogitRules":
        """Rules with an empty histogram."""
        return cls(counts=torch.zeros(vocab_size, dtype=torch.int32, device=device), **kwargs)

    def count(self, tokens: torch.Tensor) -> None:
        """Adds ``tokens`` (int64, any shape) to the histogram; those outside
        the vocabulary, such as a -1 of ``greedy``, count for nothing."""
        if self.counts is None:
            raise ValueError("these rules keep no histogram")
        tokens = tokens.reshape(-1)
        known = (tokens >= 0) & (tokens < self.counts.shape[0])
        self.counts.index_add_(0, torch.where(known, tokens, 0), known.to(torch.int32))

    def adjust(self, logits: torch.Tensor, paths: torch.Tensor | None = None, *,
               allowed: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """The adjusted logits (see ops.adjust_logits)."""
        return ops.adjust_logits(logits, counts=self.counts, paths=paths,
                                 repetition=self.repetition, presence=self.presence,
                                 frequency=self.frequency, bias=self.bias, allowed=allowed, out=out)

    def greedy(self, logits: torch.Tensor, paths: torch.Tensor | None = None, *,
               allowed: torch.Tensor | None = None) -> torch.Tensor:
        """Each row's greedy token, -1 where nothing is allowed (see
        ops.greedy_tokens)."""
        return ops.greedy_tokens(logits, counts=self.counts, paths=paths,
                                 repetition=self.repetition, presence=self.presence,
                                 frequency=self.frequency, bias=self.bias, allowed=allowed)
