"""What the engine tells about a token's log probability (``SamplingParams.logprobs`` and ``prompt_logprobs``).

They are those of the model's distribution: of the raw logits, in front of penalty, temperature and filters.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np


@dataclass(frozen=True)
class TokenLogprob:
    """A token under the distribution in front of it: its log probability, its rank (1: the likeliest), the entropy of the distribution
    in nats, and as many of the likeliest tokens with their log probabilities as were asked for."""

    token_id: int
    logprob: float
    rank: int
    entropy: float
    alternatives: tuple[tuple[int, float], ...]


def read_logprobs(packed: np.ndarray, tokens: list[int], wanted: list[int | None]) -> list[TokenLogprob | None]:
    """The rows of `ops.TokenLogprobs.packed` on the host, for ``tokens``; ``wanted``: alternatives of each (None: nothing is told)."""
    whole, k = packed.view(np.int32), (packed.shape[1] - 3) // 2
    out: list[TokenLogprob | None] = []
    for row, bits, token, n in zip(packed, whole, tokens, wanted):
        if n is None:
            out.append(None)
            continue
        pairs = zip(bits[3 + k: 3 + k + n].tolist(), row[3: 3 + n].tolist())
        out.append(TokenLogprob(int(token), float(row[0]), int(bits[2]), float(row[1]), tuple(pairs)))
    return out


__all__ = ["TokenLogprob", "read_logprobs"]
