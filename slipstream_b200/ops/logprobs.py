"""Log probabilities of given tokens under rows of logits, with their ranks, the entropy of each row and its likeliest tokens."""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from .functions import KernelError, _native_launches, error_address, logprobs_library
from .library import load_calls

MAX_TOP_LOGPROBS = 64  # csrc/logprob_calls.h


class TokenLogprobs(NamedTuple):
    """What `token_logprobs` returns; all but ``packed`` are views of it.

    ``packed``: float32 [N, 3 + 2 k], what one copy brings to the host: a row's log probability, entropy, rank (int32 bits), its k largest
    log probabilities and their tokens (int32 bits).
    ``logprobs``, ``entropy``: float32 [N], ``ranks``: int32 [N], ``top_logprobs``: float32 [N, k], ``top_tokens``: int32 [N, k]."""

    packed: torch.Tensor
    logprobs: torch.Tensor
    entropy: torch.Tensor
    ranks: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


_native = None


def _calls():
    """The call's host side (csrc/logprob_calls.cpp), loaded and told its entry point at the first call."""
    global _native
    if _native is None:
        lib, module = logprobs_library(), load_calls("logprob_calls")
        module.use(KernelError, ctypes.cast(lib.ss_token_logprobs, ctypes.c_void_p).value, error_address)
        if module.launched not in _native_launches:  # (two threads may make the first call)
            _native_launches.append(module.launched)
        _native = module
    return _native


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """``log softmax(logits_n)[tokens_n]`` of each row of ``logits`` (float32 or bfloat16 [N, V], any row stride) for ``tokens`` (int32 or
    int64 [N]), computed in float32 with the sums joined in float64.  Beside it the token's rank (1: no logit is larger, nor equal at a
    lower index), the entropy of the row, and the ``top`` (0 to 64) largest log probabilities with their tokens, the lower index
    first among equals.

    Logits of -inf are masked tokens: they add nothing to the entropy, and their log probability is -inf.  A row of nothing but -inf, or
    one that holds +inf or NaN, has NaN for its log probabilities and entropy; NaN is in no rank, has the rank 0, and is no alternative
    (where alternatives run out, their token is -1 and their log probability NaN).  A token below 0 stands for none: NaN, rank 0.  One at
    or above V is reported in the device's error word."""
    return TokenLogprobs(*(_native or _calls()).token_logprobs(logits, tokens, top))


__all__ = ["MAX_TOP_LOGPROBS", "TokenLogprobs", "token_logprobs"]
