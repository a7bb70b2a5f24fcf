"""Log probabilities of given tokens with entropy and top alternatives, and their gradient, in libcame8.

A row of logits is read once forward, into registers, and once backward; no probabilities are kept, but two floats a row.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class TokenLogProbs(NamedTuple):
    log_probs: torch.Tensor      # [...] float32
    entropy: torch.Tensor        # [...] float32
    top_log_probs: torch.Tensor  # [..., top] float32, the largest first
    top_tokens: torch.Tensor     # [..., top] int64


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogProbs:
    """``log_softmax(logits)`` at ``tokens``, the entropy of ``softmax(logits)`` and its ``top`` largest log probabilities.

    logits [..., vocab]: float32, bfloat16 or float16, up to 2^20 wide; tokens [...]: int64 or int32; one GPU; top: 0 to 64.  Of
    equal logits the lowest token comes first.  A token outside of [0, vocab) (-100, say) marks a row without one: its log
    probability is 0 and has no gradient.  Logits of -inf have probability 0 and no part in the entropy; a row of nothing else is
    NaN, as one with NaN or inf is.  ``log_probs`` and ``entropy`` are differentiable once, in reverse mode; the top alternatives
    are not.
    """
    return TokenLogProbs(*_lib.host().token_log_probs(logits, tokens, top, *_lib.current(logits)))
