"""The embedding of tokens with its gradient, in libcame8.

Backward, the positions are sorted by their tokens and the rows of a token summed in float32, in the order of its positions, so
that a gradient repeats bit for bit; the whole table's gradient is written in the same pass, rows without a token as zeros.
"""
from __future__ import annotations

import torch

from . import _lib


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[tokens]``, [..., dim].

    tokens [...]: int64 or int32; weight [vocab, dim]: float32, bfloat16 or float16; one GPU.  ``scale`` is taken in float32; one
    that would become infinite or 0 there is refused.  ``padding_idx``: a token whose row has no gradient (a negative one counts
    from the end).  A token outside of [0, vocab) gives zeros and has no gradient: where a table's rows are split over processes,
    each looks its own up and the results add.  Nothing raises for one, since the host does not read the tokens.  Differentiable
    once in ``weight``, in reverse mode.
    """
    padding = -1
    if padding_idx is not None:
        vocab = weight.shape[0] if isinstance(weight, torch.Tensor) and weight.dim() == 2 else 0
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"embedding: padding_idx must be a token of the {vocab} that weight has, got {padding_idx}")
        padding = padding_idx + vocab if padding_idx < 0 else padding_idx
    return _lib.host().embedding(tokens, weight, scale, padding, *_lib.current(weight))
