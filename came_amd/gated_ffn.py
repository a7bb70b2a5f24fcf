"""The gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) Wd^T`` with its gradients, in libcame8.

Both projections, the activation and the product are one kernel, the down projection another; backward, the activation's
gradient is formed where the product ``dy Wd`` ends, and no operand is transposed in memory.  Calls of more than 16 tokens
copy rows that end inside 16 bytes, and 16-bit matrices of an odd row stride, to aligned ones; the forward pass reads an
odd-strided ``w_down`` where it is unless there are many tokens.  Kept for the backward pass: the operands and, in float32,
``x Wg^T`` and ``x Wu^T`` (8 bytes a hidden value); the product ``h`` is formed again.  The autograd node is native
(csrc/came8_host.cpp).
"""
from __future__ import annotations

import torch

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}  # include/came8.h: CAME8_ACT_*


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T`` over the last dimension of ``x``.

    x [..., dim]; w_gate, w_up [hidden, dim]; w_down [out, hidden]: one type (float32, bfloat16 or float16), one GPU.
    activation: "silu", "gelu" (by erf) or "gelu_tanh".  Differentiable once in every operand, in
    reverse mode (an operand with a forward-mode tangent is refused).  Operands whose rows are contiguous are read where they
    are, with the row strides they have; others are copied.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    stream = torch.cuda.current_stream(x.device).cuda_stream if isinstance(x, torch.Tensor) and x.is_cuda else 0
    return _lib.host().gated_ffn(x, w_gate, w_up, w_down, act, stream)
