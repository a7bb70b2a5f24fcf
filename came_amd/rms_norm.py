"""The root-mean-square norm with the residual's addition, with its gradients or with its result in 8 bits, in libcame8.

A row is read once: the addition, the norm and the rounding to 8 bits are one kernel, and so are all gradients but the join of the
weight's partial sums.
"""
from __future__ import annotations

import torch

from . import _lib


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor | None = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension of ``h = x + residual``; returns it, and with a residual
    ``(it, h)``.

    x, residual [..., dim], weight [dim]: one type (float32, bfloat16 or float16), one GPU.  ``h`` is rounded to that type, and
    the norm is that of the rounded values; sums are float32, and so is ``eps`` (finite, at least 0).  Differentiable once in every
    operand, in reverse mode.  Operands whose rows are contiguous are read where they are, others are copied.
    """
    out = _lib.host().rms_norm(x, weight, residual, eps, *_lib.current(x))
    return out[0] if residual is None else out


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor | None = None):
    """The norm's result in 8 bits with a scale for each row: ``(codes, scales)``, and with a residual ``(codes, scales, h)``.

    ``codes[i] * scales[i]`` is the row: with ``p = h * weight`` and ``a = max |p|`` the codes are int8 of ``p * 127 / a`` rounded
    to nearest even (exactly: what scales the row as a whole moves no code), the scale is ``a / sqrt(mean(h^2) + eps) / 127``.
    The norm is not rounded to x's type before.  A row with ``a`` below 2^-100 has codes and scale 0; one that has an
    infinity or NaN has codes 0 and a scale that is not finite.  Rows of codes start at multiples of 16 bytes, as ``int8_linear`` reads
    them best.  No gradient: operands that require one are refused unless under ``torch.no_grad()``.
    """
    return _lib.host().rms_norm_int8(x, weight, residual, eps, _lib.current(x)[0])


def quantize_rows(x: torch.Tensor):
    """``(codes, scales)`` of the rows of x [..., dim] as they are, in the format of ``rms_norm_int8``: activations, or a weight
    [out, in] for ``int8_linear``."""
    return _lib.host().quantize_rows(x, _lib.current(x)[0])
