"""The product of 8-bit rows with a scale each, in libcame8, on the matrix cores."""
from __future__ import annotations

import torch

from . import _lib

_CODES = {torch.float32: _lib.CAME8_F32, torch.bfloat16: _lib.CAME8_BF16, torch.float16: _lib.CAME8_F16}


def int8_linear(q: torch.Tensor, scale: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(q @ w_q.T) * scale[..., None] * w_scale + bias``, [..., out] of ``dtype``.

    q [..., in], w_q [out, in]: int8; scale [...], w_scale [out]: float32 (``rms_norm_int8`` and ``quantize_rows`` give both);
    bias [out] of ``dtype``.  Up to 131071 codes a row, whose sums are exact in 32 bits; the scales and the bias are applied in
    float32 and the result is rounded once.  Operands whose rows are contiguous are read where they are; others are copied, as are
    rows a multiple of 4 bytes apart that do not start on words and, for more than 16 rows of q, ones any other distance apart.
    No gradient: scales or a bias that require one are refused unless under
    ``torch.no_grad()``.
    """
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"int8_linear: dtype must be float32, bfloat16 or float16, got {dtype}")
    return _lib.host().int8_linear(q, scale, w_q, w_scale, bias, code, _lib.current(q)[0])
