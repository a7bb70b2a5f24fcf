"""The global gradient norm over many tensors, and the clip by it.

One pass over the gradients, whatever their number and types, with the arithmetic of ``torch.nn.utils.clip_grad_norm_``
(norm type 2): ``norm = sqrt(sum of squares)``, ``factor = min(1, max_norm / (norm + 1e-6))``, gradients times the factor
in place.  No host synchronisation: the norm is a device tensor.
"""
from __future__ import annotations

import torch

from . import _lib

_DTYPE_CODE = {torch.float32: _lib.CAME8_F32, torch.bfloat16: _lib.CAME8_BF16, torch.float16: _lib.CAME8_F16}


def _check(t: torch.Tensor, what: str, device) -> None:
    if t.layout != torch.strided:
        raise RuntimeError(f"{what}: sparse gradients are not supported")
    if not t.is_cuda:
        raise RuntimeError(f"{what}: came_amd runs on the GPU; got a {t.device} tensor")
    if t.dtype not in _DTYPE_CODE:
        raise RuntimeError(f"{what}: unsupported dtype {t.dtype} (float32, bfloat16 and float16 are supported)")
    if t.device != device:
        raise RuntimeError(f"{what}: tensors on {device} and {t.device}; the norm is taken on one GPU")


def _contiguous(tensors: list, what: str):
    """The tensors as contiguous ones, and (tensor, contiguous copy) pairs of those that were not."""
    out, copies = [], []
    for t in tensors:
        _check(t, what, tensors[0].device)
        c = t if t.is_contiguous() else t.contiguous()
        if c is not t:
            copies.append((t, c))
        out.append(c)
    return out, copies


def _reduce(tensors: list, max_norm: float | None, scale: bool, what: str, of_parameters: bool = False):
    """(norm, factor): device scalars of one call over the tensors, or the parameters' gradients; with `scale` those are
    multiplied in place, and factor is None.  None where no parameter has a gradient."""
    device = next((t.device for t in tensors if not of_parameters or t.grad is not None), None)
    if device is None:
        return None
    stream = torch.cuda.current_stream(device).cuda_stream if device.type == "cuda" else 0
    host = _lib.host()
    found = host.grad_norm(tensors, of_parameters, float(max_norm or 0.0), scale, stream)
    if found is None:  # strided tensors, or ones that are refused
        if of_parameters:
            tensors = [g for g in [p.grad for p in tensors] if g is not None]
        tensors, copies = _contiguous(tensors, what)
        found = host.grad_norm([t.detach() for t in tensors], False, float(max_norm or 0.0), scale, stream)
        if found is None:  # nothing else is left that it refuses
            raise RuntimeError(f"{what}: tensor subclasses that dispatch in Python are not supported: their values may lie elsewhere")
        for t, c in copies if scale else ():
            t.copy_(c)
    return found


@torch.no_grad()
def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm over all elements of the tensors (a 0-d float32 tensor on their device)."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    return _reduce(tensors, None, False, "grad_norm")[0]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the parameters' gradients in place so that their 2-norm together is at most ``max_norm``; returns the norm
    before that.  A norm that is infinite or NaN makes them 0 or NaN, as in torch; with ``error_if_nonfinite`` it raises
    and leaves them as they were (and waits for the GPU to know)."""
    if not float(max_norm) >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if not isinstance(error_if_nonfinite, (bool, int)) or error_if_nonfinite not in (0, 1):  # torch's third argument is norm_type
        raise TypeError(f"error_if_nonfinite must be a bool, got {error_if_nonfinite!r}; the norm is always the 2-norm")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    parameters = list(parameters)
    if error_if_nonfinite:
        found = _reduce(parameters, None, False, "clip_grad_norm_", True)
        if found is not None and not bool(torch.isfinite(found[0])):
            raise RuntimeError("clip_grad_norm_: the gradients' norm is not finite")
    found = _reduce(parameters, max_norm, True, "clip_grad_norm_", True)
    return torch.tensor(0.0) if found is None else found[0]
