"""The gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) Wd^T`` with its gradients, in libcame8.

Both projections, the activation and the product are one kernel, the down projection another; backward, the activation's
gradient is formed where the product ``dy Wd`` ends, and no operand is copied or transposed in memory.  Kept for the
backward pass: ``x`` and, in float32, ``x Wg^T`` and ``x Wu^T`` (8 bytes a hidden value); the product ``h`` is formed again.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .grad_clip import _DTYPE_CODE

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}  # include/came8.h: CAME8_ACT_*


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor whose rows are contiguous and do not overlap, at a 4-byte aligned address (a copy where they are not, or
    lie too far apart)."""
    n = t.shape[1]
    if (t.stride(1) == 1 or n == 1) and (t.shape[0] == 1 or n <= t.stride(0) <= 1 << 20) and t.data_ptr() % 4 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _describe(x, w_gate, w_up, w_down, act: int) -> _lib.Came8Ffn:
    return _lib.Came8Ffn(x.shape[0], x.shape[1], w_gate.shape[0], w_down.shape[0], _ld(x), _ld(w_gate), _ld(w_up), _ld(w_down),
                         _DTYPE_CODE[x.dtype], act)


def _workspace(f: _lib.Came8Ffn, backward: bool, device) -> torch.Tensor:
    need = ctypes.c_size_t(0)
    _lib.check(_lib.load().came8_gated_ffn_workspace_size(ctypes.byref(f), int(backward), ctypes.byref(need)),
               "came8_gated_ffn_workspace_size")
    return torch.empty(need.value, dtype=torch.uint8, device=device)


def _forward(x, w_gate, w_up, w_down, act: int, keep: bool):
    """(y, g, u, the operands as the kernels read them); x is [tokens, dim]."""
    ops = tuple(_rows(t) for t in (x, w_gate, w_up, w_down))
    f = _describe(*ops, act)
    T, F = f.tokens, f.hidden
    with torch.cuda.device(x.device):
        y = torch.empty((T, f.out), dtype=x.dtype, device=x.device)
        g = u = None
        if keep:
            g, u = torch.empty((2, T, F), dtype=torch.float32, device=x.device).unbind(0)
        if T:
            ws = _workspace(f, False, x.device)
            _lib.check(_lib.load().came8_gated_ffn_forward(
                ctypes.byref(f), *(t.data_ptr() for t in ops), y.data_ptr(), g.data_ptr() if keep else None,
                u.data_ptr() if keep else None, ws.data_ptr(), ws.numel(),
                torch.cuda.current_stream(x.device).cuda_stream), "came8_gated_ffn_forward")
    return y, g, u, ops


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        y, g, u, _ = _forward(x, w_gate, w_up, w_down, act, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, g, u)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, g, u = ctx.saved_tensors
        ops = tuple(_rows(t) for t in (x, w_gate, w_up, w_down))
        f = _describe(*ops, ctx.act)
        dy = dy.contiguous() if dy.data_ptr() % 4 == 0 else dy.clone(memory_format=torch.contiguous_format)
        make = torch.empty if f.tokens else torch.zeros
        with torch.cuda.device(x.device):
            grads = [make(t.shape, dtype=t.dtype, device=t.device) if need else None
                     for t, need in zip(ops, ctx.needs_input_grad)]
            if f.tokens:
                ws = _workspace(f, True, x.device)
                _lib.check(_lib.load().came8_gated_ffn_backward(
                    ctypes.byref(f), *(t.data_ptr() for t in ops), dy.data_ptr(), g.data_ptr(), u.data_ptr(),
                    *(t.data_ptr() if t is not None else None for t in grads), ws.data_ptr(), ws.numel(),
                    torch.cuda.current_stream(x.device).cuda_stream), "came8_gated_ffn_backward")
        return (*grads, None)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T`` over the last dimension of ``x``.

    x [..., dim]; w_gate, w_up [hidden, dim]; w_down [out, hidden]: one type (float32, bfloat16 or float16), one GPU.
    activation: "silu", "gelu" (by erf) or "gelu_tanh".  Differentiable once in every operand.  Operands whose rows are
    contiguous are read where they are, with the row strides they have; others are copied.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError(f"gated_ffn: came_amd runs on the GPU; {name} is "
                               f"{f'a {t.device} tensor' if isinstance(t, torch.Tensor) else type(t).__name__}")
        if t.dtype not in _DTYPE_CODE:
            raise RuntimeError(f"gated_ffn: unsupported dtype {t.dtype} of {name} (float32, bfloat16 and float16 are supported)")
        if t.dtype != x.dtype or t.device != x.device:
            raise RuntimeError(f"gated_ffn: {name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.dim() != 2:
        raise ValueError(f"gated_ffn: x [..., dim], w_gate and w_up [hidden, dim], w_down [out, hidden]; got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if x.shape[-1] != w_gate.shape[1] or w_down.shape[1] != w_gate.shape[0] or 0 in (*w_gate.shape, *w_down.shape):
        raise ValueError(f"gated_ffn: widths do not match or are empty: {tuple(x.shape)}, {tuple(w_gate.shape)}, "
                         f"{tuple(w_down.shape)}")
    act = ACTIVATIONS[activation]
    rows = x.reshape(-1, x.shape[-1])
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down)):
        y = _GatedFFN.apply(rows, w_gate, w_up, w_down, act)
    else:
        y = _forward(rows, w_gate, w_up, w_down, act, False)[0]
    return y.view(*x.shape[:-1], w_down.shape[0])
