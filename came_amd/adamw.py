"""AdamW whose step runs in libcame8: every tensor of a param group in one multi-tensor launch.

  * ``AdamW``     -- fp32 moments (``exp_avg``, ``exp_avg_sq``), whatever the parameter type
  * ``AdamW8bit`` -- moments of one byte an element with a float32 scale per block (``exp_avg_q``, ``exp_avg_absmax``,
    ``exp_avg_sq_q``, ``exp_avg_sq_absmax``)

The update is that of ``torch.optim.AdamW`` (decoupled weight decay).  ``max_grad_norm`` clips by the norm over all
gradients of the optimizer inside the step: the gradients are scaled as they are read and are not changed.  A step counts
as a write to the parameters: a backward pass through a node that saved them before it raises.  Parameters must live on the
GPU.  The step count is a host number that enters the bias corrections, so a step cannot be captured in a HIP graph and
replayed.
"""
from __future__ import annotations

import ctypes
from itertools import chain

import torch
import torch.optim

from . import _lib
from .blockwise_quantization import init_qstate, num_blocks
from .grad_clip import _DTYPE_CODE, _reduce


def _refuse_options(group: dict) -> None:
    """Options of torch.optim.AdamW that change its update and that the step here does not have."""
    for option in ("amsgrad", "maximize"):
        if group.get(option):
            raise ValueError(f"param group with {option}=True: AdamW (came_amd) does not have this option")


class _AdamWBase(torch.optim.Optimizer):
    _BITS = 32
    _KEYS: dict = {}  # state tensors and their types

    def __init__(self, params, lr, betas, eps, weight_decay, max_grad_norm, **more):
        if not lr >= 0.0:
            raise ValueError(f"lr must be >= 0, got {lr}")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must be two numbers in [0, 1), got betas={betas}")
        if not eps >= 0.0:
            raise ValueError(f"eps must be >= 0, got {eps}")
        if not weight_decay >= 0.0:
            raise ValueError(f"weight_decay must be >= 0, got {weight_decay}")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"max_grad_norm must be >= 0 or None, got {max_grad_norm}")
        super().__init__(params, dict(lr=float(lr), betas=(float(betas[0]), float(betas[1])), eps=float(eps),
                                      weight_decay=float(weight_decay), **more))
        self.max_grad_norm = max_grad_norm
        self.last_grad_norm = None  # of the last step with max_grad_norm: a device scalar, before the clip

    def __getstate__(self) -> dict:  # of copies and pickles
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm}

    def __setstate__(self, state: dict) -> None:  # also torch's loading of a state_dict, without the bound
        super().__setstate__(state)
        self.__dict__.setdefault("max_grad_norm", None)
        self.last_grad_norm = None

    def add_param_group(self, param_group: dict) -> None:
        if isinstance(param_group, dict):  # torch refuses others
            _refuse_options(param_group)
            params = param_group.get("params")
            if not isinstance(params, (torch.Tensor, set, type(None))):
                params = param_group["params"] = list(params)
                each = [p[1] if isinstance(p, tuple) else p for p in params]  # named ones are pairs
                if len({id(p) for p in each}) != len(each):  # torch warns
                    raise ValueError("a parameter appears twice in a param group: one launch would step it twice at the same time")
        super().add_param_group(param_group)

    # ------------------------------------------------------------------ state
    def _init_state(self, state: dict, p: torch.Tensor, group: dict) -> None:
        raise NotImplementedError

    def _moments(self, state: dict, p: torch.Tensor, group: dict):
        """The state tensors in the order of the descriptor's fields, checked."""
        B = self._block_size(group)
        out = []
        for key, dtype in self._KEYS.items():
            t = state.get(key)
            n = num_blocks(p.numel(), B) if key.endswith("absmax") else p.numel()
            if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.numel() != n or not t.is_contiguous():
                raise RuntimeError(f"{key} state does not have the layout of this parameter and optimizer "
                                   f"(contiguous {dtype}, {n} elements)")
            if t.device != p.device:
                raise RuntimeError("optimizer state lives on a different device than its parameter")
            out.append(t)
        return out

    @staticmethod
    def _block_size(group: dict) -> int:
        return int(group.get("block_size", 256))

    def load_state_dict(self, state_dict: dict) -> None:
        """Loads every state tensor in the type it was saved in (torch's loader casts them to the parameter's), contiguous (torch
        keeps the moments of a transposed or channels-last parameter in its order).  What is refused leaves the optimizer as it
        was."""
        loaded: dict = {}
        handle = self.register_load_state_dict_pre_hook(lambda _, given: self._look_over(given, loaded))  # after the user's
        try:
            super().load_state_dict(state_dict)
        finally:
            handle.remove()
        for p, st in loaded.items():
            self.state[p].update(st)

    def _look_over(self, state_dict: dict, loaded: dict) -> None:
        """What a state_dict holds for each parameter, checked before anything changes."""
        groups, saved = state_dict["param_groups"], state_dict["state"]
        for g in groups:
            _refuse_options(g)
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            return  # torch's loader raises
        for g, own in zip(groups, self.param_groups):
            for k, p in zip(g["params"], own["params"]):
                if not saved.get(k):
                    continue
                st = loaded[p] = {}
                for key, v in saved[k].items():
                    if key == "step":  # torch.optim keeps a tensor
                        st[key] = int(v)
                    elif isinstance(v, torch.Tensor):
                        st[key] = v.detach().to(device=p.device, copy=True, memory_format=torch.contiguous_format)
                self._moments(st, p, g)

    # ------------------------------------------------------------------- step
    def _hparams(self, group: dict) -> _lib.Came8AdamwHParams:
        b1, b2 = group["betas"]
        return _lib.Came8AdamwHParams(float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                      float(group["weight_decay"]), self._BITS, self._block_size(group),
                                      int(group.get("seed", 0)) & 0xFFFFFFFF, 0)

    def _descriptors(self, group: dict):
        """{device: (descriptors, how many, [(parameter, contiguous copy or None, gradient, state)])} of the group's parameters with
        gradients: the copies are to be written back, and the states' steps to be counted, once the step is launched."""
        lists: dict = {}
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            if g.is_sparse:
                raise RuntimeError("AdamW does not support sparse gradients.")
            if not p.is_cuda:
                raise RuntimeError(
                    f"{type(self).__name__} (came_amd) runs the step on the GPU; got a parameter on {p.device}")
            if p.dtype not in _DTYPE_CODE or g.dtype not in _DTYPE_CODE:
                raise RuntimeError(f"unsupported dtype: param {p.dtype}, grad {g.dtype} "
                                   "(float32, bfloat16 and float16 are supported)")
            if g.shape != p.shape or g.device != p.device:
                raise RuntimeError(f"grad {tuple(g.shape)} on {g.device} does not match param {tuple(p.shape)} on {p.device}")
            state = self.state[p]
            if len(state) == 0:
                self._init_state(state, p, group)
            moments = self._moments(state, p, group)
            lists.setdefault(p.device, []).append((p, g, state, moments))
        out = {}
        for device, items in lists.items():
            descs, used, k = (_lib.Came8AdamwTensor * len(items))(), [], 0
            for p, g, state, moments in items:
                copy = None if p.data.is_contiguous() else p.data.contiguous()
                g = g.resolve_neg().contiguous()
                used.append((p, copy, g, state))
                if p.numel() == 0:
                    continue
                d = descs[k]
                k += 1
                d.param, d.grad = (p.data if copy is None else copy).data_ptr(), g.data_ptr()
                d.numel, d.step = p.numel(), state["step"] + 1
                d.param_dtype, d.grad_dtype = _DTYPE_CODE[p.dtype], _DTYPE_CODE[g.dtype]
                for (name, _), t in zip(self._KEYS.items(), moments):
                    setattr(d, name.removesuffix("_q"), t.data_ptr())
            out[device] = (descs, k, used)
        return out

    def _launch(self, device, descs, n: int, group: dict, factor) -> None:
        if n == 0:
            return
        hp = self._hparams(group)
        with torch.cuda.device(device):
            _lib.check(_lib.load().came8_adamw_step(descs, n, ctypes.byref(hp), factor.data_ptr() if factor is not None else None,
                                                    torch.cuda.current_stream(device).cuda_stream), "came8_adamw_step")

    def _step_native(self, group: dict, factor) -> bool:
        """The group's step, descriptors and all, natively (csrc/came8_host.cpp); False: the Python has to take it."""
        params = group["params"]
        device = next((p.device for p in params if p.grad is not None), None)
        if device is None:
            return True
        if type(params) is not list or device.type != "cuda":
            return False
        hp = self._hparams(group)
        return bool(_lib.host().adamw_step(
            params, self.state, hp.bits, hp.block_size, hp.seed, hp.lr, hp.beta1, hp.beta2, hp.eps, hp.weight_decay,
            factor.data_ptr() if factor is not None else 0, torch.cuda.current_stream(device).cuda_stream))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{type(self).__name__}.step() cannot be captured: its step count is a host number")
        factor = None
        if self.max_grad_norm is not None:
            every = list(chain.from_iterable(group["params"] for group in self.param_groups))
            found = _reduce(every, self.max_grad_norm, False, type(self).__name__, True)
            if found is None:
                return loss
            self.last_grad_norm, factor = found
        for group in self.param_groups:
            if self._step_native(group, factor):
                continue
            for device, (descs, n, used) in self._descriptors(group).items():
                self._launch(device, descs, n, group, factor)
                for p, copy, _, state in used:
                    state["step"] += 1
                    if copy is not None:
                        p.data.copy_(copy)
                torch.autograd.graph.increment_version([p for p, *_ in used])
        return loss


class AdamW(_AdamWBase):
    """AdamW with float32 moments."""

    _KEYS = {"exp_avg": torch.float32, "exp_avg_sq": torch.float32}

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, max_grad_norm: float | None = None):
        super().__init__(params, lr, betas, eps, weight_decay, max_grad_norm)

    def _init_state(self, state: dict, p: torch.Tensor, group: dict) -> None:
        state["step"] = 0
        for key in self._KEYS:
            state[key] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)


class AdamW8bit(_AdamWBase):
    """AdamW with moments of one byte an element (include/came8.h: came8_adamw_tensor).

    The first moment is held as the other optimizers' momentum is (int8 codes, blockwise absmax), the second as 8-bit
    floats relative to its block's largest, rounded at random in proportion, from a hash of ``seed``, the step count and
    the element: runs repeat bit for bit.
    """

    _BITS = 8
    _KEYS = {"exp_avg_q": torch.int8, "exp_avg_sq_q": torch.uint8, "exp_avg_absmax": torch.float32,
             "exp_avg_sq_absmax": torch.float32}

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, max_grad_norm: float | None = None, block_size: int = 256, seed: int = 0):
        if block_size not in (64, 128, 256, 512, 1024, 2048):
            raise ValueError(f"block_size must be a power of two in [64, 2048], got {block_size}")
        if not eps >= 2.0**-126:
            raise ValueError(f"eps must be > 0 with 8-bit moments (a normal float32 number), got {eps}")
        super().__init__(params, lr, betas, eps, weight_decay, max_grad_norm, block_size=int(block_size), seed=int(seed))

    def _init_state(self, state: dict, p: torch.Tensor, group: dict) -> None:
        B = self._block_size(group)
        state["step"] = 0
        state["exp_avg_q"], state["exp_avg_absmax"] = init_qstate(p.shape, device=p.device, signed=True, block_size=B)
        state["exp_avg_sq_q"], state["exp_avg_sq_absmax"] = init_qstate(p.shape, device=p.device, signed=False,
                                                                        block_size=B)
