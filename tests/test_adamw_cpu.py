"""What AdamW, AdamW8bit and the gradient clip refuse, on the host: constructor arguments, tensors that are not on the GPU,
and the C entries' argument checks (before any device work)."""
import ctypes

import pytest
import torch

import came_amd
from came_amd import _lib as L


@pytest.mark.parametrize("kw,match", [
    (dict(lr=-1.0), "lr"), (dict(betas=(0.9, 1.0)), "betas"), (dict(betas=(0.9,)), "betas"), (dict(eps=-1e-8), "eps"),
    (dict(weight_decay=-0.1), "weight_decay"), (dict(max_grad_norm=-1.0), "max_grad_norm"),
    (dict(lr=float("nan")), "lr"),
])
@pytest.mark.parametrize("cls", [came_amd.AdamW, came_amd.AdamW8bit])
def test_constructor_refuses(cls, kw, match):
    with pytest.raises(ValueError, match=match):
        cls([torch.nn.Parameter(torch.zeros(3))], **kw)


@pytest.mark.parametrize("kw,match", [(dict(block_size=100), "block_size"), (dict(block_size=32), "block_size"),
                                      (dict(block_size=4096), "block_size"), (dict(eps=0.0), "eps"),
                                      (dict(eps=1e-40), "eps")])
def test_8bit_constructor_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        came_amd.AdamW8bit([torch.nn.Parameter(torch.zeros(3))], **kw)


@pytest.mark.parametrize("cls", [came_amd.AdamW, came_amd.AdamW8bit])
def test_cpu_parameters_raise(cls):
    p = torch.nn.Parameter(torch.zeros(3))
    opt = cls([p])
    opt.step()  # no gradient: nothing to do
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="on the GPU"):
        opt.step()
    p.grad = torch.ones(3).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()


def test_clip_refuses():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="on the GPU"):
        came_amd.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        came_amd.clip_grad_norm_([p], -1.0)
    with pytest.raises(RuntimeError, match="on the GPU"):
        came_amd.grad_norm(torch.ones(3))
    assert float(came_amd.grad_norm([])) == 0.0


def _adamw_desc(**kw):
    d = L.Came8AdamwTensor()
    d.param, d.grad, d.exp_avg, d.exp_avg_sq = 0x1000, 0x2000, 0x3000, 0x4000
    d.exp_avg_absmax, d.exp_avg_sq_absmax = 0x5000, 0x6000
    d.numel, d.step = 100, 1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _hp(**kw):
    h = L.Came8AdamwHParams(1e-3, 0.9, 0.999, 1e-8, 1e-2, 8, 256, 0, 0)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("desc,hp,match", [
    (dict(param=None), {}, "null"), (dict(grad=0x2002), {}, "misaligned"), (dict(exp_avg_sq=None), {}, "null"),
    (dict(exp_avg_absmax=None), {}, "absmax"), (dict(numel=-1), {}, "numel"), (dict(numel=1 << 40), {}, "numel"),
    (dict(step=0), {}, "step"), (dict(param_dtype=7), {}, "dtype"), ({}, dict(bits=4), "bits"),
    ({}, dict(block_size=96), "block_size"), ({}, dict(block_size=32), "block_size"), ({}, dict(eps=0.0), "eps"),
    ({}, dict(beta2=1.0), "betas"), ({}, dict(lr=float("nan")), "lr"), ({}, dict(flags=1), "flags"),
    (dict(exp_avg=0x3001), dict(bits=32), "misaligned"),
])
def test_adamw_entry_refuses(desc, hp, match):
    lib = L.load()
    d, h = _adamw_desc(**desc), _hp(**hp)
    assert lib.came8_adamw_step(ctypes.byref(d), 1, ctypes.byref(h), None, None) == L.CAME8_EINVAL
    assert match in lib.came8_last_error().decode()


def test_adamw_entry_with_nothing_to_do():
    lib = L.load()
    d = _adamw_desc(numel=0, param=None, grad=None)
    assert lib.came8_adamw_step(None, -1, ctypes.byref(_hp()), None, None) == L.CAME8_EINVAL
    assert lib.came8_adamw_step(ctypes.byref(d), 1, None, None, None) == L.CAME8_EINVAL


@pytest.mark.parametrize("kw,match", [(dict(data=None), "null"), (dict(data=0x1001), "misaligned"), (dict(numel=-5), "numel"),
                                      (dict(dtype=3), "dtype")])
@pytest.mark.parametrize("name", ["came8_grad_norm", "came8_grad_clip"])
def test_norm_entries_refuse(name, kw, match):
    lib = L.load()
    d = L.Came8GradTensor(0x1000, 10, 0, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    call = getattr(lib, name)
    size = lib.came8_grad_norm_workspace_size(1)
    assert call(ctypes.byref(d), 1, 1.0, 0x100, 0x104, 0x1000, size, None) == L.CAME8_EINVAL
    assert match in lib.came8_last_error().decode()
    good = L.Came8GradTensor(0x1000, 10, 0, 0)
    assert call(ctypes.byref(good), 1, 1.0, 0x100, 0x104, 0x1000, size - 1, None) == L.CAME8_ESPACE
    assert call(ctypes.byref(good), 1, -1.0, 0x100, 0x104, 0x1000, size, None) == L.CAME8_EINVAL
    assert call(ctypes.byref(good), 1, 1.0, None, 0x104, 0x1000, size, None) == L.CAME8_EINVAL


def test_norm_workspace_grows_with_the_list():
    lib = L.load()
    assert 0 < lib.came8_grad_norm_workspace_size(0) == lib.came8_grad_norm_workspace_size(192)
    assert lib.came8_grad_norm_workspace_size(193) == 2 * lib.came8_grad_norm_workspace_size(1)


def test_second_moment_entry_refuses():
    lib = L.load()
    assert lib.came8_dequantize_second_moment(0x1000, 0x1000, 5, 0, 0x1000, None) == L.CAME8_EINVAL
    assert lib.came8_dequantize_second_moment(None, 0x1000, 5, 64, 0x1000, None) == L.CAME8_EINVAL
    assert lib.came8_dequantize_second_moment(None, None, 0, 64, None, None) == L.CAME8_OK
    with pytest.raises(RuntimeError, match="on the GPU"):
        came_amd.blockwise_quantization.dequantize_second_moment(torch.zeros(3, dtype=torch.uint8), torch.ones(1), block_size=64)
