"""What the gated feed-forward block refuses on the host, and the oracle's gradients against automatic differentiation."""
import ctypes

import pytest
import torch

import came_amd
from came_amd import _lib as L
from oracle import ffn_oracle as orc


def _ffn(**kw):
    f = L.Came8Ffn(4, 8, 16, 8, 8, 8, 8, 16, L.CAME8_BF16, 0)
    for k, v in kw.items():
        setattr(f, k, v)
    return f


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(activation=3), "activation"), (dict(activation=-1), "activation"), (dict(tokens=-1), "tokens"),
    (dict(tokens=1 << 25), "tokens"), (dict(dim=0, ld_x=0, ld_gate=0, ld_up=0), "dim"), (dict(hidden=0), "hidden"),
    (dict(out=0), "out"), (dict(out=1 << 22), "out"), (dict(ld_x=7), "stride"), (dict(ld_gate=7), "stride"),
    (dict(ld_up=1 << 22), "stride"), (dict(ld_down=15), "stride"),
    (dict(tokens=1 << 24, hidden=1 << 20, ld_down=1 << 20), "2\\^36"),
])
def test_entries_refuse_shapes(kw, match):
    lib, f, size = L.load(), _ffn(**kw), ctypes.c_size_t(0)
    assert lib.came8_gated_ffn_workspace_size(ctypes.byref(f), 0, ctypes.byref(size)) == L.CAME8_EINVAL
    p = [0x1000] * 5
    assert lib.came8_gated_ffn_forward(ctypes.byref(f), *p, None, None, 0x1000, 1 << 40, None) == L.CAME8_EINVAL
    with pytest.raises(RuntimeError, match=match):
        L.check(lib.came8_gated_ffn_backward(ctypes.byref(f), *p, *[0x1000] * 6, 0x1000, 1 << 40, None), "backward")


def test_entries_refuse_pointers_and_workspaces():
    lib, f, size = L.load(), _ffn(), ctypes.c_size_t(0)
    assert lib.came8_gated_ffn_workspace_size(ctypes.byref(f), 0, None) == L.CAME8_EINVAL
    assert lib.came8_gated_ffn_workspace_size(ctypes.byref(f), 0, ctypes.byref(size)) == L.CAME8_OK
    need = size.value
    assert lib.came8_gated_ffn_workspace_size(ctypes.byref(f), 1, ctypes.byref(size)) == L.CAME8_OK
    assert size.value >= 3 * 4 * 16 * 2
    p = [0x1000] * 5
    for i in range(5):
        for bad in (None, 0x1002):
            q = list(p)
            q[i] = bad
            assert lib.came8_gated_ffn_forward(ctypes.byref(f), *q, None, None, 0x1000, need, None) == L.CAME8_EINVAL
            assert lib.came8_gated_ffn_backward(ctypes.byref(f), *q, *[0x1000] * 6, 0x1000, size.value, None) == L.CAME8_EINVAL
    assert lib.came8_gated_ffn_forward(ctypes.byref(f), *p, 0x1000, None, 0x1000, need, None) == L.CAME8_EINVAL
    assert lib.came8_gated_ffn_backward(ctypes.byref(f), *p, None, 0x1000, *[0x1000] * 4, 0x1000, size.value, None) == L.CAME8_EINVAL
    assert lib.came8_gated_ffn_backward(ctypes.byref(f), *p, 0x1000, 0x1000, 0x1002, None, None, None, 0x1000, size.value,
                                        None) == L.CAME8_EINVAL
    assert lib.came8_gated_ffn_forward(ctypes.byref(f), *p, None, None, 0x1000, 100, None) == L.CAME8_ESPACE
    assert lib.came8_gated_ffn_forward(ctypes.byref(f), *p, None, None, None, need, None) == L.CAME8_ESPACE
    assert lib.came8_gated_ffn_backward(ctypes.byref(f), *p, *[0x1000] * 6, 0x1004, size.value, None) == L.CAME8_ESPACE
    empty = _ffn(tokens=0)
    assert lib.came8_gated_ffn_forward(ctypes.byref(empty), *p, None, None, None, 0, None) == L.CAME8_OK


def test_cpu_tensors_raise():
    x, w = torch.zeros(2, 8), torch.zeros(16, 8)
    with pytest.raises(RuntimeError, match="on the GPU"):
        came_amd.gated_ffn(x, w, w, w.t().contiguous())
    with pytest.raises(ValueError, match="activation"):
        came_amd.gated_ffn(x, w, w, w.t(), activation="tanh")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_oracle_gradients(act):
    gen = torch.Generator().manual_seed(0)
    x, wg, wu, wd, dy = (torch.randn(*s, generator=gen, dtype=torch.float64)
                         for s in ((5, 7), (11, 7), (11, 7), (3, 11), (5, 3)))
    F = torch.nn.functional
    fn = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[act]
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = F.linear(fn(F.linear(leaves[0], leaves[1])) * F.linear(leaves[0], leaves[2]), leaves[3])
    want = torch.autograd.grad(y, leaves, dy)
    got, _, kept = orc.forward(x, wg, wu, wd, act, torch.float32)
    grads = orc.backward(kept, dy)
    assert torch.allclose(got, y, rtol=1e-12, atol=1e-12)
    for w, name in zip(want, ("x", "w_gate", "w_up", "w_down")):
        assert torch.allclose(grads[name][0], w, rtol=1e-11, atol=1e-12), name
