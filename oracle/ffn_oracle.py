"""The gated feed-forward block and its gradients in 64 bits on CPU tensors, with bounds on what rounding may change.

The bounds follow one evaluation in float32 sums of n terms (an error of at most (n + 4) 2^-24 of the sum of absolute
values, in any order), with h, dg, du and the results rounded to the type once (unit ``ut``), and activations evaluated
in float32 within 32 units of the magnitudes that enter them."""
import math

import torch

U = 2.0**-24
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LIP1, LIP2 = 1.13, 0.8  # the steepest slope of the three activations, and of their derivatives


def act(g, name):
    """(value, derivative)"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if name == "gelu":
        c = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g**3))
    return g * (1 + t) / 2, (1 + t) / 2 + g / 2 * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def forward(x, wg, wu, wd, name, dtype=None):
    """y, and with a dtype (y, bound of y, what backward() needs)"""
    x, wg, wu, wd = (t.detach().cpu().double() for t in (x, wg, wu, wd))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = act(g, name)
    h = a * u
    y = h @ wd.t()
    if dtype is None:
        return y
    ut, sub = UNIT[dtype], 2.0**-25 if dtype == torch.float16 else 0.0
    D, F = x.shape[1], wd.shape[1]
    eg = (D + 4) * U * (x.abs() @ wg.abs().t())
    eu = (D + 4) * U * (x.abs() @ wu.abs().t())
    ea = LIP1 * eg + 32 * U * g.abs()
    eh = u.abs() * ea + a.abs() * eu + ea * eu + (ut + 4 * U) * h.abs() + sub
    ey = (1 + ut) * (eh @ wd.abs().t() + (F + 4) * U * (h.abs() + eh) @ wd.abs().t()) + ut * y.abs() + sub
    return y, ey, (x, wg, wu, wd, g, u, a, da, h, eg, eu, ea, eh, ut, sub)


def backward(kept, dy):
    """{name: (gradient, bound)} of x, w_gate, w_up and w_down"""
    x, wg, wu, wd, g, u, a, da, h, eg, eu, ea, eh, ut, sub = kept
    dy = dy.detach().cpu().double()
    T, F, E = x.shape[0], wd.shape[1], wd.shape[0]
    dh = dy @ wd
    du, dg = dh * a, dh * u * da
    edh = (E + 4) * U * (dy.abs() @ wd.abs())
    eda = LIP2 * eg + 32 * U * (1 + g.abs())
    edu = a.abs() * edh + (dh.abs() + edh) * ea + (ut + 4 * U) * du.abs() + sub
    edg = ((u * da).abs() * edh + (dh.abs() + edh) * (da.abs() * eu + (u.abs() + eu) * eda) + (ut + 8 * U) * dg.abs() + sub)
    out = {}

    def product(name, value, pairs, n):
        e = sum(eb.t().abs() @ w if t else eb @ w for eb, w, t, _ in pairs)
        s = sum((v.abs() + eb).t() @ w if t else (v.abs() + eb) @ w for eb, w, t, v in pairs)
        out[name] = value, (1 + ut) * (e + (n + 4) * U * s) + ut * value.abs() + sub

    product("x", dg @ wg + du @ wu, [(edg, wg.abs(), False, dg), (edu, wu.abs(), False, du)], 2 * F)
    product("w_gate", dg.t() @ x, [(edg, x.abs(), True, dg)], T)
    product("w_up", du.t() @ x, [(edu, x.abs(), True, du)], T)
    e = dy.abs().t() @ eh
    s = dy.abs().t() @ (h.abs() + eh)
    v = dy.t() @ h
    out["w_down"] = v, (1 + ut) * (e + (T + 4) * U * s) + ut * v.abs() + sub
    return out
