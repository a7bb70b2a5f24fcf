"""Plain statements of AdamW with fp32 and 8-bit moments and of the gradient clip, on CPU tensors.

``moments64`` and ``param64`` are the definition in 64 bits from a given state.  ``step8_f32`` restates the 8-bit step's moments in float32,
operation by operation (elementwise torch operations round each result and contract none), so that codes can be compared
for equality."""
import math

import torch

TINY = 2.0**-100
MASK = 0xFFFFFFFF


def _mix(x):
    x = (x * 0x9E3779B1) & MASK
    x = x ^ (x >> 15)
    x = (x * 0x85EBCA77) & MASK
    return x ^ (x >> 13)


def random_bits(n, seed, step):
    """20 random bits an element, 16 of them from a hash of (seed, step, the element's pair)."""
    i = torch.arange(n, dtype=torch.int64)
    x = _mix(((i >> 1) & MASK) ^ _mix(_mix(seed & MASK) ^ (step & MASK)))
    return torch.where(i % 2 == 1, x >> 16, x & 0xFFFF) << 4 | 8


def code_values():
    """What the 256 codes of a second moment stand for, in units of 8/15 of their block's largest (64 bits)."""
    c = torch.arange(256, dtype=torch.float64)
    return torch.where(c < 8, c * 2.0**-33, (1 + c % 8 / 8) * torch.pow(2.0, torch.floor(c / 8) - 31))


def _blocks(x, B):
    x = x.reshape(-1)
    return torch.cat([x, x.new_zeros(-x.numel() % B)]).view(-1, B)


def decode64(mq, ma, vq, va, B):
    n = mq.numel()
    m = mq.reshape(-1).double() * (ma.double() / 127).repeat_interleave(B)[:n]
    v = code_values()[vq.reshape(-1).long()] * (va.double() * 8 / 15).repeat_interleave(B)[:n]
    return m, v


def moments64(g, m, v, betas, scale=1.0):
    """(m, v) after a step in 64 bits; every argument flat."""
    b1, b2 = betas
    g = g.double() * scale
    return b1 * m.double() + (1 - b1) * g, b2 * v.double() + (1 - b2) * g * g


def param64(p, m, v, t, lr, betas, eps, wd):
    """p after step t in 64 bits, from the moments after it."""
    b1, b2 = betas
    m, v = m.double(), v.double()
    return p.double() * (1 - lr * wd) - lr / (1 - b1**t) * m / ((v / (1 - b2**t)).sqrt() + eps)


def step8_f32(g, mq, ma, vq, va, t, betas, seed, B, scale=None):
    """((mq, ma, vq, va), m, v) after a step, in float32 as the library computes them; m, v as they enter p."""
    b1, b2 = betas
    n = g.numel()
    f = torch.float32
    g = g.reshape(-1).to(f)
    if scale is not None:
        g = g * scale
    sm = (ma / torch.full_like(ma, 127.0)).repeat_interleave(B)[:n]
    sv = (va * (8.0 / 15.0)).repeat_interleave(B)[:n]
    m = (mq.reshape(-1).to(f) * sm) * b1 + g * (1 - b1)
    v = (((vq.reshape(-1).int() << 20).view(f) * 2.0**96) * sv) * b2 + (g * g) * (1 - b2)
    mb, vb = _blocks(m, B), _blocks(v, B)
    am, av = mb.abs().amax(1, True), vb.amax(1, True)
    one = torch.ones_like(am)
    im = torch.where(am < TINY, 0 * one, (127 * one) / am)
    iv = torch.where(av < TINY, 0 * one, (1.875 * one) / av)
    am, av = torch.where(am < TINY, one, am), torch.where(av < TINY, one, av)
    q = torch.round(mb * im).clamp(-127, 127)
    bits = ((vb * iv) * 2.0**-96).view(torch.int32).long()
    c = ((bits + _blocks(random_bits(n, seed, t), B)) >> 20).clamp(max=255)
    return (q.reshape(-1)[:n].nan_to_num(0).to(torch.int8), am.reshape(-1), c.reshape(-1)[:n].to(torch.uint8),
            av.reshape(-1)), m, v


def norm64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
