"""Embedding, root-mean-square norm, 8-bit rows and their product, and token log probabilities in 64 bits on CPU tensors, with
bounds on what rounding may change.

The bounds follow one evaluation in float32, U = 2^-24 a rounding, with every result rounded to its type once (``UNIT``).  A
sum of n terms in any order is off by at most n U of the sum of magnitudes; a row's sums go through CHAIN additions at most (the
elements of a thread, the lanes of a wavefront, the wavefronts).  The hardware's exponential is off by 2 U, and its argument's
roundings by 2 U of the argument."""
import numpy as np
import torch

U = 2.0**-24
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 2.0**-150, torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}  # half of the least subnormal
CHAIN = 100


def rounded(bound, value, dtype):
    """A bound with the result's own rounding."""
    return bound * (1 + 2 * UNIT[dtype]) + UNIT[dtype] * value.abs() + LEAST[dtype]


def embedding(tokens, weight, scale):
    """Exactly what is returned: a product in float32, rounded once."""
    t, V = tokens.cpu().long(), weight.shape[0]
    inside = (t >= 0) & (t < V)
    y = (weight.detach().cpu()[t.clamp(0, V - 1)].float() * torch.tensor(scale, dtype=torch.float32)).to(weight.dtype)
    return torch.where(inside[..., None], y, torch.zeros_like(y))


def embedding_gradient(tokens, dy, vocab, scale, padding=None):
    """(dweight, bound)"""
    t, d = tokens.cpu().long().reshape(-1), dy.detach().cpu().double().reshape(-1, dy.shape[-1])
    keep = (t >= 0) & (t < vocab)
    if padding is not None:
        keep &= t != padding
    t, d = t[keep], d[keep]
    s = float(torch.tensor(scale, dtype=torch.float32))
    dw = torch.zeros(vocab, d.shape[1], dtype=torch.float64).index_add_(0, t, d) * s
    mag = torch.zeros_like(dw).index_add_(0, t, d.abs()) * abs(s)
    n = torch.zeros(vocab, 1, dtype=torch.float64).index_add_(0, t, torch.ones(len(t), 1, dtype=torch.float64))
    return dw, rounded(n * U * mag, dw, dy.dtype)


def rms_norm(x, weight, eps, residual=None):
    """(y, bound before y's rounding, h)"""
    x = x.detach().cpu()
    h = x if residual is None else (x.float() + residual.detach().cpu().float()).to(x.dtype)
    hd, w = h.double(), weight.detach().cpu().double()
    e = float(torch.tensor(eps, dtype=torch.float32))
    y = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + e) * w
    return y, (CHAIN / 2 + 6) * U * y.abs(), h


def rms_norm_gradients(h, weight, eps, dy, dh=None):
    """((dx, bound), (dweight, bound))"""
    hd, w, g = h.detach().cpu().double(), weight.detach().cpu().double(), dy.detach().cpu().double()
    D = hd.shape[-1]
    e = float(torch.tensor(eps, dtype=torch.float32))
    r = 1 / torch.sqrt(hd.square().mean(-1, keepdim=True) + e)
    er = (CHAIN / 2 + 4) * U  # of r, relative
    gw = g * w
    s, mag = (gw * hd).sum(-1, keepdim=True), (gw * hd).abs().sum(-1, keepdim=True)
    c, ec = r * r * s / D, r * r / D * ((CHAIN + 1) * U * mag + (2 * er + 4 * U) * s.abs())
    dx = r * (gw - hd * c)
    ex = r * (2 * U * gw.abs() + hd.abs() * ec + U * (gw.abs() + (hd * c).abs())) + (er + 2 * U) * dx.abs()
    if dh is not None:
        d = dh.detach().cpu().double()
        ex = ex + U * (dx.abs() + d.abs())
        dx = dx + d
    terms = (g * hd * r).reshape(-1, D)
    dw = terms.sum(0)
    ew = (er + (len(terms) + CHAIN) * U) * terms.abs().sum(0)
    return (dx, rounded(ex, dx, dy.dtype)), (dw, rounded(ew, dw, dy.dtype))


def codes(p, top):
    """127 p / top to nearest, ties to even, exactly, where p and top are products of two float32 values (48 bits): next to a border
    between two codes, border * top and 127 p are compared in numbers of 64 bits' mantissa, which hold both (56 and 55)."""
    q = p * 127 / top
    lower = torch.floor(q)
    near = (q - lower - 0.5).abs() < 1e-9
    out = torch.round(q)
    if near.any():
        assert np.finfo(np.longdouble).nmant >= 63
        k, v, a = (t[near].numpy().astype(np.longdouble) for t in (lower, p, top.expand_as(p)))
        above = 127 * v - (k + np.longdouble(0.5)) * a
        up = (above > 0) | ((above == 0) & (k % 2 != 0))
        out[near] = torch.from_numpy((k + up).astype(np.float64))
    return out


def quantize_rows(x):
    """(codes, scales) of values x, or of products of two of them; the scales unrounded."""
    x = x.detach().cpu().double()
    top = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top) & (top >= 2.0**-100)
    q = torch.where(fine, codes(torch.where(fine, x, 0.0), torch.where(fine, top, 1.0)), 0.0).to(torch.int8)
    return q, torch.where(top < 2.0**-100, torch.zeros_like(top), top / 127).squeeze(-1)


def rms_norm_int8(x, weight, eps, residual=None):
    """(codes, scales, bound of the scales, h): codes as quantize_rows has them of h weight, which the norm scales as a whole"""
    y, _, h = rms_norm(x, weight, eps, residual)
    p = h.double() * weight.detach().cpu().double()
    q, _ = quantize_rows(p)
    s = y.abs().amax(-1) / 127
    s = torch.where(p.abs().amax(-1) < 2.0**-100, torch.zeros_like(s), s)
    return q, s, (CHAIN / 2 + 8) * U * s, h


def int8_linear(q, scale, wq, ws, bias, dtype):
    """(y, bound)"""
    acc = q.cpu().double() @ wq.cpu().double().t()
    y = acc * scale.cpu().double()[..., None] * ws.cpu().double()
    e = 3 * U * y.abs()
    if bias is not None:
        b = bias.cpu().double()
        e = e + U * (y + b).abs() + e * U
        y = y + b
    return y, rounded(e, y, dtype)


def log_probs(logits, tokens):
    """((log_probs, bound), (entropy, bound), kept): the bounds of float32 results; kept: for log_probs_gradient"""
    z, t = logits.detach().cpu().double(), tokens.cpu().long()
    m = z.amax(-1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    far = torch.where(e > 0, d, torch.zeros_like(d)).abs()
    s, first, second = e.sum(-1), (e * far).sum(-1), (e * far * far).sum(-1)
    l = torch.log(s)
    es = U * (4 * first / s + 4 + CHAIN)  # of s, relative
    el = es + 2 * U * l.abs() + U
    H = l + first / s
    eh = el + U * (4 * second + (6 + CHAIN) * first) / s + first / s * (es + 2 * U) + U * H.abs()
    logp = d - l[..., None]
    given = (t >= 0) & (t < z.shape[-1])
    lp = logp.gather(-1, t.clamp(0, z.shape[-1] - 1)[..., None]).squeeze(-1)
    dl = lp + l  # z[token] - m
    elp = el + U * (dl.abs() + lp.abs())
    none = torch.zeros_like(lp)
    return (torch.where(given, lp, none), torch.where(given, elp, none)), (H, eh), (logp, el, H, eh, given, t)


def log_probs_gradient(kept, dlp, dent, dtype):
    """(dlogits, bound)"""
    logp, el, H, eh, given, t = kept
    col = lambda v: v[..., None]  # noqa: E731
    g = col(torch.where(given, dlp.cpu().double(), torch.zeros_like(H))) if dlp is not None else torch.zeros_like(col(H))
    gh = col(dent.cpu().double()) if dent is not None else torch.zeros_like(col(H))
    p = torch.exp(logp)
    lp = torch.where(p > 0, logp, torch.zeros_like(logp))
    dz = -p * (g + gh * (lp + col(H)))
    elp = col(el) + 2 * U * (lp.abs() + lp.abs())
    ep = elp + U * (4 * lp.abs() + 4)  # of p, relative
    mag = g.abs() + gh.abs() * (lp.abs() + col(H).abs())
    bound = p * ((ep + 5 * U) * mag + gh.abs() * (elp + col(eh)))
    one = torch.zeros_like(p).scatter_(-1, col(t.clamp(0, p.shape[-1] - 1)), 1.0)
    bound = bound + U * one * (g.abs() + mag * p)
    return dz + one * g, rounded(bound, dz + one * g, dtype)
