"""Performance cases of what a language model has around its gated feed-forward blocks: the embedding of tokens with its
gradient, the root-mean-square norm with the residual's addition, the product of 8-bit integers that serves a trained
weight, and the log probabilities of tokens with entropy and top alternatives.

A case is a dict of plain values:

  op      "embed", "norm", "int8" or "logprob"
  dtype   of weights, activations and logits (int8: of the activations and of the product's result)
  tokens  rows;  train: with gradients or without
  vocab, dim, scale, pad
          (embed) the table's rows and width, the factor, the share of positions that hold the padding token 0
  dim, residual
          (norm) the rows' width, with a residual stream to add and return or without
  dim, out, norm, bias
          (int8) the product's widths; its activations come from the norm with the residual's addition, or are rows as
          they are
  vocab, top, masked, ignored
          (logprob) the rows' width, how many top alternatives, the share of the vocabulary (at its end) whose logits
          are -inf, the share of rows without a token

Tokens are drawn log-uniformly, which is Zipf's law: the most frequent token is a fifteenth of a text.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # the plain forms; True: the framework's operators

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
TINY = 2.0**-100  # rows whose largest is below hold zeros in 8 bits


def _embed(name, dtype, tokens, vocab, dim, train, scale=1.0, pad=0.0):
    return dict(name=name, op="embed", dtype=dtype, tokens=tokens, vocab=vocab, dim=dim, train=train, scale=scale, pad=pad)


def _norm(name, dtype, tokens, dim, residual, train):
    return dict(name=name, op="norm", dtype=dtype, tokens=tokens, dim=dim, residual=residual, train=train)


def _int8(name, dtype, tokens, dim, out, norm, bias):
    return dict(name=name, op="int8", dtype=dtype, tokens=tokens, dim=dim, out=out, norm=norm, bias=bias)


def _logprob(name, dtype, tokens, vocab, top, train, masked=0.0, ignored=0.0):
    return dict(name=name, op="logprob", dtype=dtype, tokens=tokens, vocab=vocab, top=top, train=train, masked=masked,
                ignored=ignored)


def listed():
    return [
        # a batch of sequences decodes one token each in a 7B-shape model: latency
        _embed("embed_token_bf16", "bf16", 16, 32000, 4096, False),
        # its training batch: the rows, and the gradient of the whole table
        _embed("embed_train_bf16", "bf16", 8192, 32000, 4096, True),
        # a medium model in fp32, scaled embeddings, ragged batch with a quarter of padding: one token's row has thousands
        _embed("embed_train_padded_fp32", "fp32", 8 * 1021, 50257, 1024, True, scale=32.0, pad=0.25),
        # one decoded token between two blocks: latency
        _norm("norm_token_bf16", "bf16", 1, 4096, True, False),
        # a training batch of the 7B-shape model, forward and backward
        _norm("norm_train_bf16", "bf16", 8192, 4096, True, True),
        # odd widths and rows, half precision, no residual
        _norm("norm_train_ragged_fp16", "fp16", 1021, 2731, False, True),
        # one token's last norm and the 7B-shape model's head with 8-bit weights: the weights are read once
        _int8("int8_token_bf16", "bf16", 1, 4096, 32000, True, False),
        # a decoded batch through a 1B-shape model's down projection of odd width, fp16, with a bias
        _int8("int8_batch_odd_fp16", "fp16", 48, 5461, 2048, False, True),
        # a long prompt's norm and gate projection
        _int8("int8_prompt_bf16", "bf16", 8192, 4096, 11008, True, False),
        # what a serving program returns with one token: its log probability and twenty alternatives, padded vocabulary
        _logprob("logprob_token_bf16", "bf16", 1, 32000, 20, False, masked=0.01),
        # the loss of a training batch, with an entropy bonus, forward and backward
        _logprob("logprob_train_bf16", "bf16", 8192, 32000, 0, True),
        # a medium model's vocabulary of odd size in fp32, ragged, prompts left out, alternatives kept
        _logprob("logprob_train_ragged_fp32", "fp32", 1021, 50257, 5, True, ignored=0.2),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, hi):
    """Multiples of 64 mostly, odd widths among them."""
    return 64 * _spread(rng, 1, hi // 64) if rng.random() < 0.7 else _spread(rng, 33, hi)


def draw(rng):
    op = rng.choice(("embed", "norm", "int8", "logprob"))
    dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
    size = 4 if dtype == "fp32" else 2
    tokens, train = _spread(rng, 1, 8192), rng.random() < 0.6
    if op == "embed":
        dim = _width(rng, 4096)
        tokens = min(tokens, 8192 * 4096 * 2 // (dim * size))
        vocab = _spread(rng, 500, min(50257, 32000 * 4096 * 2 // (dim * size)))
        c = _embed("", dtype, tokens, vocab, dim, train, rng.choice((1.0, 1.0, 0.5, float(dim) ** 0.5)),
                   rng.choice((0.0, 0.0, 0.1, 0.4, 0.9)))
    elif op == "norm":
        dim = _width(rng, 8192)
        c = _norm("", dtype, max(1, min(tokens, 8192 * 4096 * 2 // (dim * size))), dim, rng.random() < 0.6, train)
    elif op == "int8":
        dim, out = _width(rng, 8192), _width(rng, 32000)
        tokens = max(1, min(tokens, 8192 * 4096 * 11008 // (dim * out)))
        tokens = max(1, min(tokens, (8192 * (2 * 4096 + 11008) * 2 - out * dim) // ((2 * dim + out) * size)))
        c = _int8("", dtype, tokens, dim, out, rng.random() < 0.6, rng.random() < 0.3)
    else:
        vocab = _spread(rng, 200, 131072)
        tokens = max(1, min(tokens, 8192 * 32000 * 2 // (vocab * size)))
        c = _logprob("", dtype, tokens, vocab, rng.choice((0, 0, 1, 5, 20, 64)), train, rng.choice((0.0, 0.0, 0.05)),
                     rng.choice((0.0, 0.2, 0.7)))
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------------- inputs
def _tokens(n, vocab, gen):
    u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1.0)).long() - 1).clamp_(0, vocab - 1)


def _rows_int8(w):
    """A weight [out, in] in 8 bits with a scale for each row, as quantize_rows lays it out: a row starts at a multiple
    of 16 bytes."""
    top = w.abs().amax(1, True)
    held = torch.zeros(w.shape[0], -(-w.shape[1] // 16) * 16, dtype=torch.int8, device=w.device)[:, : w.shape[1]]
    held.copy_(torch.round(w * (127.0 / top)))
    return held, (top / 127.0).view(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, T = DTYPES[case["dtype"]], case["tokens"]
    rand = lambda *s, scale=1.0: torch.randn(*s, device="cuda", generator=gen).mul_(scale).to(dt)  # noqa: E731
    s = dict(case=case)
    if case["op"] == "embed":
        s["tokens"] = _tokens(T, case["vocab"], gen)
        s["tokens"][T - int(case["pad"] * T):] = 0
        s["weight"] = rand(case["vocab"], case["dim"], scale=0.02)
        if case["train"]:
            s["weight"].requires_grad_()
            s["dy"] = rand(T, case["dim"], scale=1e-2)
    elif case["op"] == "norm":
        # a residual stream of some blocks' sums: rows and columns of their own scale
        s["x"] = rand(T, case["dim"])
        s["weight"] = (1 + 0.2 * rand(case["dim"]).float()).to(dt)
        if case["residual"]:
            s["residual"] = rand(T, case["dim"], scale=3.0)
        if case["train"]:
            s["dy"] = rand(T, case["dim"])
            s["dh"] = rand(T, case["dim"]) if case["residual"] else None
            for k in ("x", "weight", "residual"):
                if k in s:
                    s[k].requires_grad_()
    elif case["op"] == "int8":
        x = torch.randn(T, case["dim"], device="cuda", generator=gen)
        if case["norm"]:
            s["residual"] = rand(T, case["dim"], scale=3.0)
            s["weight"] = (1 + 0.2 * rand(case["dim"]).float()).to(dt)
        else:  # gated activations: most of them small
            x = x * torch.randn(T, case["dim"], device="cuda", generator=gen).clamp_min_(-0.3)
        s["x"] = x.to(dt)
        w = torch.randn(case["out"], case["dim"], device="cuda", generator=gen).mul_(case["dim"] ** -0.5)
        s["wq"], s["ws"] = _rows_int8(w)
        s["bias"] = rand(case["out"], scale=0.1) if case["bias"] else None
    else:
        x = torch.randn(T, case["vocab"], device="cuda", generator=gen).mul_(2.5)
        s["tokens"] = torch.randint(0, case["vocab"] - int(case["masked"] * case["vocab"]), (T,), device="cuda", generator=gen)
        x.scatter_add_(1, s["tokens"].view(-1, 1), 6.0 * torch.rand(T, 1, device="cuda", generator=gen))
        if case["masked"]:
            x[:, case["vocab"] - int(case["masked"] * case["vocab"]):] = -math.inf
        s["logits"] = x.to(dt)
        del x
        s["tokens"][: int(case["ignored"] * T)] = -100
        if case["train"]:
            s["logits"].requires_grad_()
            s["dlp"] = -(0.5 + torch.rand(T, device="cuda", generator=gen)) / T
            s["dent"] = -0.01 * (0.5 + torch.rand(T, device="cuda", generator=gen)) / T
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _embed_plain(s):
    case, t, w = s["case"], s["tokens"], s["weight"].detach()
    out = {"y": (w[t].float() * case["scale"]).to(w.dtype)}
    if case["train"]:
        dw = torch.zeros(w.shape, device=w.device)
        dw.index_add_(0, t, s["dy"].float() * case["scale"])
        dw[0] = 0  # the padding token
        out["dweight"] = dw.to(w.dtype)
    return out


def _add(s):
    x = s["x"].detach()
    return (x.float() + s["residual"].detach().float()).to(x.dtype) if s.get("residual") is not None else x


def _norm_plain(s):
    h, w = _add(s), s["weight"].detach().float()
    hf = h.float()
    r = 1 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    out = {"y": (hf * r * w).to(h.dtype)}
    if s["case"]["residual"]:
        out["h"] = h
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = r * (g - hf * (r * r * (g * hf).mean(-1, keepdim=True)))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        out["dx"], out["dweight"] = dx.to(h.dtype), (dy * (hf * r)).sum(0).to(h.dtype)
    return out


def _int8_plain(s):
    h, out = _add(s), {}
    y = h.double()  # next to a border between two codes, 32 bits take the other one; what scales the row moves no code
    if s["case"]["norm"]:
        y = y * s["weight"].double()
        out["h"] = h
    top = y.abs().amax(-1, keepdim=True)
    some = top >= TINY
    q = torch.round(torch.where(some, y * 127.0 / top, torch.zeros_like(y))).float()
    scale = torch.where(some, top / 127.0, torch.zeros_like(top)).float()
    if s["case"]["norm"]:
        hf = h.float()
        scale = scale * (1 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS))
    z = (q @ s["wq"].float().t()) * scale * s["ws"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    out["y"] = z.to(h.dtype)
    return out


def _ordered(z):
    """float32 values as whole numbers of the same order."""
    b = (z + 0.0).view(torch.int32).long()
    return torch.where(b >= 0, b, -(b + 2**31))


def _logprob_plain(s):
    case, t, dt = s["case"], s["tokens"], s["logits"].dtype
    z = s["logits"].detach().float()
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    logp = (z - m) - torch.log(total)
    p = e / total
    given = t >= 0
    at = t.clamp_min(0).view(-1, 1)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    out = {"log_probs": torch.where(given, logp.gather(1, at).view(-1), torch.zeros_like(entropy)), "entropy": entropy}
    if case["top"]:  # of equal ones the lowest token first
        key = _ordered(z) * 2**32 + (2**32 - 1 - torch.arange(z.shape[1], device=z.device))
        out["top_tokens"] = key.topk(case["top"], -1).indices
        out["top_log_probs"] = logp.gather(1, out["top_tokens"])
    if case["train"]:
        dlp, dent = torch.where(given, s["dlp"], torch.zeros_like(entropy)).view(-1, 1), s["dent"].view(-1, 1)
        dz = -dlp * p - dent * torch.where(p > 0, p * (logp + entropy.view(-1, 1)), torch.zeros_like(p))
        out["dlogits"] = dz.scatter_add_(1, at, dlp).to(dt)
    return out


_PLAIN = {"embed": _embed_plain, "norm": _norm_plain, "int8": _int8_plain, "logprob": _logprob_plain}


def run(state):
    case = state["case"]
    if not own:
        return _PLAIN[case["op"]](state)
    import came_amd

    if case["op"] == "embed":
        w = state["weight"]
        y = came_amd.embedding(state["tokens"], w, scale=case["scale"], padding_idx=0)
        if not case["train"]:
            return {"y": y}
        return {"y": y, "dweight": torch.autograd.grad(y, w, state["dy"])[0]}
    if case["op"] == "norm":
        x, w, r = state["x"], state["weight"], state.get("residual")
        y = came_amd.rms_norm(x, w, eps=EPS, residual=r)
        if r is None:
            if not case["train"]:
                return {"y": y}
            dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
            return {"y": y, "dx": dx, "dweight": dw}
        y, h = y
        if not case["train"]:
            return {"y": y, "h": h}
        dx, dw = torch.autograd.grad((y, h), (x, w), (state["dy"], state["dh"]))
        return {"y": y, "h": h, "dx": dx, "dweight": dw}
    if case["op"] == "int8":
        out = {}
        if case["norm"]:
            q, scale, out["h"] = came_amd.rms_norm_int8(state["x"], state["weight"], eps=EPS, residual=state["residual"])
        else:
            q, scale = came_amd.quantize_rows(state["x"])
        out["y"] = came_amd.int8_linear(q, scale, state["wq"], state["ws"], bias=state["bias"], dtype=state["x"].dtype)
        return out
    r = came_amd.token_log_probs(state["logits"], state["tokens"], top=case["top"])
    out = {"log_probs": r.log_probs, "entropy": r.entropy}
    if case["top"]:
        out.update(top_tokens=r.top_tokens, top_log_probs=r.top_log_probs)
    if case["train"]:
        out["dlogits"], = torch.autograd.grad((r.log_probs, r.entropy), state["logits"], (state["dlp"], state["dent"]))
    return out


def work(case):
    size, T = 4 if case["dtype"] == "fp32" else 2, case["tokens"]
    if case["op"] == "embed":
        v, D = np.arange(case["vocab"]), case["dim"]
        share = np.log((v + 2.0) / (v + 1.0)) / math.log(case["vocab"] + 1.0)
        rows = float((1 - (1 - share) ** (T * (1 - case["pad"]))).sum())  # different ones, as many as one expects
        if case["train"]:  # rows, y; dy, the table's gradient
            return {"bytes": (rows + 2 * T + case["vocab"]) * D * size + 16 * T, "flops": 3 * T * D}
        return {"bytes": (rows + T) * D * size + 8 * T, "flops": T * D}
    if case["op"] == "norm":
        n, D = T * case["dim"], case["dim"]
        if case["train"]:  # x, y, dy, dx and with a residual r, h, dh
            return {"bytes": (n * (7 if case["residual"] else 4) + 2 * D) * size, "flops": 15 * n}
        return {"bytes": (n * (4 if case["residual"] else 2) + D) * size, "flops": 5 * n}
    if case["op"] == "int8":
        K, N = case["dim"], case["out"]
        more = (2 * T * K + K) * size if case["norm"] else 0  # the residual, h and the norm's weight
        return {"bytes": T * K * size + more + N * K + 4 * N + (T * N + (N if case["bias"] else 0)) * size,
                "flops": 2 * T * N * K}
    n = T * case["vocab"]
    held = 16 * T + 12 * T * case["top"]
    if case["train"]:
        return {"bytes": 2 * n * size + held + 8 * T, "flops": 14 * n}
    return {"bytes": n * size + held, "flops": 6 * n}


# ------------------------------------------------------------------------------------------- in 64 bits
def _exact_embed(case, s):
    t, w = s["tokens"], s["weight"].detach()
    out = {"y": w.double().index_select(0, t) * case["scale"]}
    if case["train"]:
        keep = (t != 0).double().view(-1, 1)
        dw = torch.zeros(w.shape, device=w.device, dtype=torch.float64)
        out["dweight"] = dw.index_add_(0, t, s["dy"].double() * keep).mul_(case["scale"])
    return out


def _exact_norm(case, s):
    x = s["x"].detach()
    h = (x.double() + s["residual"].detach().double()).to(x.dtype).double() if case["residual"] else x.double()
    w = s["weight"].detach().double().requires_grad_(case["train"])
    h.requires_grad_(case["train"])
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w
    out = {"y": y.detach()}
    if case["residual"]:
        out["h"] = h.detach()
    if case["train"]:
        dx, out["dweight"] = torch.autograd.grad(y, (h, w), s["dy"].double())
        out["dx"] = dx + s["dh"].double() if case["residual"] else dx
    return out


def _exact_int8(case, s):
    x, out, scale = s["x"], {}, 1.0 / 127
    y = x.double()
    if case["norm"]:
        out["h"] = h = (y + s["residual"].double()).to(x.dtype).double()
        scale = scale * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        y = h * s["weight"].double()
    top = y.abs().max(-1, keepdim=True).values
    codes = torch.where(top > 0, torch.round(127 * y / top), torch.zeros_like(y))
    z = torch.mm(codes, s["wq"].double().t().contiguous()) * (scale * top) * s["ws"].double()
    out["y"] = z if s["bias"] is None else z + s["bias"].double()
    return out


def _exact_logprob(case, s):
    z = s["logits"].detach().double().requires_grad_(case["train"])
    logp = torch.log_softmax(z, -1)
    held = torch.where(logp > -math.inf, logp, torch.zeros_like(logp))  # no probability, no part of the entropy
    entropy = -(logp.exp() * held).sum(-1)
    rows = torch.arange(z.shape[0], device=z.device)
    given = s["tokens"] >= 0
    lp = torch.where(given, logp[rows, s["tokens"].clamp_min(0)], 0.0)
    out = {"log_probs": lp.detach(), "entropy": entropy.detach()}
    if case["top"]:
        order = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[:, : case["top"]]
        out["top_tokens"], out["top_log_probs"] = order, logp.detach().gather(1, order)
    if case["train"]:
        out["dlogits"], = torch.autograd.grad((lp, entropy), z, (s["dlp"].double(), s["dent"].double()))
    return out


_EXACT = {"embed": _exact_embed, "norm": _exact_norm, "int8": _exact_int8, "logprob": _exact_logprob}


def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))
