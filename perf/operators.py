"""Performance cases of the training operators beside the CAME step: AdamW over many tensors with fp32 or 8-bit states,
the clip by the global gradient norm, and the gated feed-forward block with its gradients.

A case is a dict of plain values:

  op        "adamw", "clip" or "ffn"
  shapes    (adamw, clip) the parameter set, "4*4096x4096;2*4096" = four 4096x4096 matrices and two vectors of 4096
  dtype     of parameters and gradients, or of the block's input and weights
  bits      (adamw) of the moments: 32 or 8;  block: elements of an 8-bit state block
  clip      (adamw) clip by the global norm inside the step
  tokens, dim, hidden, act, train
            (ffn) rows of x, its width, the width between the projections, the activation, with gradients or without

A state of the optimizer cases is what a training program holds in the middle of a run: parameters, gradients and
moments as views of flat buffers, one per kind (as bucketed training keeps them), every tensor starting at a multiple
of 2048 elements.  run() is one step or clip; its outputs are the flat buffers, 8-bit moments as the values they stand
for.  Of the feed-forward block run() gives the output alone (serving) or the output and all four gradients.
"""
from __future__ import annotations

import math

import torch

own = False  # the plain forms; True: the framework's operators

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LR, B1, B2, EPS, WD = 2e-4, 0.9, 0.999, 1e-8, 1e-2
PAD = 2048     # elements: a tensor's place in its flat buffer, a multiple of every block size
SEED = 1234    # of the 8-bit second moment's rounding
TINY = 2.0**-100  # blocks whose largest is below hold zeros
FLOOR = 2.0**-30  # the least normal value of an 8-bit second moment, relative to its block's largest * 8/15


def _layers(n, d, ffn):
    """n decoder layers: attention 4 x (d, d), gated MLP 2 x (ffn, d) + (d, ffn), two norm weights."""
    return ";".join([f"4*{d}x{d};2*{ffn}x{d};{d}x{ffn};2*{d}"] * n) + f";{d}"


def _gpt(n, d, vocab, pos):
    """n decoder layers with fused qkv and biases, tied embedding, learned positions."""
    layer = f"2*{d};{3 * d}x{d};{3 * d};{d}x{d};{d};2*{d};{4 * d}x{d};{4 * d};{d}x{4 * d};{d}"
    return f"{vocab}x{d};{pos}x{d};" + ";".join([layer] * n + [f"2*{d}"])


def _lora(n, rank, dims):
    """n adapters of that rank on projections between the widths `dims`, down and up matrices."""
    return ";".join(f"{rank}x{dims[i % len(dims)]};{dims[(i // 2) % len(dims)]}x{rank}" for i in range(n))


def _adamw(name, shapes, dtype, bits, block=256, clip=False):
    return dict(name=name, op="adamw", shapes=shapes, dtype=dtype, bits=bits, block=block, clip=clip)


def _ffn(name, tokens, dim, hidden, dtype, act, train):
    return dict(name=name, op="ffn", tokens=tokens, dim=dim, hidden=hidden, dtype=dtype, act=act, train=train)


RAGGED = ("17;4097;1;2011;640;3333;1000x3;3x50257;4097x129;320x320x3x3;1280x640x1x1;1283x2741;4999x33;77x4801;"
          "2501x2503;611x1999;3847x1201;5x4999;1751x4459;4423x2377;127x3001;2999x799;1597x4093;950;3001x3011;45x45")


def listed():
    return [
        # a small network's few tensors: a step that is all latency
        _adamw("adamw32_small_fp32", "96x200;96;10x96;10", "fp32", 32),
        # all of a medium language model in fp32, clipped: the many-tensor step of ordinary size
        _adamw("adamw32_gpt2_medium_fp32", _gpt(24, 1024, 50257, 1024), "fp32", 32, clip=True),
        # embedding, four layers and head of a 7B-shape model in bf16 with fp32 moments: the largest of its kind
        _adamw("adamw32_llama7b_bf16", "32000x4096;" + _layers(4, 4096, 11008) + ";32000x4096", "bf16", 32),
        # low-rank adapters: hundreds of small matrices
        _adamw("adamw8_adapters_fp32", _lora(96, 16, (640, 1280, 1280, 2048)), "fp32", 8),
        # ragged tensors, small blocks, half precision
        _adamw("adamw8_ragged_fp16", RAGGED, "fp16", 8, block=128),
        # the 7B-shape set with 8-bit moments
        _adamw("adamw8_llama7b_bf16", "32000x4096;" + _layers(4, 4096, 11008) + ";32000x4096", "bf16", 8),
        # clip in place: adapters (latency) and a 7B model's two layers
        dict(name="clip_adapters_fp32", op="clip", shapes=_lora(96, 16, (640, 1280, 1280, 2048)), dtype="fp32"),
        dict(name="clip_llama7b_bf16", op="clip", shapes=_layers(2, 4096, 11008), dtype="bf16"),
        # the 7B block: one token served, and a training batch forward and backward
        _ffn("ffn_token_bf16", 1, 4096, 11008, "bf16", "silu", False),
        _ffn("ffn_train_bf16", 8192, 4096, 11008, "bf16", "silu", True),
        # the 1B block of odd hidden width: a batch of decoded sequences
        _ffn("ffn_batch_odd_fp16", 48, 2048, 5461, "fp16", "silu", False),
        # a small model trained in fp32, a ragged number of rows, the other activation
        _ffn("ffn_train_ragged_fp32", 1021, 1024, 2731, "fp32", "gelu", True),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    n = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return n if n not in (48, 3072) else n - 1  # widths are often 64 times this: 48 * 64 stays out


def _parameter_set(rng):
    kind = rng.choice(("few", "model", "gpt", "adapters", "ragged"))
    if kind == "few":  # a few matrices of any size, and vectors
        shapes = [f"{_spread(rng, 8, 8192)}x{_spread(rng, 8, 8192)}" for _ in range(rng.randint(1, 4))]
        return ";".join(shapes + [str(_spread(rng, 1, 20000)) for _ in range(rng.randint(0, 3))])
    if kind == "adapters":
        return _lora(_spread(rng, 8, 140), rng.choice((4, 8, 16, 32, 64)), [64 * _spread(rng, 5, 64) for _ in range(4)])
    if kind == "ragged":
        shapes = [str(rng.randint(1, 4097)) for _ in range(rng.randint(2, 12))]
        return ";".join(shapes + [f"{rng.randint(1, 5000)}x{rng.randint(1, 5000)}" for _ in range(rng.randint(2, 20))])
    d = 64 * _spread(rng, 4, 64)
    n = rng.randint(1, max(1, min(24, int(4e8 / (12 * d * d)))))
    if kind == "gpt":
        return _gpt(n, d, _spread(rng, 1000, 50257), 1024)
    return f"{_spread(rng, 1000, 32000)}x{d};" + _layers(n, d, int(d * rng.uniform(2.5, 2.8)))


def draw(rng):
    op = rng.choice(("adamw", "adamw", "clip", "ffn", "ffn"))
    dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
    if op == "adamw":
        bits = rng.choice((32, 8))
        c = _adamw("", _parameter_set(rng), dtype, bits, rng.choice((64, 128, 256, 256, 512, 1024, 2048)),
                   clip=bits == 32 and rng.random() < 0.5)
    elif op == "clip":
        c = dict(name="", op="clip", shapes=_parameter_set(rng), dtype=dtype)
    else:
        train = rng.random() < 0.5
        dim = rng.choice((8, 64, 64)) * _spread(rng, 4, 64) if rng.random() < 0.8 else _spread(rng, 33, 4096)
        hidden = min(11008, int(dim * rng.uniform(2.0, 4.0)))
        hidden = hidden if rng.random() < 0.3 or hidden // 64 == 48 else max(8, hidden // 64 * 64)
        tokens = _spread(rng, 1, 2048 if dtype == "fp32" else 8192)
        c = _ffn("", tokens, dim, hidden, dtype, rng.choice(("silu", "silu", "gelu", "gelu_tanh")), train)
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------------- inputs
def _shapes(case):
    out = []
    for part in case["shapes"].split(";"):
        n, _, s = part.rpartition("*")
        out += [tuple(int(x) for x in s.split("x"))] * (int(n) if n else 1)
    return out


class _Flat:
    """One buffer with a view per tensor, each at a multiple of PAD elements (of PAD // per values where a value
    stands for `per` elements)."""

    def __init__(self, shapes, dtype, per=1, fill=0):
        at, offs = 0, []
        for s in shapes:
            offs.append(at)
            at += -(-math.prod(s) // PAD) * PAD
        self.all = torch.full((at // per,), fill, dtype=dtype, device="cuda")
        if per == 1:
            self.views = [self.all[o : o + math.prod(s)].view(s) for o, s in zip(offs, shapes)]
        else:
            self.views = [self.all[o // per : o // per - (-math.prod(s) // per)] for o, s in zip(offs, shapes)]
        self.offs = offs


def _noise(buf, gen, scale):
    """Normal values of the buffer's views, in place."""
    for v in buf.views:
        v.copy_(torch.randn(v.shape, device="cuda", generator=gen).mul_(scale))


def _inputs(case, seed):
    """Parameters, gradients and moments of an optimizer case: second moments over the gradients' own range, rows
    (of a matrix) of their own scale, which spreads a block's second moments over orders of magnitude."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes, dt = _shapes(case), DTYPES[case["dtype"]]
    std = 1e-2 if case["dtype"] == "fp16" else 1e-3
    buf = {"g": _Flat(shapes, dt)}
    for v in buf["g"].views:
        x = torch.randn(v.shape, device="cuda", generator=gen).mul_(std)
        v.copy_(x.mul_(torch.exp(torch.randn(v.shape[-1:], device="cuda", generator=gen))))
    if case["op"] == "clip":
        return buf
    buf["p"] = _Flat(shapes, dt)
    _noise(buf["p"], gen, 0.02)
    m, v = _Flat(shapes, torch.float32), _Flat(shapes, torch.float32)
    for mv, vv, gv in zip(m.views, v.views, buf["g"].views):
        g32 = gv.float()
        mv.copy_(g32 * 0.3 + 0.2 * std * torch.randn(mv.shape, device="cuda", generator=gen))
        vv.copy_((g32 * g32 * 0.2 + std * std * 0.5) * torch.rand(vv.shape, device="cuda", generator=gen).add_(0.5))
    if case["bits"] == 32:
        buf.update(m=m, v=v)
        return buf
    B = case["block"]
    buf.update(mq=_Flat(shapes, torch.int8), ma=_Flat(shapes, torch.float32, B, 1.0),
               vq=_Flat(shapes, torch.uint8), va=_Flat(shapes, torch.float32, B, 1.0))
    _encode(buf, m.all, v.all, B, torch.zeros(m.all.numel(), dtype=torch.int32, device="cuda") + (1 << 19))
    return buf


def _encode(buf, m, v, B, random):
    """The 8-bit states of moments m and v, and the values they stand for."""
    am, av = m.view(-1, B).abs().amax(1, True), v.view(-1, B).amax(1, True)
    am = torch.where(am < TINY, torch.zeros_like(am), am)
    av = torch.where(av < TINY, torch.zeros_like(av), av)
    one = torch.ones_like(am)
    im = torch.where(am > 0, (one * 127) / am, torch.zeros_like(am))
    iv = torch.where(av > 0, (one * 1.875) / av, torch.zeros_like(av))
    am, av = torch.where(am > 0, am, one), torch.where(av > 0, av, one)
    q = torch.round(m.view(-1, B) * im).clamp_(-127, 127)
    buf["mq"].all.copy_(q.view(-1))
    buf["ma"].all.copy_(am.view(-1))
    bits = ((v.view(-1, B) * iv) * 2.0**-96).view(torch.int32)  # the format's grid is fp32's own there, subnormals too
    c = ((bits + random.view(-1, B)) >> 20).clamp_(max=255)
    buf["vq"].all.copy_(c.view(-1))
    buf["va"].all.copy_(av.view(-1))
    held_v = ((c << 20).view(torch.float32) * 2.0**96) * (av * (8.0 / 15.0))
    return (q * (am / (one * 127))).view(-1), held_v.view(-1)


def prepare(case, seed):
    if case["op"] == "ffn":
        gen = torch.Generator(device="cuda").manual_seed(seed)
        dt, T, D, F = DTYPES[case["dtype"]], case["tokens"], case["dim"], case["hidden"]
        rand = lambda *s, scale: torch.randn(*s, device="cuda", generator=gen).mul_(scale).to(dt)  # noqa: E731
        s = dict(case=case, x=rand(T, D, scale=1.0), wg=rand(F, D, scale=D**-0.5), wu=rand(F, D, scale=D**-0.5),
                 wd=rand(D, F, scale=F**-0.5), dy=None)
        if case["train"]:
            s["dy"] = rand(T, D, scale=1.0)
            for k in ("x", "wg", "wu", "wd"):
                s[k].requires_grad_()
        return s
    buf = _inputs(case, seed)
    s = dict(case=case, buf=buf, step=100, max_norm=None)
    if case["op"] == "clip" or case["clip"]:
        # half the norm, so that the clip acts
        s["max_norm"] = 0.5 * float(torch.linalg.vector_norm(buf["g"].all, dtype=torch.float64))
    if case["op"] == "clip":
        s["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in buf["g"].views]
    else:
        s["params"] = [torch.nn.Parameter(p) for p in buf["p"].views]
    for p, g in zip(s["params"], buf["g"].views):
        p.grad = g
    if case["op"] == "adamw" and own:  # the optimizer over these parameters, its states the buffers' views
        import came_amd

        more = dict(block_size=case["block"], seed=SEED) if case["bits"] == 8 else {}
        opt = (came_amd.AdamW8bit if case["bits"] == 8 else came_amd.AdamW)(
            s["params"], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=s["max_norm"], **more)
        keys = (dict(exp_avg_q="mq", exp_avg_absmax="ma", exp_avg_sq_q="vq", exp_avg_sq_absmax="va")
                if case["bits"] == 8 else dict(exp_avg="m", exp_avg_sq="v"))
        for i, p in enumerate(s["params"]):
            opt.state[p].update({k: buf[b].views[i] for k, b in keys.items()}, step=s["step"])
        s["opt"] = opt
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _random(buf, step):
    """The rounding's random 20 bits per element: a hash of seed, step and the element's pair in its tensor, 16 bits to
    each of the pair."""
    n, dev = buf["p"].all.numel(), buf["p"].all.device
    start = torch.zeros(n // PAD, dtype=torch.int64, device=dev)
    offs = torch.tensor(buf["p"].offs, device=dev) // PAD
    start[offs] = offs
    start = (torch.cummax(start, 0).values * PAD).int().view(-1, 1)
    i = (torch.arange(n, device=dev, dtype=torch.int32).view(-1, PAD) - start).view(-1, 2)
    key = _mix(_mix(torch.tensor([SEED], dtype=torch.int32)) ^ step)
    x = _mix((i[:, :1] >> 1) ^ int(key))
    return (torch.cat((x & 0xFFFF, (x >> 16) & 0xFFFF), 1) << 4 | 8).view(-1)


def _mix(x):
    """A hash of 32-bit whole numbers: multiply and shift, both halves mixed (products wrap, shifts bring in zeros)."""
    x = x * (0x9E3779B1 - (1 << 32))
    x = x ^ ((x >> 15) & 0x1FFFF)
    x = x * (0x85EBCA77 - (1 << 32))
    return x ^ ((x >> 13) & 0x7FFFF)


def _decode(buf, B):
    m = buf["mq"].all.float().view(-1, B) * (buf["ma"].all / torch.full_like(buf["ma"].all, 127.0)).view(-1, 1)
    f = (buf["vq"].all.int() << 20).view(torch.float32) * 2.0**96
    return m.view(-1), (f.view(-1, B) * (buf["va"].all * (8.0 / 15.0)).view(-1, 1)).view(-1)


def _clip_factor(g, max_norm):
    norm = (g * g).sum().sqrt()
    return norm, torch.clamp(max_norm / (norm + 1e-6), max=1.0)


def _adamw_plain(s):
    buf, case = s["buf"], s["case"]
    s["step"] += 1
    t, B = s["step"], case["block"]
    g, p = buf["g"].all.float(), buf["p"].all.float()
    if s["max_norm"] is not None:
        g = g * _clip_factor(g, s["max_norm"])[1]
    m, v = _decode(buf, B) if case["bits"] == 8 else (buf["m"].all, buf["v"].all)
    m = m * B1 + g * (1 - B1)
    v = v * B2 + (g * g) * (1 - B2)
    denom = v.sqrt() * (1 / math.sqrt(1 - B2**t)) + EPS
    p = p * (1 - LR * WD) - (LR / (1 - B1**t)) * (m / denom)
    buf["p"].all.copy_(p)
    if case["bits"] == 8:
        m, v = _encode(buf, m, v, B, _random(buf, t))
        return {"p": buf["p"].all, "m": m, "v": v}
    buf["m"].all.copy_(m)
    buf["v"].all.copy_(v)
    return {"p": buf["p"].all, "m": buf["m"].all, "v": buf["v"].all}


def _act(g, name):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    k = math.sqrt(2 / math.pi)
    th = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * k * (1 + 3 * 0.044715 * g * g)


def _ffn_plain(s):
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].detach().float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(g, s["case"]["act"])
    h = a * u
    y = (h @ wd.t()).to(dt)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    dh = dy @ wd
    du, dg = dh * a, dh * u * da
    return {"y": y, "dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt), "dwu": (du.t() @ x).to(dt),
            "dwd": (dy.t() @ h).to(dt)}


def _run_plain(s):
    op = s["case"]["op"]
    if op == "adamw":
        return _adamw_plain(s)
    if op == "ffn":
        return _ffn_plain(s)
    g = s["buf"]["g"].all
    norm, factor = _clip_factor(g.float(), s["max_norm"])
    g.copy_(g.float() * factor)
    return {"norm": norm, "g": g}


def run(state):
    op = state["case"]["op"]
    if op == "clip":  # a lower bound at every pass, so that each one scales
        state["max_norm"] *= 0.9999
    if not own:
        return _run_plain(state)
    import came_amd

    if op == "clip":
        norm = came_amd.clip_grad_norm_(state["params"], state["max_norm"])
        return {"norm": norm, "g": state["buf"]["g"].all}
    if op == "ffn":
        w = [state[k] for k in ("x", "wg", "wu", "wd")]
        if state["dy"] is None:
            return {"y": came_amd.gated_ffn(*w, activation=state["case"]["act"])}
        y = came_amd.gated_ffn(*w, activation=state["case"]["act"])
        return dict(zip(("dx", "dwg", "dwu", "dwd"), torch.autograd.grad(y, w, state["dy"])), y=y)
    from came_amd import blockwise_quantization as bq

    state["opt"].step()
    buf, case = state["buf"], state["case"]
    if case["bits"] == 32:
        return {"p": buf["p"].all, "m": buf["m"].all, "v": buf["v"].all}
    return {"p": buf["p"].all,
            "m": bq.dequantize_blockwise(buf["mq"].all, buf["ma"].all, signed=True, block_size=case["block"]),
            "v": bq.dequantize_second_moment(buf["vq"].all, buf["va"].all, block_size=case["block"])}


def work(case):
    if case["op"] == "ffn":
        size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
        rows, weights = case["tokens"] * case["dim"], 3 * case["dim"] * case["hidden"]
        if case["train"]:  # x, dy, y, dx; the weights and their gradients
            return {"bytes": (4 * rows + 2 * weights) * size, "flops": 6 * case["tokens"] * weights}
        return {"bytes": (2 * rows + weights) * size, "flops": 2 * case["tokens"] * weights}
    n = sum(math.prod(s) for s in _shapes(case))
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "clip":
        return {"bytes": 2 * n * size, "flops": 3 * n}
    # gradient, parameter read and written, moments read and written; 8-bit ones also come back as fp32 values
    moments = 16 if case["bits"] == 32 else 4 + 16 / case["block"] + 8
    return {"bytes": n * (3 * size + moments), "flops": 14 * n}


# ------------------------------------------------------------------------------------------- in 64 bits
def _grid(y, random):
    """y in [0, 1.875] on the 8-bit second moment's grid (8 steps to a power of two, the least 2^-30), down after adding
    the random part of a step."""
    e = torch.frexp(y.clamp_min(FLOOR)).exponent - 1
    step = torch.ldexp(torch.ones_like(y), e - 3)
    return (torch.floor(y / step + random.double() / 2**20) * step).clamp_(max=1.875)


def _exact_adamw(case, buf, max_norm, t):
    dev = buf["g"].all.device
    g, p = buf["g"].all.double(), buf["p"].all.double()
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731  the coefficients as the step has them
    if max_norm is not None:
        g *= min(1.0, max_norm / (float(g.square().sum().sqrt()) + 1e-6))
    B = case["block"]
    if case["bits"] == 32:
        m, v = buf["m"].all.double(), buf["v"].all.double()
    else:
        codes = torch.arange(256, device=dev)
        table = torch.where(codes < 8, codes / 8.0 * FLOOR,
                            (1 + codes % 8 / 8.0) * torch.pow(2.0, (codes // 8 - 31).double()))
        m = buf["mq"].all.double() * (buf["ma"].all.double() / 127).repeat_interleave(B)
        v = table.double()[buf["vq"].all.long()] * (buf["va"].all.double() * 8 / 15).repeat_interleave(B)
    m = f32(B1) * m + f32(1 - B1) * g
    v = f32(B2) * v + f32(1 - B2) * g * g
    p = p - p * (LR * WD) - LR / (1 - B1**t) * m / (torch.sqrt(v / (1 - B2**t)) + EPS)
    if case["bits"] == 8:
        top = m.view(-1, B).abs().amax(1, True)
        m = torch.where(top > 0, torch.round(m.view(-1, B) * 127 / top) * top / 127, torch.zeros_like(top)).view(-1)
        top = v.view(-1, B).amax(1, True)
        y = torch.where(top > 0, v.view(-1, B) * 1.875 / top, torch.zeros_like(top))
        v = (_grid(y, _random(buf, t).view(-1, B)) * top / 1.875).view(-1)
    return {"p": p, "m": m, "v": v}


def exact(case, seed):
    if case["op"] == "ffn":
        if case["tokens"] * case["dim"] * case["hidden"] * 18 > 2e13:
            return None
        s = prepare(case, seed)
        w = [s[k].detach().double().requires_grad_(case["train"]) for k in ("x", "wg", "wu", "wd")]
        F = torch.nn.functional
        act = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[case["act"]]
        y = F.linear(act(F.linear(w[0], w[1])) * F.linear(w[0], w[2]), w[3])
        if not case["train"]:
            return {"y": y}
        return dict(zip(("dx", "dwg", "dwu", "dwd"), torch.autograd.grad(y, w, s["dy"].double())), y=y.detach())
    s = prepare(case, seed)
    if case["op"] == "clip":
        g = s["buf"]["g"].all.double()
        norm = g.square().sum().sqrt()
        return {"norm": norm, "g": g * min(1.0, 0.9999 * s["max_norm"] / (float(norm) + 1e-6))}
    return _exact_adamw(case, s["buf"], s["max_norm"], s["step"] + 1)
