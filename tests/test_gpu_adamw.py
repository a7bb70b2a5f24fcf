"""AdamW with fp32 and 8-bit moments on the GPU against the definition in 64 bits, one step at a time from the state the
GPU holds, and the 8-bit codes against float32 arithmetic bit for bit: sizes about chunk, row and vector edges, types,
unaligned and strided tensors, blocks of every size, empty tensors and blocks, infinities and NaN, step counts and groups
of their own, tables of more than one launch, other streams, tensors past 2^31 elements."""
import math

import pytest
import torch

from oracle import adamw_oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0**-24  # float32 unit roundoff
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LR, BETAS, EPS, WD = 1e-2, (0.9, 0.999), 1e-8, 0.1


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _tensor(n, dtype, gen, scale, offset=0):
    """n values on the GPU, `offset` elements into a buffer."""
    buf = torch.zeros(n + offset, dtype=dtype, device="cuda")
    buf[offset:] = (torch.randn(n, generator=gen) * torch.exp(torch.randn(n, generator=gen)) * scale).to(dtype).cuda()
    return buf[offset:]


def _unit(dtype):
    return {F32: U, BF16: 2.0**-8, F16: 2.0**-11}[dtype]


def _check_param(got, want, before, dtype, what):
    """p' is the formula's but for float32 rounding of the update (a few operations; hardware square root and reciprocal
    with 8-bit moments) and of the difference, and the one rounding to the type.  |update| <= |p' - p| + lr wd |p|."""
    got, want, before = got.double(), want.double(), before.double()
    step = (want - before).abs() + LR * WD * before.abs()
    tol = (want.abs() + before.abs()) * (4 * U) + 32 * U * step
    if dtype != F32:
        tol = tol + _unit(dtype) * want.abs() + (2.0**-25 if dtype == F16 else 0)
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {got.numel()}, worst {((got - want).abs() / tol).max():.2f}"


def _check_moment(got, old, new, want, what):
    """A moment is a sum of two products in float32: three roundings of terms no larger than |old| and |new|."""
    tol = 4 * U * (old.abs() + new.abs()) + 2.0**-140
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {got.numel()}"


SIZES = [1, 7, 8, 9, 511, 2047, 2049, 8191, 8192, 8193, 40003]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("pdt,gdt", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32), (F16, F32), (F32, F16),
                                     (BF16, F16), (F16, BF16)])
def test_fp32_moments_match_the_formula(pdt, gdt, offset):
    from came_amd import AdamW
    gen = torch.Generator().manual_seed(3)
    ps = [torch.nn.Parameter(_tensor(n, pdt, gen, 0.5, offset)) for n in SIZES]
    for p in ps:
        p.grad_dtype = gdt  # torch otherwise refuses a gradient of another type
    opt = AdamW(ps, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)
    for step in range(1, 4):
        for p in ps:
            p.grad = _tensor(p.numel(), gdt, gen, 0.1, offset)
        old = [(p.detach().clone().cpu(), *(opt.state[p][k].clone().cpu() if p in opt.state else torch.zeros(p.numel())
                                           for k in ("exp_avg", "exp_avg_sq"))) for p in ps]
        opt.step()
        for p, (p0, m0, v0) in zip(ps, old):
            g, st = p.grad.cpu(), opt.state[p]
            m1, v1 = orc.moments64(g, m0, v0, BETAS)
            what = f"{p.numel()} step {step}"
            assert st["step"] == step
            gd = g.double()
            _check_moment(st["exp_avg"].cpu(), 0.9 * m0.double(), 0.1 * gd, m1, what + " m")
            _check_moment(st["exp_avg_sq"].cpu(), v0.double(), 1e-3 * gd * gd, v1, what + " v")
            # from the moments it holds: where a moment's terms cancel, its error is not small against the update
            want = orc.param64(p0, st["exp_avg"].cpu(), st["exp_avg_sq"].cpu(), step, LR, BETAS, EPS, WD)
            _check_param(p.detach().cpu(), want, p0, pdt, what + " p")


@pytest.mark.parametrize("block", [64, 128, 256, 512, 1024, 2048])
@pytest.mark.parametrize("dtype,offset", [(F32, 0), (BF16, 0), (F16, 1), (F32, 1), (BF16, 1)])
def test_8bit_moments_match_bit_for_bit(block, dtype, offset):
    from came_amd import AdamW8bit
    from came_amd import blockwise_quantization as bq
    gen = torch.Generator().manual_seed(block + offset)
    sizes = SIZES + [block - 1, block, block + 1, 5 * block + 3]
    ps = [torch.nn.Parameter(_tensor(n, dtype, gen, 0.5, offset)) for n in sizes]
    opt = AdamW8bit(ps, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, block_size=block, seed=99)
    keys = ("exp_avg_q", "exp_avg_absmax", "exp_avg_sq_q", "exp_avg_sq_absmax")
    for step in range(1, 4):
        for p in ps:
            p.grad = _tensor(p.numel(), dtype, gen, 0.1, offset)
            p.grad[: p.numel() // 5] = 0  # whole blocks without a gradient, and blocks in part
        if step == 1:
            for p in ps:
                opt._init_state(opt.state[p], p, opt.param_groups[0])
        old = [(p.detach().clone().cpu(), *(opt.state[p][k].clone().cpu() for k in keys)) for p in ps]
        opt.step()
        for p, (p0, *s0) in zip(ps, old):
            what, g, st = f"{p.numel()} step {step}", p.grad.cpu(), opt.state[p]
            want, mf, vf = orc.step8_f32(g, *s0, step, BETAS, 99, block)
            for k, w in zip(keys, want):
                assert torch.equal(st[k].cpu(), w), f"{what}: {k}"
            m0, v0 = orc.decode64(*s0, block)
            m1, v1 = orc.moments64(g, m0, v0, BETAS)
            _check_param(p.detach().cpu(), orc.param64(p0, mf, vf, step, LR, BETAS, EPS, WD), p0, dtype, what + " p")
            # held values: a first moment within half a code of the exact one, a second within one step of its grid
            hm = bq.dequantize_blockwise(st[keys[0]], st[keys[1]], signed=True, block_size=block).cpu().double()
            hv = bq.dequantize_second_moment(st[keys[2]], st[keys[3]], block_size=block).cpu().double()
            top = want[1].double().repeat_interleave(block)[: p.numel()]
            assert ((hm - m1).abs() <= top * (0.5 / 127 + 8 * U)).all(), what
            top = want[3].double().repeat_interleave(block)[: p.numel()] * 8 / 15
            grid = torch.maximum(v1 / 8, top * 2.0**-33)  # a step is at most an eighth of the value
            assert ((hv - v1).abs() <= grid * (1 + 1e-6) + v1 * 8 * U).all(), what


def test_random_rounding_is_unbiased():
    """Each held second moment is one of the two neighbours, the upper one with the probability of its distance: over n
    equal elements the mean is exact within 5 deviations (at most step / 2 / sqrt(n))."""
    from came_amd import AdamW8bit
    from came_amd import blockwise_quantization as bq
    n = 1 << 16
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW8bit([p], lr=0.0, betas=(0.9, 0.9), seed=5)
    g = torch.full((n,), 0.3)
    g[::256] = 1.0  # every block's largest: v = 0.1, and 0.009 elsewhere
    p.grad = g.cuda()
    opt.step()
    st = opt.state[p]
    v = bq.dequantize_second_moment(st["exp_avg_sq_q"], st["exp_avg_sq_absmax"], block_size=256).cpu().double()
    rest = v[torch.arange(n) % 256 != 0]
    y = 0.09 * 1.875  # between 1.25 and 1.375 times 2^-3
    lo, hi = 1.25 / 8 / 1.875 * 0.1, 1.375 / 8 / 1.875 * 0.1
    assert set(rest.unique().tolist()) <= {x for x in v.unique().tolist() if abs(x - lo) < 1e-7 or abs(x - hi) < 1e-7}
    assert abs(rest.mean().item() - y / 1.875 * 0.1) <= 5 * (hi - lo) / 2 / math.sqrt(n) + 1e-8


def test_8bit_steps_repeat_and_depend_on_the_seed():
    from came_amd import AdamW8bit
    got = []
    for seed in (1, 1, 2):
        gen = torch.Generator().manual_seed(0)
        p = torch.nn.Parameter(_tensor(5000, F32, gen, 1.0))
        opt = AdamW8bit([p], seed=seed)
        for _ in range(3):
            p.grad = _tensor(5000, F32, gen, 1.0)
            opt.step()
        got.append((p.detach().clone(), opt.state[p]["exp_avg_sq_q"].clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert not torch.equal(got[0][1], got[2][1])


def test_blocks_without_values_and_with_infinite_ones():
    """Zero and tiny gradients leave zero codes and unit scales; an infinity or NaN stays in its block and element."""
    from came_amd import AdamW8bit
    n, B = 1024, 256
    p = torch.nn.Parameter(torch.ones(n, device="cuda"))
    opt = AdamW8bit([p], lr=LR, weight_decay=0.0, block_size=B)
    g = torch.zeros(n)
    g[256:512] = 1e-33  # its square and tenth are under 2^-100
    g[600], g[601] = float("inf"), 1.0
    g[800] = float("nan")
    p.grad = g.cuda()
    opt.step()
    st = {k: v.cpu() for k, v in opt.state[p].items() if isinstance(v, torch.Tensor)}
    assert (st["exp_avg_q"][:512] == 0).all() and (st["exp_avg_sq_q"][:512] == 0).all()
    assert (st["exp_avg_absmax"][:2] == 1).all() and (st["exp_avg_sq_absmax"][:2] == 1).all()
    assert torch.isinf(st["exp_avg_absmax"][2]) and torch.isnan(st["exp_avg_absmax"][3])
    after = p.detach().cpu()
    fine = torch.ones(n, dtype=torch.bool)
    fine[[600, 800]] = False
    assert torch.isfinite(after[fine]).all() and not torch.isfinite(after[~fine]).any()
    assert (after[:256] == 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_counts_and_tensors_of_every_kind(bits):
    """200 tensors (several launches), two groups of their own rates, parameters without gradients in some steps (their
    own step counts), empty, strided and transposed ones, mixed types: each as if it were stepped alone."""
    import came_amd
    cls = came_amd.AdamW8bit if bits == 8 else came_amd.AdamW
    gen = torch.Generator().manual_seed(7)

    def make():
        gen.manual_seed(7)
        out = []
        for i in range(200):
            dt = (F32, BF16, F16)[i % 3]
            if i % 11 == 3:
                q = torch.zeros(0, 5, dtype=dt, device="cuda")
            elif i % 7 == 2:
                q = _tensor(33 * 20, dt, gen, 1.0).view(33, 20).t()
            else:
                q = _tensor(1 + 37 * i, dt, gen, 1.0)
            out.append(torch.nn.Parameter(q))
        return out

    a, b = make(), make()
    opt = cls([{"params": a[:120]}, {"params": a[120:], "lr": 3e-3, "weight_decay": 0.0}], lr=1e-2)
    alone = [cls([q], lr=1e-2 if i < 120 else 3e-3, weight_decay=1e-2 if i < 120 else 0.0) for i, q in enumerate(b)]
    for step in range(3):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = q.grad = None
            if (i + step) % 5:
                p.grad_dtype = q.grad_dtype = F32 if i % 2 else p.dtype
                p.grad = _tensor(p.numel(), p.grad_dtype, gen, 0.1).view(p.shape)
                q.grad = p.grad.clone()
        opt.step()
        for i, o in enumerate(alone):
            if b[i].grad is not None:
                o.step()
    for i, (p, q) in enumerate(zip(a, b)):
        assert torch.equal(p, q), i
        for k, v in opt.state[p].items():
            w = alone[i].state[q][k]
            assert torch.equal(v, w) if isinstance(v, torch.Tensor) else v == w, (i, k)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_clip_in_the_step(bits):
    """max_grad_norm scales by the norm over all groups' gradients and leaves the gradients as they are."""
    import came_amd
    cls = came_amd.AdamW8bit if bits == 8 else came_amd.AdamW
    gen = torch.Generator().manual_seed(1)
    ps = [torch.nn.Parameter(_tensor(n, F32, gen, 1.0)) for n in (3, 5000, 70001)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = cls([{"params": ps[:1]}, {"params": ps[1:]}], lr=LR, max_grad_norm=0.5)
    ref = cls([{"params": qs[:1]}, {"params": qs[1:]}], lr=LR)
    for _ in range(2):
        for p, q in zip(ps, qs):
            p.grad = _tensor(p.numel(), F32, gen, 0.1)
            q.grad = p.grad.clone()
        kept = [p.grad.clone() for p in ps]
        opt.step()
        norm = came_amd.clip_grad_norm_(qs, 0.5)
        ref.step()
        assert torch.equal(norm, opt.last_grad_norm)
        assert all(torch.equal(p.grad, k) for p, k in zip(ps, kept))
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    import came_amd
    cls = came_amd.AdamW8bit if bits == 8 else came_amd.AdamW
    gen = torch.Generator().manual_seed(2)
    p = torch.nn.Parameter(_tensor(1000, BF16, gen, 1.0))
    opt = cls([p])
    p.grad = _tensor(1000, BF16, gen, 1.0)
    opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    two = cls([q])
    two.load_state_dict(opt.state_dict())
    p.grad = _tensor(1000, BF16, gen, 1.0)
    q.grad = p.grad.clone()
    opt.step()
    two.step()
    assert torch.equal(p, q)
    for k, v in opt.state[p].items():
        w = two.state[q][k]
        assert (torch.equal(v, w) and v.dtype == w.dtype) if isinstance(v, torch.Tensor) else v == w
    other = (came_amd.AdamW if bits == 8 else came_amd.AdamW8bit)([q])
    with pytest.raises(RuntimeError, match="layout"):
        other.load_state_dict(opt.state_dict())


def test_torch_adamw_state_carries_over():
    """A torch.optim.AdamW checkpoint continues here: the next steps agree within float32 rounding (three roundings of
    the parameter and of an update of at most a few lr a step)."""
    from came_amd import AdamW
    gen = torch.Generator().manual_seed(4)
    p = torch.nn.Parameter(_tensor(3000, F32, gen, 1.0))
    ref = torch.optim.AdamW([p], lr=LR, weight_decay=WD, foreach=False)
    p.grad = _tensor(3000, F32, gen, 1.0)
    ref.step()
    q = torch.nn.Parameter(p.detach().clone())
    opt = AdamW([q], lr=LR, weight_decay=WD)
    opt.load_state_dict(ref.state_dict())
    for _ in range(3):
        p.grad = _tensor(3000, F32, gen, 1.0)
        q.grad = p.grad.clone()
        ref.step()
        opt.step()
    assert ((p - q).abs() <= 3 * (8 * U * p.abs() + 64 * U * LR)).all()


def test_on_another_stream_and_not_in_a_capture():
    from came_amd import AdamW
    gen = torch.Generator().manual_seed(6)
    p = torch.nn.Parameter(_tensor(1 << 20, F32, gen, 1.0))
    q = torch.nn.Parameter(p.detach().clone())
    a, b = AdamW([p], max_grad_norm=1.0), AdamW([q], max_grad_norm=1.0)
    g = _tensor(1 << 20, F32, gen, 1.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        p.grad = g * 2.0
        a.step()
    torch.cuda.current_stream().wait_stream(s)
    q.grad = g * 2.0
    b.step()
    assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            a.step()
    assert a.state[p]["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_2_31_elements(bits):
    """The elements past 2^31 (and past 2^32 bytes of the gradient) are stepped as a tensor of their own values would be;
    the 8-bit rounding goes by the place in the tensor, so its second moments are compared by their neighbours."""
    import came_amd
    n, tail = (1 << 31) + 1027, 5000
    gen = torch.Generator().manual_seed(8)
    p = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    p.grad = torch.zeros(n, dtype=BF16, device="cuda")
    with torch.no_grad():
        p[-tail:] = _tensor(tail, BF16, gen, 1.0)
    p.grad[-tail:] = _tensor(tail, BF16, gen, 1.0)
    p0, g0 = p.detach()[-tail:].cpu(), p.grad[-tail:].cpu()
    opt = (came_amd.AdamW8bit if bits == 8 else came_amd.AdamW)([p], lr=LR, weight_decay=WD, max_grad_norm=1e9)
    opt.step()
    m1, v1 = orc.moments64(g0, torch.zeros(tail), torch.zeros(tail), BETAS)
    _check_param(p.detach()[-tail:].cpu(), orc.param64(p0, m1, v1, 1, LR, BETAS, EPS, WD), p0, BF16, "tail")
    assert float(p.detach()[: n - tail].abs().amax()) == 0
    assert abs(float(opt.last_grad_norm) / orc.norm64([g0]) - 1) < 1e-6
    if bits == 8:
        assert int(opt.state[p]["exp_avg_q"][-tail:].abs().amax()) == 127
        assert int(opt.state[p]["exp_avg_q"][: n - tail].count_nonzero()) == 0
    else:
        _check_moment(opt.state[p]["exp_avg"][-tail:].cpu(), torch.zeros(tail).double(), g0.double(), m1, "m")
