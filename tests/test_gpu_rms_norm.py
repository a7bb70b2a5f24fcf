"""came_amd.rms_norm, rms_norm_int8 and quantize_rows against their formulas in 64 bits."""
import pytest
import torch

from oracle import lm_oracle as orc

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# around the widths that 16 lanes, a wavefront, 256 and 1024 threads hold, and past them
WIDTHS = [1, 2, 7, 8, 33, 64, 65, 127, 128, 129, 255, 257, 511, 512, 513, 1000, 1025, 2047, 2049, 2731, 4096, 4097, 5461, 8192, 8193,
          16383, 16384, 16385, 40001]


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _close(got, want, bound, what):
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), (what, float((err - bound).max()), int((err > bound).sum()))


def _operands(T, D, dtype, residual, gen):
    x = torch.randn(T, D, generator=gen).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(D, generator=gen)).to(dtype).cuda()
    r = (3 * torch.randn(T, D, generator=gen)).to(dtype).cuda() if residual else None
    return x, w, r


def _check(x, w, r, dy, dh, eps=1e-6):
    from came_amd import rms_norm
    leaves = [t.detach().requires_grad_() for t in (x, w, r) if t is not None]
    out = rms_norm(leaves[0], leaves[1], eps=eps, residual=leaves[2] if r is not None else None)
    y, h = (out, None) if r is None else out
    want, bound, ho = orc.rms_norm(x, w, eps, r)
    if r is not None:
        assert torch.equal(h.detach().cpu(), ho)
    _close(y.detach(), want, orc.rounded(bound, want, x.dtype), "y")
    with torch.no_grad():
        plain = rms_norm(x, w, eps=eps, residual=r)
        assert torch.equal(plain if r is None else plain[0], y)
    (dx, ex), (dw, ew) = orc.rms_norm_gradients(ho, w, eps, dy, dh)
    grads = torch.autograd.grad((y,) if r is None else (y, h), leaves, (dy,) if r is None else (dy, dh))
    _close(grads[0], dx, ex, "dx")
    _close(grads[1], dw, ew, "dweight")
    if r is not None:
        assert torch.equal(grads[0], grads[2])
    assert [g.shape for g in grads] == [t.shape for t in leaves] and all(g.dtype == x.dtype for g in grads)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", WIDTHS)
def test_matches_the_formulas(D, dtype):
    gen = torch.Generator().manual_seed(D)
    for T, residual in ((1, True), (5, False), (70, True)):
        x, w, r = _operands(T, D, dtype, residual, gen)
        dy, dh = (torch.randn(T, D, generator=gen).to(dtype).cuda() for _ in range(2))
        _check(x, w, r, dy, dh if residual else None)


@pytest.mark.parametrize("T,D,dtype", [(4099, 72, BF16), (40000, 8, F32), (2500, 1030, F16), (1300, 20000, BF16), (1021, 2731, F16)])
def test_many_rows(T, D, dtype):
    gen = torch.Generator().manual_seed(T)
    x, w, r = _operands(T, D, dtype, True, gen)
    dy, dh = (torch.randn(T, D, generator=gen).to(dtype).cuda() for _ in range(2))
    _check(x, w, r, dy, dh, eps=1e-3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", WIDTHS)
def test_rows_in_8_bits(D, dtype):
    """Every code is the nearest one, of rows as they are and of the norm's."""
    from came_amd import quantize_rows, rms_norm, rms_norm_int8
    gen = torch.Generator().manual_seed(D + 1)
    for T, residual in ((1, False), (37, True)):
        x, w, r = _operands(T, D, dtype, residual, gen)
        x[0, D // 2] *= 40
        q, s = quantize_rows(x)
        qo, so = orc.quantize_rows(x)
        assert torch.equal(q.cpu(), qo) and ((s.cpu().double() - so).abs() <= orc.U * so).all()
        got = rms_norm_int8(x, w, residual=r)
        qo, so, bound, h = orc.rms_norm_int8(x, w, 1e-6, r)
        if residual:
            assert torch.equal(got[2].cpu(), h) and torch.equal(got[2], rms_norm(x, w, residual=r)[1])
        assert torch.equal(got[0].cpu(), qo) and ((got[1].cpu().double() - so).abs() <= bound).all()
        assert (got[0].cpu().int().abs().amax(-1) == 127).all()
        for codes in (got[0], quantize_rows(x)[0]):  # rows start at 16 bytes, zeros behind them
            ld = codes.stride(0) if T > 1 else -(-D // 16) * 16
            assert ld == -(-D // 16) * 16 and codes.data_ptr() % 16 == 0
            behind = codes.as_strided((T, ld), (ld, 1))[:, D:]
            assert not behind.any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,D", [(4000, 640), (40, 20000)])
def test_values_next_to_a_border_take_the_nearest_code(T, D, dtype):
    """Halves of codes, and what is next to them: exact ties go to the even code."""
    from came_amd import quantize_rows, rms_norm_int8
    gen = torch.Generator().manual_seed(D)
    x = (torch.randint(-127, 127, (T, D), generator=gen) + 0.5) * (1 + 2.0**-23 * torch.randint(-3, 4, (T, D), generator=gen))
    x[:, 0] = 127.0
    x = (x * torch.exp(torch.randn(T, 1, generator=gen))).to(dtype).cuda()
    x[:, 1] = x[:, 0] / 2
    w = torch.exp(0.3 * torch.randn(D, generator=gen)).to(dtype).cuda()
    assert torch.equal(quantize_rows(x)[0].cpu(), orc.quantize_rows(x)[0])
    assert (quantize_rows(x)[0][:, 1] == 64).all()  # 63.5
    assert torch.equal(rms_norm_int8(x, w)[0].cpu(), orc.rms_norm_int8(x, w, 1e-6)[0])


def test_rows_without_finite_or_normal_values():
    from came_amd import quantize_rows, rms_norm, rms_norm_int8
    x = torch.randn(9, 100, generator=torch.Generator().manual_seed(0))
    x[1] = 0
    x[2] = 0
    x[2, 5] = 2.0**-101
    x[3, 7] = float("inf")
    x[4, 8] = float("nan")
    x[5] *= 1e30 / x[5].abs().max()
    x[6] = 0
    x[6, 99] = -(2.0**-99)
    x[7, 3], x[7, 4] = float("inf"), float("nan")
    x = x.cuda()
    q, s = quantize_rows(x)
    qo, so = orc.quantize_rows(x)
    assert torch.equal(q.cpu(), qo) and torch.equal(s.cpu().nan_to_num(nan=-1.0), so.float().nan_to_num(nan=-1.0))
    assert not q[[1, 2, 3, 4, 7]].any() and float(s[1]) == 0 and float(s[2]) == 0 and torch.isinf(s[3]) and torch.isnan(s[[4, 7]]).all()
    for rows in (x, x.to(BF16)):
        w = torch.ones(100, device="cuda", dtype=rows.dtype)
        want = orc.rms_norm(rows, w, 1e-6)[0]
        y = rms_norm(rows, w).cpu()
        fine = [0, 1, 2, 6, 8]
        assert torch.isfinite(y[fine]).all() and torch.isnan(y[[4, 7]]).all() and torch.isnan(y[3, 7])
        assert torch.equal(torch.isfinite(want[fine]), torch.isfinite(y[fine]))
        c, sc = rms_norm_int8(rows, w)
        assert torch.isfinite(sc[fine]).all() and not torch.isfinite(sc[[3, 4, 7]]).any() and not c[[3, 4, 7]].any()
    with torch.no_grad():  # a row of zeros without eps has no direction
        assert torch.isnan(rms_norm(x[1], torch.ones(100, device="cuda"), eps=0.0)).all()


def test_shapes_strides_and_types_of_operands():
    from came_amd import quantize_rows, rms_norm, rms_norm_int8
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(6, 4, 50, generator=gen).to(BF16).cuda()
    w = torch.randn(33, generator=gen).to(BF16).cuda()
    for x in (wide[..., 1:34], wide[::2, :, 17:], wide.transpose(0, 1)[..., :33], wide[:1, :1, :33].expand(5, 4, 33),
              torch._neg_view(wide)[..., :33], wide[0, 0, 2:35]):
        c = x.resolve_neg().contiguous().clone()
        r = torch.randn(x.shape, generator=gen).to(BF16).cuda()
        assert torch.equal(rms_norm(x, w), rms_norm(c, w))
        for a, b in zip(rms_norm(x, w, residual=r), rms_norm(c, w, residual=r)):
            assert torch.equal(a, b) and a.shape == x.shape
        for a, b in zip(rms_norm(r, w, residual=x), rms_norm(r, w, residual=c)):
            assert torch.equal(a, b)
        for a, b in zip(rms_norm_int8(x, w, residual=r), rms_norm_int8(c, w, residual=r)):
            assert torch.equal(a, b)
        assert all(torch.equal(a, b) for a, b in zip(quantize_rows(x), quantize_rows(c)))
        leaf, other = x.detach().requires_grad_(), c.detach().requires_grad_()
        dy = torch.randn(*x.shape[::-1], generator=gen).to(BF16).cuda().permute(*range(x.dim() - 1, -1, -1))
        a, = torch.autograd.grad(rms_norm(leaf, w), leaf, dy)
        b, = torch.autograd.grad(rms_norm(other, w), other, dy.contiguous())
        assert torch.equal(a, b)
    for strided in (torch.randn(66, generator=gen).to(BF16).cuda()[::2], w.expand(33)):
        assert torch.equal(rms_norm(wide[..., :33], strided), rms_norm(wide[..., :33], strided.contiguous()))


def test_no_rows_and_single_gradients():
    from came_amd import quantize_rows, rms_norm, rms_norm_int8
    gen = torch.Generator().manual_seed(4)
    x, w, r = _operands(12, 40, F32, True, gen)
    dy, dh = (torch.randn(12, 40, generator=gen).cuda() for _ in range(2))
    every = [t.detach().requires_grad_() for t in (x, w, r)]
    y, h = rms_norm(every[0], every[1], residual=every[2])
    want = torch.autograd.grad((y, h), every, (dy, dh))
    for needs in ((True, False, False), (False, True, False), (False, False, True), (True, True, False), (False, True, True)):
        ops = [t.detach().requires_grad_(n) for t, n in zip((x, w, r), needs)]
        y, h = rms_norm(ops[0], ops[1], residual=ops[2])
        got = torch.autograd.grad((y, h), [t for t, n in zip(ops, needs) if n], (dy, dh))
        assert all(torch.equal(a, b) for a, b in zip(got, [g for g, n in zip(want, needs) if n]))
    y, h = rms_norm(every[0], every[1], residual=every[2])
    a = torch.autograd.grad(h, every, dh, allow_unused=True, retain_graph=True)  # h alone is used
    assert torch.equal(a[0], dh) and torch.equal(a[2], dh) and (a[1] is None or not a[1].any())
    b = torch.autograd.grad(y, every, dy)  # y alone
    c = torch.autograd.grad(rms_norm((x + r).requires_grad_(), every[1]), every[1], dy)[0]
    assert torch.equal(b[1], c) and torch.equal(b[0], b[2])
    empty = x[:0].detach().requires_grad_()
    weight = w.detach().requires_grad_()
    y, h = rms_norm(empty, weight, residual=r[:0])
    gx, gw = torch.autograd.grad((y, h), (empty, weight), (y, h))
    assert y.shape == (0, 40) and gx.shape == (0, 40) and not gw.any()
    assert rms_norm_int8(x[:0], w)[0].shape == (0, 40) and quantize_rows(x[:0])[1].shape == (0,)


def test_a_residual_that_is_x():
    from came_amd import rms_norm
    gen = torch.Generator().manual_seed(5)
    x, w, _ = _operands(9, 130, F32, False, gen)
    dy, dh = (torch.randn(9, 130, generator=gen).cuda() for _ in range(2))
    a, b = (t.detach().requires_grad_() for t in (x, w))
    y, h = rms_norm(a, b, residual=a)
    ga, gb = torch.autograd.grad((y, h), (a, b), (dy, dh))
    (dx, ex), (dw, ew) = orc.rms_norm_gradients(2 * x, w, 1e-6, dy, dh)
    _close(ga, 2 * dx, 2 * ex, "dx")
    _close(gb, dw, ew, "dweight")


@pytest.mark.parametrize("D", [24, 3000])
def test_gradients_against_differences(D):
    """Along a random direction, the change of <dy, y> in 64 bits against <gradient, direction>."""
    from came_amd import rms_norm
    gen = torch.Generator().manual_seed(6)
    x, w, r = _operands(5, D, F32, True, gen)
    dy, dh = (torch.randn(5, D, generator=gen).cuda() for _ in range(2))
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    y, h = rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=1e-2)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    ops = [t.cpu().double() for t in (x, w, r)]

    def value(x, w, r):
        h = x + r
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-2) * w
        return (y * dy.cpu().double()).sum() + (h * dh.cpu().double()).sum()

    for k in range(3):
        d = torch.randn(ops[k].shape, generator=gen, dtype=torch.float64)
        e = 1e-4
        diff = (value(*[t + e * d if i == k else t for i, t in enumerate(ops)]) -
                value(*[t - e * d if i == k else t for i, t in enumerate(ops)])) / (2 * e)
        along = (grads[k].cpu().double() * d).sum()
        assert abs(diff - along) <= 1e-4 * (grads[k].cpu().double() * d).norm(), k


def test_rows_do_not_mix():
    from came_amd import rms_norm
    gen = torch.Generator().manual_seed(7)
    for D in (40, 700, 3000, 9000):
        x, w, r = _operands(50, D, F32, True, gen)
        dy, dh = (torch.randn(50, D, generator=gen).cuda() for _ in range(2))
        clean = x.detach().requires_grad_()
        bad = x.clone()
        bad[11, D - 1], bad[40, 0] = float("nan"), float("inf")
        bad.requires_grad_()
        (y0, h0), (y1, h1) = (rms_norm(t, w, residual=r) for t in (clean, bad))
        g0, = torch.autograd.grad((y0, h0), clean, (dy, dh))
        g1, = torch.autograd.grad((y1, h1), bad, (dy, dh))
        rows = torch.ones(50, dtype=torch.bool, device="cuda")
        rows[[11, 40]] = False
        assert torch.equal(y0[rows], y1[rows]) and torch.equal(g0[rows], g1[rows]) and torch.isnan(y1[11]).all()


def test_the_same_inputs_give_the_same_bits():
    from came_amd import rms_norm
    gen = torch.Generator().manual_seed(8)
    x, w, r = _operands(3000, 1100, BF16, True, gen)
    dy, dh = (torch.randn(3000, 1100, generator=gen).to(BF16).cuda() for _ in range(2))
    seen = None
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (x, w)]
        y, h = rms_norm(leaves[0], leaves[1], residual=r)
        got = [y.detach(), *torch.autograd.grad((y, h), leaves, (dy, dh))]
        torch.empty(1 << 24, device="cuda").fill_(float("nan"))
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, got))
        seen = got


def test_rows_past_2_31_elements():
    from came_amd import quantize_rows, rms_norm
    T, D = 70_000, 32_768
    x = torch.zeros(T, D, dtype=F16, device="cuda")
    x[-1] = 2.0
    w = torch.ones(D, dtype=F16, device="cuda")
    y = rms_norm(x, w)
    assert (y[-1] == 1).all() and not y[:-1].any()
    q, s = quantize_rows(x)
    assert (q[-1] == 127).all() and not q[:-1].any() and not s[:-1].any()


def test_on_another_stream_and_in_a_graph():
    from came_amd import quantize_rows, rms_norm, rms_norm_int8
    gen = torch.Generator().manual_seed(9)
    x, w, r = _operands(130, 300, BF16, True, gen)
    dy, dh = (torch.randn(130, 300, generator=gen).to(BF16).cuda() for _ in range(2))
    leaves = [t.detach().requires_grad_() for t in (x, w)]

    def both():
        y, h = rms_norm(leaves[0], leaves[1], residual=r)
        with torch.no_grad():
            q = rms_norm_int8(leaves[0], leaves[1], residual=r) + quantize_rows(x)
        return [y.detach(), h.detach(), *q, *torch.autograd.grad((y, h), leaves, (dy, dh))]

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for k in range(4):
        r.copy_(torch.randn(130, 300, generator=gen).to(BF16).cuda())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(both(), held))


def test_gradients_of_gradients_and_refusals():
    from came_amd import quantize_rows, rms_norm, rms_norm_int8
    x, w = torch.randn(3, 8, device="cuda", requires_grad=True), torch.ones(8, device="cuda")
    g, = torch.autograd.grad(rms_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="rms_norm is differentiable once"):
        g.sum().backward()
    for call in (lambda: rms_norm_int8(x, w), lambda: quantize_rows(x)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    for bad in ((x, w[:7]), (x, w[None]), (x[:, :0], w[:0]), (torch.zeros((), device="cuda"), w)):
        with pytest.raises(ValueError):
            rms_norm(*bad)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            rms_norm(x, w, eps=eps)
    with pytest.raises(ValueError, match="residual"):
        rms_norm(x, w, residual=x[:2])
    for bad, match in (((x.double(), w.double()), "dtype"), ((x, w.to(BF16)), "weight"), ((x, w.cpu()), "GPU")):
        with pytest.raises(RuntimeError, match=match):
            rms_norm(*bad)
    y = rms_norm(x, w)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
