"""came_amd.int8_linear: sums exact, results within the rounding of their scales."""
import pytest
import torch

from oracle import lm_oracle as orc

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _codes(*shape, gen):
    return torch.randint(-128, 128, shape, generator=gen).to(torch.int8).cuda()


def _operands(T, K, N, dtype, bias, gen):
    return (_codes(T, K, gen=gen), (torch.rand(T, generator=gen) + 0.1).cuda() / 100, _codes(N, K, gen=gen),
            (torch.rand(N, generator=gen) + 0.1).cuda() / 1000, torch.randn(N, generator=gen).to(dtype).cuda() if bias else None)


def _check(q, s, w, ws, b, dtype):
    from came_amd import int8_linear
    y = int8_linear(q, s, w, ws, bias=b, dtype=dtype)
    want, bound = orc.int8_linear(q, s, w, ws, b, dtype)
    err = (y.cpu().double() - want).abs()
    assert y.dtype == dtype and y.shape == (*q.shape[:-1], w.shape[0])
    assert (err <= bound).all(), (float((err - bound).max()), int((err > bound).sum()))
    return y


@pytest.mark.parametrize("dtype,bias", [(F32, True), (BF16, False), (F16, True)])
@pytest.mark.parametrize("T,K,N", [(1, 1, 1), (1, 64, 16), (1, 129, 17), (1, 4096, 500), (3, 1000, 33), (15, 63, 100), (16, 512, 48),
                                   (17, 513, 31), (32, 200, 65), (33, 2731, 90), (48, 5461, 130), (64, 128, 16), (64, 777, 1),
                                   (2, 15, 40), (3, 16, 20), (1, 16, 8193), (1, 4096, 8300), (2, 5461, 8200), (2, 1025, 9001), (1, 9001, 8192),
                                   (16, 11008, 700), (20, 6144, 4096), (20, 6145, 100), (40, 1000, 4097), (64, 6144, 70)])
def test_few_rows(T, K, N, dtype, bias):
    gen = torch.Generator().manual_seed(T + K + N)
    _check(*_operands(T, K, N, dtype, bias, gen), dtype)


@pytest.mark.parametrize("dtype,bias", [(F32, False), (BF16, True), (F16, False)])
@pytest.mark.parametrize("T,K,N", [(65, 1, 1), (65, 16, 70), (66, 17, 64), (100, 128, 65), (129, 127, 129), (200, 4096, 33),
                                   (257, 145, 260), (300, 1003, 300), (130, 2048, 1000), (700, 260, 515), (1021, 512, 1031)])
def test_tiles(T, K, N, dtype, bias):
    gen = torch.Generator().manual_seed(T + K + N)
    _check(*_operands(T, K, N, dtype, bias, gen), dtype)


@pytest.mark.parametrize("T,K,N", [(2048, 1100, 2304), (4100, 640, 4100)])
def test_large_tiles(T, K, N):
    gen = torch.Generator().manual_seed(K)
    _check(*_operands(T, K, N, BF16, True, gen), BF16)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_the_largest_sums(T):
    """131071 products of -128 by -128 are the most that 32 bits hold."""
    from came_amd import int8_linear
    K = 131071
    q, w = torch.full((T, K), -128, dtype=torch.int8, device="cuda"), torch.full((20, K), -128, dtype=torch.int8, device="cuda")
    w[3] = 127
    s, ws = torch.ones(T, device="cuda"), torch.ones(20, device="cuda")
    y = int8_linear(q, s, w, ws, dtype=F32).cpu()
    want = torch.full((T, 20), float(K * 128 * 128))
    want[:, 3] = -float(K * 128 * 127)
    assert torch.equal(y, want)


@pytest.mark.parametrize("T", [5, 64, 65, 200])
def test_operands_where_they_lie(T):
    """Slices whose rows start anywhere, with other codes behind them, give what contiguous copies give."""
    from came_amd import int8_linear
    gen = torch.Generator().manual_seed(T)
    wide, weights = _codes(T, 400, gen=gen), _codes(150, 700, gen=gen)
    s, ws = torch.rand(T, generator=gen).cuda(), torch.rand(150, generator=gen).cuda()
    for k0, K in ((0, 400), (1, 333), (3, 17), (4, 100), (16, 128), (7, 130), (2, 1)):
        q = wide[:, k0 : k0 + K]
        for w in (weights[:, k0 : k0 + K], weights[:, 300 - k0 : 300 - k0 + K], weights.t()[:K].t(), weights[:K, :150].t()[:, :K]):
            if w.shape[1] != K:
                continue
            want = int8_linear(q.contiguous(), s, w.contiguous(), ws[: w.shape[0]], dtype=F32)
            assert torch.equal(int8_linear(q, s, w, ws[: w.shape[0]], dtype=F32), want)
            exact, bound = orc.int8_linear(q, s, w, ws[: w.shape[0]], None, F32)
            assert ((want.cpu().double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("T", [3, 16, 70, 300])
@pytest.mark.parametrize("width", [401, 402, 403, 404])
def test_rows_any_distance_apart(T, width):
    """Rows that start on words, on two in four, one in four or none, with other codes between them."""
    from came_amd import int8_linear
    gen = torch.Generator().manual_seed(width)
    wide, weights = _codes(T, width, gen=gen), _codes(130, width + 5, gen=gen)
    s, ws = torch.rand(T, generator=gen).cuda(), torch.rand(130, generator=gen).cuda()
    for k0, K in ((0, 400), (1, 399), (2, 80), (3, 145)):
        q, w = wide[:, k0 : k0 + K], weights[:, 3 - k0 : 3 - k0 + K]
        got = int8_linear(q, s, w, ws, dtype=F32)
        exact, bound = orc.int8_linear(q, s, w, ws, None, F32)
        assert ((got.cpu().double() - exact).abs() <= bound).all(), (k0, K)


def test_shapes_and_strides():
    from came_amd import int8_linear, quantize_rows
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(4, 50, 77, generator=gen).cuda()
    q, s = quantize_rows(x)
    w, ws = quantize_rows(torch.randn(90, 77, generator=gen).cuda())
    y = int8_linear(q, s, w, ws, dtype=F32)
    assert torch.equal(y.view(200, 90), int8_linear(q.reshape(200, 77), s.flatten(), w, ws, dtype=F32))
    assert torch.equal(y.transpose(0, 1), int8_linear(q.transpose(0, 1), s.t(), w, ws, dtype=F32))
    assert torch.equal(y[1, 3], int8_linear(q[1, 3], s[1, 3], w, ws, dtype=F32))
    assert torch.equal(y[:, ::3], int8_linear(q[:, ::3], s[:, ::3], w, ws, dtype=F32))
    assert int8_linear(q[:0], s[:0], w, ws).shape == (0, 50, 90)
    exact = (x.double() @ (w.double() * ws[:, None].double()).t()).cpu()
    step = s.cpu().double()[..., None] * 0.51 * (w.double().abs().sum(1) * ws.double()).cpu()
    assert ((y.cpu().double() - exact).abs() <= step).all()  # half a code of every activation


def test_scales_that_are_not_finite():
    """They make their row, or column, NaN or infinite, and no other."""
    gen = torch.Generator().manual_seed(4)
    for T in (9, 100):
        q, s, w, ws, _ = _operands(T, 100, 50, F32, False, gen)
        from came_amd import int8_linear
        clean = int8_linear(q, s, w, ws, dtype=F32)
        s[3], ws[20] = float("nan"), float("inf")
        q[5] = 0
        y = int8_linear(q, s, w, ws, dtype=F32)
        rows, cols = torch.ones(T, dtype=torch.bool, device="cuda"), torch.ones(50, dtype=torch.bool, device="cuda")
        rows[[3, 5]], cols[20] = False, False
        assert torch.equal(y[rows][:, cols], clean[rows][:, cols]) and torch.isnan(y[3]).all()
        assert torch.isnan(y[5, 20]) and not y[5, cols].any() and not torch.isfinite(y[:, 20]).any()


def test_the_norm_and_the_product_together():
    """What a serving program runs: the norm with the residual's addition in 8 bits, then the product, against 64 bits."""
    from came_amd import int8_linear, quantize_rows, rms_norm_int8
    gen = torch.Generator().manual_seed(5)
    for T in (1, 30, 500):
        x, r = (torch.randn(T, 640, generator=gen).to(BF16).cuda() for _ in range(2))
        nw = (1 + 0.2 * torch.randn(640, generator=gen)).to(BF16).cuda()
        w = torch.randn(1000, 640, generator=gen) / 25
        wq, ws = quantize_rows(w.cuda())
        q, s, h = rms_norm_int8(x, nw, residual=r)
        y = int8_linear(q, s, wq, ws)
        held = (wq.double() * ws[:, None].double()).cpu()
        exact = orc.rms_norm(x, nw, 1e-6, r)[0]
        half = 0.51 * s.cpu().double()[:, None] * held.abs().sum(1)
        want = exact @ held.t()
        assert ((y.cpu().double() - want).abs() <= half + orc.UNIT[BF16] * (want.abs() + half)).all()


def test_on_another_stream_and_in_a_graph():
    from came_amd import int8_linear
    gen = torch.Generator().manual_seed(6)
    for T in (4, 90):
        q, s, w, ws, b = _operands(T, 600, 333, BF16, True, gen)
        want = int8_linear(q, s, w, ws, bias=b)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = int8_linear(q, s, w, ws, bias=b)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = int8_linear(q, s, w, ws, bias=b)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(want, got)
        for _ in range(4):
            q.copy_(_codes(T, 600, gen=gen))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(int8_linear(q, s, w, ws, bias=b), held)


def test_results_past_2_31_elements():
    from came_amd import int8_linear
    T, N = 70_000, 32_768
    q, w = torch.zeros(T, 16, dtype=torch.int8, device="cuda"), torch.ones(N, 16, dtype=torch.int8, device="cuda")
    q[-1] = 2
    y = int8_linear(q, torch.ones(T, device="cuda"), w, torch.ones(N, device="cuda"), dtype=F16)
    assert (y[-1] == 32).all() and not y[:-1].any()


def test_refusals():
    from came_amd import int8_linear
    gen = torch.Generator().manual_seed(7)
    q, s, w, ws, b = _operands(3, 8, 5, BF16, True, gen)
    for bad in ((q, s[:2], w, ws), (q, s, w[:, :7], ws), (q, s, w, ws[:4]), (q, s, w[:0], ws[:0]), (q, s, w[0], ws)):
        with pytest.raises(ValueError):
            int8_linear(*bad)
    big = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError, match="131071"):
        int8_linear(big, s[:1], big, ws[:1])
    for bad, match in (((q.int(), s, w, ws), "q must be"), ((q, s.double(), w, ws), "scale must be"), ((q, s, w.cpu(), ws), "GPU"),
                       ((q, s, w, ws.half()), "w_scale must be"), ((q, s.requires_grad_(), w, ws), "no gradient")):
        with pytest.raises(RuntimeError, match=match):
            int8_linear(*bad)
    s = s.detach()
    with pytest.raises(RuntimeError, match="bias"):
        int8_linear(q, s, w, ws, bias=b, dtype=F32)
    with pytest.raises(ValueError, match="dtype"):
        int8_linear(q, s, w, ws, dtype=torch.int8)
