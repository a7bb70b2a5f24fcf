"""came_amd.embedding against its definition: rows bit for bit, gradients within the rounding of float32 sums."""
import pytest
import torch

from oracle import lm_oracle as orc

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _tokens(kind, T, V, gen):
    if kind == "zipf":
        u = torch.rand(T, generator=gen, dtype=torch.float64)
        return (torch.exp(u * torch.log(torch.tensor(V + 1.0, dtype=torch.float64))).long() - 1).clamp(0, V - 1)
    if kind == "same":
        return torch.full((T,), V // 2)
    if kind == "last":
        return torch.full((T,), V - 1)
    if kind == "outside":  # a third of them
        return torch.randint(-V, 2 * V, (T,), generator=gen)
    if kind == "runs":  # runs of lengths around a share's
        lens = torch.randint(1, 70, (T,), generator=gen)
        return torch.repeat_interleave(torch.randperm(max(V, T), generator=gen)[:T] % V, lens)[:T]
    return torch.randint(0, V, (T,), generator=gen)


def _check(tokens, weight, dy, scale=1.0, padding=None):
    from came_amd import embedding
    w = weight.detach().requires_grad_()
    y = embedding(tokens, w, scale=scale, padding_idx=padding)
    assert y.dtype == w.dtype and y.shape == (*tokens.shape, w.shape[1])
    assert torch.equal(y.detach().cpu(), orc.embedding(tokens, w, scale))
    with torch.no_grad():
        assert torch.equal(embedding(tokens, w, scale=scale), y)
    g, = torch.autograd.grad(y, w, dy)
    want, bound = orc.embedding_gradient(tokens, dy, w.shape[0], scale, None if padding is None else padding % w.shape[0])
    err = (g.cpu().double() - want).abs()
    assert g.shape == w.shape and g.dtype == w.dtype
    assert (err <= bound).all(), (float((err - bound).max()), int((err > bound).sum()))
    return g


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 50, 8), (2, 3, 7), (17, 9, 129), (63, 1000, 64), (64, 257, 513), (65, 40, 1000),
                                   (300, 5000, 96), (1021, 300, 2049), (4099, 777, 40)])
def test_matches_the_definition(T, V, D, dtype):
    gen = torch.Generator().manual_seed(T + V + D)
    w = torch.randn(V, D, generator=gen).to(dtype).cuda()
    dy = torch.randn(T, D, generator=gen).to(dtype).cuda()
    _check(_tokens("any", T, V, gen).cuda(), w, dy)


@pytest.mark.parametrize("kind", ["zipf", "same", "last", "outside", "runs"])
@pytest.mark.parametrize("dtype,tokens", [(F32, torch.int32), (BF16, torch.int64), (F16, torch.int32)])
@pytest.mark.parametrize("T,V,D", [(700, 31, 72), (9001, 2100, 130)])
def test_distributions_of_tokens(kind, dtype, tokens, T, V, D):
    gen = torch.Generator().manual_seed(len(kind) + T)
    t = _tokens(kind, T, V, gen).to(tokens).cuda()
    w = torch.randn(V, D, generator=gen).to(dtype).cuda()
    dy = torch.randn(T, D, generator=gen).to(dtype).cuda()
    _check(t, w, dy, scale=0.37, padding=3)
    _check(t, w, dy, scale=-11.3137, padding=-V // 2 if V > 3 else None)


def test_long_runs_are_summed_over_many_shares():
    """One token at 70000 positions: shares of 35 of them, thousands of sums joined."""
    gen = torch.Generator().manual_seed(1)
    w = torch.randn(5, 16, generator=gen).cuda()
    dy = torch.randn(70000, 16, generator=gen).cuda()
    t = torch.full((70000,), 2)
    t[torch.randint(0, 70000, (9000,), generator=gen)] = 4
    _check(t.cuda(), w, dy)


def test_more_tokens_than_one_pass_of_ranges():
    """A vocabulary past 256 ranges of the most tokens a workgroup counts."""
    gen = torch.Generator().manual_seed(2)
    V = 300_001
    t = torch.cat([torch.randint(0, V, (3000,), generator=gen), torch.tensor([0, V - 1, V, -1, 255_999, 256_000])]).cuda()
    w = torch.randn(V, 3, generator=gen).cuda()
    _check(t, w, torch.randn(len(t), 3, generator=gen).cuda())


def test_shapes_strides_and_types_of_operands():
    from came_amd import embedding
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(40, 100, generator=gen).to(BF16).cuda()
    t = torch.randint(0, 40, (6, 10), generator=gen).cuda()
    for w in (wide[:, 3:72], wide.t()[:40], wide[::2][:, 1:], wide[0].expand(40, 100), torch._neg_view(wide)):
        tt = t % w.shape[0]
        for tokens in (tt, tt.t(), tt[::2, 1::3], tt.int()):
            want = orc.embedding(tokens, w.resolve_neg(), 2.0)
            assert torch.equal(embedding(tokens, w, scale=2.0).cpu(), want)
    leaf = wide.clone().requires_grad_()
    dy = torch.randn(6, 100, 10, generator=gen).to(BF16).cuda().transpose(1, 2)
    a, = torch.autograd.grad(embedding(t, leaf), leaf, dy)
    b, = torch.autograd.grad(embedding(t, leaf), leaf, dy.contiguous())
    c, = torch.autograd.grad(embedding(t.flatten(), leaf), leaf, torch._neg_view(-dy.reshape(60, 100)))
    assert torch.equal(a, b) and torch.equal(a, c)
    view = leaf[:, 1:70]  # a gradient of a slice
    d, = torch.autograd.grad(embedding(t, view), leaf, dy[..., 1:70])
    assert torch.equal(d[:, 1:70], a[:, 1:70]) and not d[:, 0].any() and not d[:, 70:].any()
    assert embedding(torch.tensor(7, device="cuda"), wide).shape == (100,)
    none = embedding(t[:0], leaf)
    assert none.shape == (0, 10, 100)
    e, = torch.autograd.grad(none, leaf, torch.zeros_like(none))
    assert not e.any()


def test_rows_behind_the_last_and_other_rows_stay():
    """Infinities and NaN of one token's positions reach its row of the gradient alone; tokens outside write nothing."""
    gen = torch.Generator().manual_seed(4)
    w = torch.randn(20, 33, generator=gen).cuda()
    t = torch.randint(0, 20, (500,), generator=gen)
    dy = torch.randn(500, 33, generator=gen)
    dy[t == 7] = float("inf")
    dy[t == 8] = float("nan")
    from came_amd import embedding
    leaf = w.requires_grad_()
    g, = torch.autograd.grad(embedding(t.cuda(), leaf), leaf, dy.cuda())
    rows = torch.ones(20, dtype=torch.bool)
    rows[[7, 8]] = False
    assert torch.isfinite(g.cpu()[rows]).all() and torch.isinf(g[7]).all() and torch.isnan(g[8]).all()


def test_the_same_inputs_give_the_same_bits():
    from came_amd import embedding
    gen = torch.Generator().manual_seed(5)
    t = _tokens("zipf", 20000, 1500, gen).cuda()
    w = torch.randn(1500, 200, generator=gen).cuda().requires_grad_()
    dy = torch.randn(20000, 200, generator=gen).cuda()
    first, = torch.autograd.grad(embedding(t, w), w, dy)
    for _ in range(3):
        torch.empty(1 << 24, device="cuda").fill_(float("nan"))  # other values where workspaces may lie
        again, = torch.autograd.grad(embedding(t, w), w, dy)
        assert torch.equal(first, again)


def test_rows_past_2_31_elements():
    from came_amd import embedding
    V, D = 70_000, 32_768
    w = torch.zeros(V, D, dtype=F16, device="cuda")
    w[-1] = 2.0
    w[-2, -1] = 3.0
    t = torch.tensor([V - 1, V - 2, 0, V - 1], device="cuda")
    y = embedding(t, w.requires_grad_())
    assert (y[0] == 2).all() and (y[3] == 2).all() and float(y[1].detach().sum()) == 3 and not y[2].any()
    g, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert (g[-1] == 2).all() and (g[-2] == 1).all() and (g[0] == 1).all() and not g[1:-2].any()


def test_on_another_stream_and_in_a_graph():
    from came_amd import embedding
    gen = torch.Generator().manual_seed(6)
    t = torch.randint(0, 90, (400,), generator=gen).cuda()
    w = torch.randn(90, 65, generator=gen).cuda().requires_grad_()
    dy = torch.randn(400, 65, generator=gen).cuda()

    def both():
        y = embedding(t, w, scale=0.5, padding_idx=1)
        return y.detach(), torch.autograd.grad(y, w, dy)[0]

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
        t.copy_(torch.randint(0, 90, (400,), generator=gen).cuda() if k else t)
        graph.replay()
        torch.cuda.synchronize()
        eager = both()
        assert all(torch.equal(a, b) for a, b in zip(eager, held))


def test_gradients_of_gradients_and_refusals():
    from came_amd import embedding
    t, w = torch.zeros(3, dtype=torch.long, device="cuda"), torch.randn(4, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(embedding(t, w).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="embedding is differentiable once"):
        g.sum().backward()
    for bad, match in (((t.float(), w), "int64 or int32"), ((t, w.double()), "dtype"), ((t.cpu(), w), "GPU"), ((t, [1]), "GPU")):
        with pytest.raises(RuntimeError, match=match):
            embedding(*bad)
    for shape in ((0, 8), (4, 0), (8,)):
        with pytest.raises(ValueError):
            embedding(t, torch.zeros(shape, device="cuda"))
    for padding in (4, -5):
        with pytest.raises(ValueError, match="padding_idx"):
            embedding(t, w, padding_idx=padding)
    y = embedding(t, w)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
