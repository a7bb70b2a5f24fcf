"""came_amd.token_log_probs against its definition in 64 bits."""
import pytest
import torch

from oracle import lm_oracle as orc

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _close(got, want, bound, what):
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), (what, float((err - bound).max()), int((err > bound).sum()))


def _order(z, top):
    """The `top` largest, of equal ones the lowest first."""
    return torch.sort(z.detach().cpu().double(), dim=-1, descending=True, stable=True).indices[..., :top]


def _check(z, t, top=0, dlp=None, dent=None):
    from came_amd import token_log_probs
    leaf = z.detach().requires_grad_()
    r = token_log_probs(leaf, t, top=top)
    (lp, elp), (H, eh), kept = orc.log_probs(z, t)
    _close(r.log_probs.detach(), lp, elp, "log_probs")
    _close(r.entropy.detach(), H, eh, "entropy")
    assert r.top_tokens.shape == r.top_log_probs.shape == (*t.shape, top)
    if top:
        order = _order(z, top)
        assert torch.equal(r.top_tokens.cpu(), order)
        want = kept[0].gather(-1, order)
        far = (want + kept[1][..., None] * 0).abs()
        some = torch.isfinite(want)
        assert torch.equal(r.top_log_probs.cpu()[~some].double(), want[~some])
        bound = kept[1][..., None] + orc.U * (4 * far + 2 * kept[2][..., None])
        _close(r.top_log_probs.cpu()[some], want[some], bound[some], "top_log_probs")
        assert not r.top_log_probs.requires_grad
    gen = torch.Generator().manual_seed(t.numel())
    both = [torch.randn(t.shape, generator=gen).cuda() if g is None else g for g in (dlp, dent)]
    for a, b in ((both[0], both[1]), (both[0], None), (None, both[1])):
        g, = torch.autograd.grad([o for o, d in zip((r.log_probs, r.entropy), (a, b)) if d is not None], leaf,
                                 [d for d in (a, b) if d is not None], retain_graph=True)
        want, bound = orc.log_probs_gradient(kept, a, b, z.dtype)
        _close(g, want, bound, "dlogits")
        assert g.dtype == z.dtype and g.shape == z.shape
    with torch.no_grad():
        again = token_log_probs(z, t, top=top)
        assert torch.equal(again.log_probs, r.log_probs) and torch.equal(again.top_tokens, r.top_tokens)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 2, 0), (2, 7, 7), (1, 64, 64), (5, 200, 20), (700, 513, 3), (600, 1025, 64), (3, 1000, 64),
                                     (1, 4097, 20), (40, 8191, 5), (600, 3000, 20), (1, 32000, 20), (3, 50257, 5), (513, 9001, 0),
                                     (2, 131072, 64), (520, 16385, 8), (514, 33000, 1)])
def test_matches_the_definition(T, V, top, dtype):
    gen = torch.Generator().manual_seed(T + V + top)
    z = (3 * torch.randn(T, V, generator=gen)).to(dtype).cuda()
    t = torch.randint(0, V, (T,), generator=gen).cuda()
    if T > 4:
        t[::3] = torch.tensor([-100, -1, V, 2**31 + 5])[torch.arange(len(t[::3])) % 4].cuda()  # rows without a token
    _check(z, t, top)
    _check(z, t.clamp(-(2**31), 2**31 - 1).int(), top)


@pytest.mark.parametrize("top", [1, 20, 64])
@pytest.mark.parametrize("kind", ["same", "two", "up", "down", "steps", "last"])
@pytest.mark.parametrize("T,V", [(1, 200), (2, 9000), (3, 70000), (600, 5000), (530, 20000)])
def test_alternatives_of_equal_and_sorted_logits(T, V, kind, top):
    """Equal logits go by their tokens; sorted ones leave the largest to a few threads."""
    from came_amd import token_log_probs
    k = torch.arange(V, dtype=torch.float32)
    z = {"same": torch.zeros(V), "two": (k % 2), "up": k / V, "down": -k / V, "steps": torch.floor(k / 100), "last": (k >= V - 70).float()}[kind]
    z = z.expand(T, V).clone().cuda()
    t = torch.zeros(T, dtype=torch.long, device="cuda")
    for logits in (z, z.to(BF16)):
        r = token_log_probs(logits, t, top=top)
        order = _order(logits[:1], top).expand(T, top)
        assert torch.equal(r.top_tokens.cpu(), order)
        want = torch.log_softmax(logits[0].double(), -1).cpu()[order]
        assert ((r.top_log_probs.cpu().double() - want).abs() <= 1e-5).all()


@pytest.mark.parametrize("T,V", [(9, 300), (9, 40000), (600, 2000), (520, 12345)])
def test_masked_logits(T, V):
    """-inf, and the type's lowest value, in most places; rows that a mask leaves one logit or none."""
    from came_amd import token_log_probs
    gen = torch.Generator().manual_seed(V)
    for dtype in (F32, BF16):
        z = torch.randn(T, V, generator=gen)
        z[:, V // 2 :] = -INF
        z[1] = -INF
        z[1, V - 1] = 3.0
        z[2, : V // 2] = torch.finfo(dtype).min
        z[2, 5] = 0.0
        z[3, : V - 3] = -INF
        z[3, V - 3 :] = 1.0
        z[4] = torch.finfo(dtype).min
        z = z.to(dtype).cuda()
        t = torch.randint(0, V // 2, (T,), generator=gen).cuda()
        t[1], t[2], t[3] = V - 1, 5, V - 2
        (lp, elp), (H, eh), kept = orc.log_probs(z, t)
        leaf = z.requires_grad_()
        r = token_log_probs(leaf, t, top=1)
        _close(r.log_probs.detach(), lp, elp, "log_probs")
        _close(r.entropy.detach(), H, eh, "entropy")
        assert float(r.log_probs[1].detach()) == 0 and float(r.entropy[1].detach()) == 0 and int(r.top_tokens[1]) == V - 1 and int(r.top_tokens[4]) == 0
        dlp, dent = (torch.randn(T, generator=gen).cuda() for _ in range(2))
        g, = torch.autograd.grad((r.log_probs, r.entropy), leaf, (dlp, dent))
        want, bound = orc.log_probs_gradient(kept, dlp, dent, dtype)
        _close(g, want, bound, "dlogits")
        assert not g.cpu()[z.cpu() == -INF].any()
        masked = token_log_probs(z, torch.full_like(t, V // 2))  # tokens that the mask leaves out
        assert (masked.log_probs[5:] == -INF).all() and float(masked.log_probs[1].detach()) == -INF


@pytest.mark.parametrize("T,V", [(8, 100), (8, 60000), (520, 3000)])
def test_rows_that_are_not_finite(T, V):
    from came_amd import token_log_probs
    gen = torch.Generator().manual_seed(V)
    z = torch.randn(T, V, generator=gen)
    z[1] = -INF
    z[2, V // 3] = float("nan")
    z[3, V - 1] = INF
    z[4] = float("nan")
    t = torch.zeros(T, dtype=torch.long)
    t[5] = -100
    leaf = z.cuda().requires_grad_()
    r = token_log_probs(leaf, t.cuda(), top=2)
    bad = torch.zeros(T, dtype=torch.bool)
    bad[1:5] = True
    for o in (r.log_probs, r.entropy, r.top_log_probs):
        assert torch.isnan(o.detach().cpu()[bad]).all() and torch.isfinite(o.detach().cpu()[~bad]).all()
    assert r.top_tokens[1].tolist() == [0, 1] and int(r.top_tokens[2, 0]) == V // 3 and int(r.top_tokens[3, 0]) == V - 1
    assert r.top_tokens[4].tolist() == [0, 1]
    g, = torch.autograd.grad((r.log_probs, r.entropy), leaf, (torch.ones(T, device="cuda"), torch.ones(T, device="cuda")))
    assert torch.isfinite(g.cpu()[~bad]).all() and torch.isnan(g.cpu()[[1, 4]]).all()
    r = token_log_probs(leaf, torch.full((T,), -1, device="cuda"))  # no token, and no gradient of the entropy: zeros
    g, = torch.autograd.grad(r.log_probs, leaf, torch.ones(T, device="cuda"))
    assert not g.any() and not r.log_probs.any()


def test_shapes_strides_and_types_of_operands():
    from came_amd import token_log_probs
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(4, 6, 400, generator=gen).to(BF16).cuda()
    for z in (wide[..., 1:398], wide.transpose(0, 1), wide[::2, 1::2, 3:], wide[:1].expand(4, 6, 400), torch._neg_view(wide), wide[2, 3]):
        t = torch.randint(0, z.shape[-1], tuple(z.shape[:-1])[::-1], generator=gen).cuda().permute(list(range(z.dim() - 2, -1, -1)))
        a, b = (token_log_probs(x, y, top=4) for x, y in ((z, t), (z.resolve_neg().contiguous().clone(), t.contiguous())))
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and a.log_probs.shape == z.shape[:-1]
        leaf, other = z.detach().requires_grad_(), z.resolve_neg().contiguous().clone().requires_grad_()
        dy = torch.randn(tuple(t.shape)[::-1], generator=gen).cuda().permute(list(range(t.dim() - 1, -1, -1)))
        g, = torch.autograd.grad(token_log_probs(leaf, t).log_probs, leaf, dy)
        h, = torch.autograd.grad(token_log_probs(other, t).log_probs, other, dy.contiguous())
        assert torch.equal(g, h)
    none = token_log_probs(wide[:0].requires_grad_(), torch.zeros(0, 6, dtype=torch.long, device="cuda"), top=3)
    assert none.log_probs.shape == (0, 6) and none.top_tokens.shape == (0, 6, 3)
    none.log_probs.sum().backward()


def test_kept_results_keep_no_workspace():
    from came_amd import token_log_probs
    r = token_log_probs(torch.randn(3, 50000, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda"), top=5)
    assert all(o.untyped_storage().nbytes() == o.numel() * o.element_size() for o in r)


def test_gradients_against_differences():
    from came_amd import token_log_probs
    gen = torch.Generator().manual_seed(4)
    z = torch.randn(6, 300, generator=gen).cuda().requires_grad_()
    t = torch.randint(0, 300, (6,), generator=gen).cuda()
    a, b = (torch.randn(6, generator=gen).cuda() for _ in range(2))
    r = token_log_probs(z, t)
    g, = torch.autograd.grad((r.log_probs, r.entropy), z, (a, b))
    d = torch.randn(6, 300, generator=gen, dtype=torch.float64)

    def value(x):
        logp = torch.log_softmax(x, -1)
        return (logp[torch.arange(6), t.cpu()] * a.cpu().double()).sum() - ((logp.exp() * logp).sum(-1) * b.cpu().double()).sum()

    x, e = z.detach().cpu().double(), 1e-4
    diff = (value(x + e * d) - value(x - e * d)) / (2 * e)
    assert abs(diff - (g.cpu().double() * d).sum()) <= 1e-4 * (g.cpu().double() * d).norm()


def test_rows_past_2_31_elements():
    from came_amd import token_log_probs
    T, V = 70_000, 32_000
    z = torch.zeros(T, V, dtype=F16, device="cuda")
    z[-1, 31_999] = 8.0
    t = torch.full((T,), 31_999, device="cuda")
    r = token_log_probs(z.requires_grad_(), t)
    want = torch.log_softmax(z[-2:].detach().double(), -1)[:, -1]
    assert torch.allclose(r.log_probs[-2:].double(), want, atol=1e-5) and torch.equal(r.log_probs[:-1], r.log_probs[:1].expand(T - 1))
    dlp = torch.zeros(T, device="cuda")
    dlp[-1] = 1.0
    g, = torch.autograd.grad(r.log_probs, z, dlp)
    p = torch.softmax(z[-1].detach().double(), -1)
    p[31_999] -= 1
    assert not g[:-1].any() and torch.allclose(g[-1].double(), -p, atol=1e-6, rtol=2.0**-10)


def test_the_same_inputs_give_the_same_bits():
    from came_amd import token_log_probs
    gen = torch.Generator().manual_seed(5)
    for T, V in ((2, 100_000), (700, 20_000)):
        z = torch.randn(T, V, generator=gen).cuda()
        t = torch.randint(0, V, (T,), generator=gen).cuda()
        first = token_log_probs(z, t, top=20)
        for _ in range(3):
            torch.empty(1 << 24, device="cuda").fill_(float("nan"))
            assert all(torch.equal(a, b) for a, b in zip(first, token_log_probs(z, t, top=20)))


def test_on_another_stream_and_in_a_graph():
    from came_amd import token_log_probs
    gen = torch.Generator().manual_seed(6)
    for T, V in ((3, 40_000), (70, 500)):
        z = torch.randn(T, V, generator=gen).cuda().requires_grad_()
        t = torch.randint(0, V, (T,), generator=gen).cuda()
        dlp, dent = (torch.randn(T, generator=gen).cuda() for _ in range(2))

        def both():
            r = token_log_probs(z, t, top=6)
            return [o.detach() for o in r] + list(torch.autograd.grad((r.log_probs, r.entropy), z, (dlp, dent)))

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
        for _ in range(4):
            with torch.no_grad():
                z.copy_(torch.randn(T, V, generator=gen).cuda())
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(both(), held))


def test_gradients_of_gradients_and_refusals():
    from came_amd import token_log_probs
    z, t = torch.randn(3, 8, device="cuda", requires_grad=True), torch.zeros(3, dtype=torch.long, device="cuda")
    g, = torch.autograd.grad(token_log_probs(z, t).log_probs.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="token_log_probs is differentiable once"):
        g.sum().backward()
    for top in (-1, 9, 65):
        with pytest.raises(ValueError, match="top"):
            token_log_probs(z, t, top=top)
    for bad in ((z, t[:2]), (z, t[None]), (z[:, :0], t), (torch.zeros((), device="cuda"), t),
                (torch.zeros(1, (1 << 20) + 1, device="cuda"), t[:1])):
        with pytest.raises(ValueError):
            token_log_probs(*bad)
    for bad, match in (((z.double(), t), "dtype"), ((z, t.float()), "int64 or int32"), ((z, t.cpu()), "GPU")):
        with pytest.raises(RuntimeError, match=match):
            token_log_probs(*bad)
    r = token_log_probs(z, t)
    with torch.no_grad():
        z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.entropy.sum().backward()
