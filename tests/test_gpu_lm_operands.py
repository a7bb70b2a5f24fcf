"""Operands of the embedding, the norm and the token log probabilities that calls may have and programs seldom do."""
import pytest
import torch

from oracle import lm_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_tokens_that_are_negative_views(dtype):
    """Tensors whose values are the negatives of what their memory holds."""
    from came_amd import embedding, token_log_probs
    gen = torch.Generator().manual_seed(0)
    t = torch.randint(0, 40, (5, 9), generator=gen).to(dtype).cuda()
    held = -t
    for view, want in ((torch._neg_view(held), t), (torch._neg_view(held)[::2, 1:], t[::2, 1:])):
        assert view.is_neg() and torch.equal(view, want)
        table = torch.randn(40, 12, generator=gen).cuda().requires_grad_()
        a, b = embedding(view, table), embedding(want, table)
        dy = torch.randn(a.shape, generator=gen).cuda()
        assert torch.equal(a, b)
        assert torch.equal(torch.autograd.grad(a, table, dy)[0], torch.autograd.grad(b, table, dy)[0])
        z = torch.randn(*want.shape, 40, generator=gen).cuda().requires_grad_()
        a, b = token_log_probs(z, view, top=2), token_log_probs(z, want, top=2)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        dlp = torch.randn(want.shape, generator=gen).cuda()
        assert torch.equal(torch.autograd.grad(a.log_probs, z, dlp)[0], torch.autograd.grad(b.log_probs, z, dlp)[0])


@pytest.mark.parametrize("D", [64, 3000, 20000])
@pytest.mark.parametrize("size", [3e-20, 1e-18, 1.0, 1e17])
def test_norm_gradients_of_small_and_large_rows_without_eps(D, size):
    """1/sqrt(mean(h^2)) squared is no float32 for rows of 3e-20, but nothing that the gradient is made of is that large.  Squares
    of 9e-40 are subnormal: a term's rounding is 2^-150, D of them in the mean 2^-150 / 9e-40 = 8e-7 of it, 13 U.  With the oracle's
    (CHAIN / 2 + 4) U of r and (CHAIN + 1) U of the other sum, which r enters twice: below 300 U, of the terms' magnitudes.  A sum of
    squares past float32 (20000 of 1e34 and up to 4e34: 4.7e38, where 3.4e38 is the largest) makes r zero, as is documented, and the
    gradients with it."""
    from came_amd import rms_norm
    gen = torch.Generator().manual_seed(D)
    x = (size * (1 + torch.rand(6, D, generator=gen)) * (2.0 * torch.randint(0, 2, (6, D), generator=gen) - 1)).cuda().requires_grad_()
    w = (1 + 0.2 * torch.randn(D, generator=gen)).cuda().requires_grad_()
    dy = torch.randn(6, D, generator=gen).cuda()
    dx, dw = torch.autograd.grad(rms_norm(x, w, eps=0.0), (x, w), dy)
    h, g, v = x.detach().cpu().double(), dy.cpu().double(), w.detach().cpu().double()
    if (h.square().sum(-1) > 1.01 * torch.finfo(torch.float32).max).all():
        assert not dx.any() and not dw.any()
        return
    r = 1 / h.square().mean(-1, keepdim=True).sqrt()
    gw = g * v
    want = r * (gw - h * (r * r * (gw * h).mean(-1, keepdim=True)))
    size_of = r * (gw.abs() + h.abs() * r * r * (gw * h).abs().mean(-1, keepdim=True))
    assert ((dx.cpu().double() - want).abs() <= 300 * orc.U * size_of).all()
    terms = g * h * r
    assert ((dw.cpu().double() - terms.sum(0)).abs() <= 300 * orc.U * terms.abs().sum(0)).all()


def test_an_eps_that_float32_does_not_hold():
    """One that would be infinite there is refused; one that would be 0 is kept above it, and so is a row of zeros finite."""
    from came_amd import rms_norm, rms_norm_int8
    x, w = torch.zeros(3, 40, device="cuda"), torch.ones(40, device="cuda")
    x[1] = 1.0
    for op in (rms_norm, rms_norm_int8):
        for eps in (1e39, 1e300):
            with pytest.raises(ValueError, match="eps"):
                op(x, w, eps=eps)
    leaf = x.clone().requires_grad_()
    y = rms_norm(leaf, w, eps=1e-60)
    assert not y[0].any() and (y[1] == 1).all()
    assert torch.isfinite(torch.autograd.grad(y, leaf, torch.full_like(y, 1e-3))[0]).all()


def test_a_scale_that_float32_does_not_hold():
    """One that would be infinite or 0 there is refused."""
    from came_amd import embedding
    x, t = torch.zeros(3, 40, device="cuda"), torch.tensor([1, 7], device="cuda")
    x[1] = 1.0
    for scale in (1e39, -1e39, 1e-60):
        with pytest.raises(ValueError, match="scale"):
            embedding(t, x, scale=scale)
    assert not embedding(t, x, scale=0.0).any() and torch.isnan(embedding(t, x, scale=float("nan"))[0]).all()
    assert (embedding(t, x, scale=1e38)[0] == 1e38).all() and (embedding(t, x, scale=1e-40)[0] > 0).all()


def test_batched_gradients_and_function_transforms_raise():
    """Tensors that stand for several have no memory that a kernel could read."""
    from came_amd import embedding, int8_linear, quantize_rows, rms_norm, rms_norm_int8, token_log_probs
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(16, device="cuda")
    t = torch.zeros(4, dtype=torch.long, device="cuda")
    calls = [lambda x: embedding(t, x), lambda x: rms_norm(x, w), lambda x: token_log_probs(x, t).log_probs]
    for fn in calls:
        leaf = x.clone().requires_grad_()
        y = fn(leaf)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaf, torch.randn(3, *y.shape, device="cuda"), is_grads_batched=True)
        torch.cuda.synchronize()
        for transform in (torch.func.vmap, torch.func.jacfwd, torch.func.jacrev):
            with pytest.raises(RuntimeError):
                transform(fn)(x[None] if transform is torch.func.vmap else x)
    q, s = quantize_rows(x)
    for fn in (lambda x: rms_norm_int8(x, w)[1], lambda x: quantize_rows(x)[1], lambda x: int8_linear(q, s, q, x[:, 0])):
        with pytest.raises(RuntimeError):
            torch.func.vmap(fn)(x[None])
    torch.cuda.synchronize()
