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
