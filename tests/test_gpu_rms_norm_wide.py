"""came_amd.rms_norm's weight gradient where a row has more columns than one launch's join has at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim", [(2, (1 << 25) + 70), (1, (1 << 27) + 33)])
def test_gradients_of_the_widest_rows(rows, dim):
    """Rows of ones.  A thread's and a wavefront's sum of them is exact, the sum of the 16 wavefronts' takes 15 roundings and the
    width one; r has half of those and 4 of its own, 12 in all, and dw = r sum dy one a row and one in the join: 15 of the terms'
    magnitudes, and the result's own half step."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from came_amd import rms_norm
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.ones(rows, dim, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(dim, dtype=torch.bfloat16, device="cuda").requires_grad_()
    dy = torch.randn(rows, dim, dtype=torch.bfloat16, device="cuda", generator=gen)
    y = rms_norm(x, w)
    assert (y == 1).all()
    g, = torch.autograd.grad(y, w, dy)
    want = dy.double().sum(0) / (1 + 1e-6) ** 0.5
    off = 15 * 2.0**-24 * dy.double().abs().sum(0)
    bound = off * (1 + 2.0**-7) + 2.0**-8 * want.abs() + 2.0**-134
    err = (g.double() - want).abs()
    assert (err <= bound).all(), float((err - bound).max())
