"""Infinities through the gated feed-forward block: operands that the kernels take apart (large fp32 products into three
parts, the down projection's input of few 16-bit tokens into two) give infinity where the formulas do, whatever the size of
the other operand's values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("T", [3, 140, 2100])
def test_fp32_infinity_times_values_of_any_size(T):
    """All operands positive: a token's infinity makes its row of y infinite, and dy's its row of x's gradient and every weight
    gradient, with weights of 1e3 to 1e7, whose rests beyond 8 bits are large and of either sign."""
    from came_amd import gated_ffn
    D, F, E = 520, 1500, 600
    gen = torch.Generator().manual_seed(21)

    def values(*s):
        return torch.pow(10.0, 3 + 4 * torch.rand(*s, generator=gen)).cuda()

    wg, wu, wd = values(F, D), values(F, D), values(E, F)
    x, dy = torch.rand(T, D, generator=gen).cuda(), torch.rand(T, E, generator=gen).cuda()
    bad = x.clone()
    bad[1, 519] = float("inf")
    with torch.no_grad():
        y = gated_ffn(bad, wg, wu, wd)
    rows = torch.ones(T, dtype=torch.bool, device="cuda")
    rows[1] = False
    assert (y[1] == float("inf")).all() and torch.isfinite(y[rows]).all()
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    dy[1, 599] = float("inf")
    gated_ffn(*leaves).backward(dy)
    dx, dwg, dwu, dwd = (t.grad for t in leaves)
    assert (dx[1] == float("inf")).all() and torch.isfinite(dx[rows]).all()
    assert (dwg == float("inf")).all() and (dwu == float("inf")).all()
    assert (dwd[599] == float("inf")).all() and torch.isfinite(dwd[:599]).all()


@pytest.mark.parametrize("T", [3, 2100])
def test_fp32_infinity_times_infinity(T):
    from came_amd import gated_ffn
    ops = [torch.rand(*s, device="cuda") + 0.1 for s in ((T, 520), (1500, 520), (1500, 520), (600, 1500))]
    ops[0][2, 5] = ops[1][:, 5] = ops[2][:, 5] = float("inf")
    with torch.no_grad():
        y = gated_ffn(*ops)
    assert (y == float("inf")).all()  # every other row: a positive number times infinity


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T", [1, 16, 17])
def test_an_infinite_down_weight(T, dtype):
    """An infinity in a row of w_down is an infinity, of h's sign, in that column of y, and in no other."""
    from came_amd import gated_ffn
    gen = torch.Generator().manual_seed(22)
    x, wg, wu, wd = (torch.rand(*s, generator=gen).to(dtype).cuda() for s in ((T, 72), (100, 72), (100, 72), (40, 100)))
    wu[7] = -wu[7]  # h of column 7 is negative
    with torch.no_grad():
        want = gated_ffn(x, wg, wu, wd)
        bad = wd.clone()
        bad[3, 7], bad[5, 99] = float("inf"), float("inf")
        y = gated_ffn(x, wg, wu, bad)
    assert (y[:, 3] == -float("inf")).all() and (y[:, 5] == float("inf")).all()
    rest = [e for e in range(40) if e not in (3, 5)]
    assert torch.equal(y[:, rest], want[:, rest])


def test_large_fp32_products_of_small_values():
    """Rows of 1e-14 to 1e-8, gradients of 1e-6: a value's third part is 2^-16 of it, and all parts stay normal numbers."""
    from oracle import ffn_oracle as orc
    from came_amd import gated_ffn
    gen = torch.Generator().manual_seed(23)
    T, D, F, E = 2100, 520, 1500, 600
    x = (torch.randn(T, D, generator=gen) * torch.pow(10.0, torch.linspace(-14, -8, T))[:, None]).cuda()
    w = [(torch.randn(*s, generator=gen) * s[1] ** -0.5).cuda() for s in ((F, D), (F, D), (E, F))]
    dy = (torch.randn(T, E, generator=gen) * 1e-6).cuda()
    want, bound, kept = orc.forward(x, *w, "silu", F32)
    leaves = [t.clone().requires_grad_() for t in (x, *w)]
    y = gated_ffn(*leaves)
    y.backward(dy)
    grads = orc.backward(kept, dy)
    assert ((y.detach().cpu().double() - want).abs() <= bound).all()
    for leaf, name in zip(leaves, ("x", "w_gate", "w_up", "w_down")):
        g, b = grads[name]
        assert ((leaf.grad.cpu().double() - g).abs() <= b).all(), name
