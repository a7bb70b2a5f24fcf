"""The gated feed-forward block on the GPU against the formulas in 64 bits, within bounds that follow its roundings: rows
from none to several tiles, widths about vector, fragment and tile edges and odd ones, types, activations, operands with
row strides of their own and copied ones, single gradients, products past 2^31 elements, other streams, graphs."""
import pytest
import torch

from oracle import ffn_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("x", "w_gate", "w_up", "w_down")


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _operands(T, D, F, E, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    def rand(*s, scale):
        return (torch.randn(*s, generator=gen) * scale).to(dtype).cuda()
    ops = [rand(T, D, scale=1.0), rand(F, D, scale=1.5 * D**-0.5), rand(F, D, scale=D**-0.5), rand(E, F, scale=F**-0.5)]
    return ops, rand(T, E, scale=1.0)


def _check(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}, "
                           f"{got[bad][0]:.6g} for {want[bad][0]:.6g} +- {bound[bad][0]:.3g}")


def _check_all(ops, dy, act, needs=(True,) * 4, what=""):
    """Forward alone, forward of a training step, and every gradient that is wanted."""
    from came_amd import gated_ffn
    dtype = ops[0].dtype
    want, bound, kept = orc.forward(*ops, act, dtype)
    with torch.no_grad():
        _check(gated_ffn(*ops, activation=act), want, bound, f"{what} y without gradients")
    leaves = [t.detach().requires_grad_(n) for t, n in zip(ops, needs)]
    y = gated_ffn(*leaves, activation=act)
    _check(y, want, bound, f"{what} y")
    y.backward(dy)
    grads = orc.backward(kept, dy)
    for name, leaf, n in zip(NAMES, leaves, needs):
        assert (leaf.grad is not None) == n
        if n:
            assert leaf.grad.dtype == dtype
            _check(leaf.grad, *grads[name], f"{what} gradient of {name}")


SHAPES = [(1, 1, 1, 1), (1, 8, 8, 8), (1, 64, 64, 64), (1, 300, 517, 300), (2, 16, 1, 3), (3, 7, 5, 9), (5, 1040, 24, 72),
          (16, 128, 256, 128), (17, 33, 65, 31), (33, 96, 1001, 96), (64, 64, 64, 64), (65, 511, 130, 512), (127, 129, 191, 130),
          (128, 128, 128, 128), (129, 256, 320, 64), (200, 40, 41, 42), (257, 100, 333, 77), (300, 512, 1365, 512),
          (1000, 96, 40, 1111), (513, 264, 520, 264)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_matches_the_formulas(shape, dtype):
    ops, dy = _operands(*shape, dtype, seed=sum(shape))
    _check_all(ops, dy, "silu")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_activations_over_their_range(act, dtype):
    """Gate values from far below to far above zero."""
    ops, dy = _operands(100, 64, 136, 64, dtype, seed=5)
    ops[1] = (ops[1].float() * torch.linspace(0.1, 12, 136, device="cuda")[:, None]).to(dtype)
    _check_all(ops, dy, act)


@pytest.mark.parametrize("shape", [(1030, 512, 1376, 512), (700, 1000, 600, 1100), (2050, 128, 300, 520)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_several_tiles(shape, dtype):
    ops, dy = _operands(*shape, dtype, seed=9)
    _check_all(ops, dy, "silu")


def test_large_fp32_products_keep_fp32_accuracy():
    """fp32 products of many tiles take their operands apart: rows of magnitudes from 1e-8 to 1e8 each keep float32's accuracy
    against their own, and a row's infinity, NaN or near-largest value stays in that row."""
    from came_amd import gated_ffn
    ops, dy = _operands(2100, 520, 1500, 600, F32, seed=12)
    ops[0] = ops[0] * torch.pow(10.0, torch.linspace(-8, 8, 2100, device="cuda"))[:, None]
    dy = dy * torch.pow(10.0, torch.linspace(8, -8, 2100, device="cuda"))[:, None]
    _check_all(ops, dy, "gelu_tanh")
    ops, dy = _operands(2100, 520, 1500, 600, F32, seed=13)
    with torch.no_grad():
        want = gated_ffn(*ops)
        bad = ops[0].clone()
        bad[5, 519], bad[700, 3], bad[2099, 0] = float("inf"), float("nan"), 3.4e38
        got = gated_ffn(bad, *ops[1:])
    rows = torch.ones(2100, dtype=torch.bool, device="cuda")
    rows[[5, 700, 2099]] = False
    assert torch.equal(got[rows], want[rows]) and not torch.isfinite(got[[5, 700]]).any()


@pytest.mark.parametrize("T", [3, 140, 2100])
def test_fp32_values_next_to_the_largest_and_infinity(T):
    """A row with a value that would round to infinity in a shorter type keeps float32's accuracy, and infinity times positive
    weights is infinity, in every kernel."""
    from came_amd import gated_ffn
    ops, _ = _operands(T, 520, 1500, 600, F32, seed=14)
    ops = [t.abs() for t in ops]
    ops[1][:, 0] *= 2.0**-100
    ops[2][:, 0] *= 2.0**-100
    ops[0][T - 1, 0] = torch.finfo(F32).max
    with torch.no_grad():
        want, bound, _ = orc.forward(*ops, "silu", F32)
        _check(gated_ffn(*ops), want, bound, "next to the largest")
        rows = ops[0].clone()
        rows[1, 519] = float("inf")
        got = gated_ffn(rows, *ops[1:])
    assert torch.isinf(got[1]).all() and torch.isfinite(got[[0, T - 1]]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 9, 140])
def test_operands_where_they_lie(T, dtype):
    """Row strides: x a slice of wider rows that starts unaligned, gate and up halves of one matrix and interleaved rows of
    one; copies: a transposed weight, an expanded x; leading dimensions."""
    from came_amd import gated_ffn
    D, F, E = 72, 100, 40
    (x, wg, wu, wd), dy = _operands(T, D, F, E, dtype, seed=2)
    wide = torch.randn(T, D + 9, device="cuda").to(dtype)
    wide[:, 3 : 3 + D] = x
    both = torch.cat([wg, wu])
    _check_all([wide[:, 3 : 3 + D], both[:F], both[F:], wd], dy, "silu", what="halves")
    turns = torch.stack([wg, wu], 1)
    _check_all([x, turns[:, 0], turns[:, 1], wd], dy, "silu", what="interleaved")
    _check_all([x, wg.t().contiguous().t(), wu, wd.t().contiguous().t()], dy, "silu", what="transposed")
    _check_all([x[:1].expand(T, D), wg, wu, wd], dy, "silu", what="expanded")
    with torch.no_grad():
        y = gated_ffn(x, wg, wu, wd)
        assert torch.equal(gated_ffn(x.view(1, T, 1, D), wg, wu, wd), y.view(1, T, 1, E))
        assert torch.equal(gated_ffn(x[0], wg, wu, wd), gated_ffn(x[:1], wg, wu, wd)[0])
        assert gated_ffn(x[:0], wg, wu, wd).shape == (0, E)


def test_a_gradient_that_is_not_contiguous_and_no_tokens():
    from came_amd import gated_ffn
    ops, dy = _operands(20, 24, 56, 24, F32)
    leaves = [t.clone().requires_grad_() for t in ops]
    gated_ffn(*leaves).backward(dy.t().contiguous().t())
    other = [t.clone().requires_grad_() for t in ops]
    gated_ffn(*other).backward(dy)
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(leaves, other))
    empty = [ops[0][:0].clone().requires_grad_(), *(t.clone().requires_grad_() for t in ops[1:])]
    gated_ffn(*empty).sum().backward()
    assert all((t.grad == 0).all() for t in empty) and empty[0].grad.shape == (0, 24)


@pytest.mark.parametrize("needs", [(True, False, False, False), (False, True, False, False), (False, False, True, False),
                                   (False, False, False, True), (False, True, True, True), (True, False, True, False)])
def test_single_gradients(needs):
    ops, dy = _operands(70, 80, 96, 112, BF16, seed=3)
    _check_all(ops, dy, "gelu", needs)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradients_against_differences(act):
    """Along a random direction, the change of <dy, y> in 64 bits against <gradient, direction>: a central difference of
    step e is off by e^2 of third derivatives (1e-8 of the value here), float32 gradients by about 1e-6."""
    from came_amd import gated_ffn
    ops, dy = _operands(37, 24, 40, 24, F32, seed=4)
    leaves = [t.clone().requires_grad_() for t in ops]
    gated_ffn(*leaves, activation=act).backward(dy)
    gen = torch.Generator().manual_seed(1)
    e = 1e-4
    for k in range(4):
        d = torch.randn(ops[k].shape, generator=gen, dtype=torch.float64) * float(ops[k].float().std())
        moved = [[t.cpu().double() + (s * e * d if i == k else 0) for i, t in enumerate(ops)] for s in (1, -1)]
        diff = sum(s * (orc.forward(*m, act) * dy.cpu().double()).sum() for s, m in zip((1, -1), moved)) / (2 * e)
        along = (leaves[k].grad.cpu().double() * d).sum()
        scale = (leaves[k].grad.cpu().double() * d).norm()
        assert abs(diff - along) <= 1e-4 * scale, (NAMES[k], float(diff), float(along), float(scale))


def test_rows_do_not_mix():
    """An infinity or NaN in one row of x reaches that row of y and of x's gradient, and no other."""
    from came_amd import gated_ffn
    ops, dy = _operands(150, 64, 72, 64, BF16, seed=6)
    clean = [t.clone().requires_grad_() for t in ops]
    y0 = gated_ffn(*clean)
    y0.backward(dy)
    bad = [t.clone() for t in ops]
    bad[0][140, 63] = float("nan")
    bad[0][3, 0] = float("inf")
    bad[0].requires_grad_()
    y1 = gated_ffn(*bad)
    y1.backward(dy)
    rows = torch.ones(150, dtype=torch.bool, device="cuda")
    rows[[3, 140]] = False
    assert torch.equal(y0[rows], y1[rows]) and not torch.isfinite(y1[~rows]).all(1).any()
    assert torch.equal(clean[0].grad[rows], bad[0].grad[rows])


@pytest.mark.parametrize("T", [1, 24, 300])
def test_the_same_inputs_give_the_same_bits(T):
    from came_amd import gated_ffn
    ops, dy = _operands(T, 520, 1111, 520, BF16, seed=8)
    seen = []
    for _ in range(3):
        leaves = [t.clone().requires_grad_() for t in ops]
        y = gated_ffn(*leaves)
        y.backward(dy)
        seen.append([y.detach(), *(t.grad for t in leaves)])
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1030, 512, 1376, 512), (2048, 1024, 2752, 1024)], ids=lambda s: "x".join(map(str, s)))
def test_many_steps_give_the_same_bits(shape, dtype):
    """Wavefronts that run apart over many steps of a tile: results and gradients repeat bit for bit."""
    from came_amd import gated_ffn
    ops, dy = _operands(*shape, dtype, seed=10)
    first = None
    for _ in range(12):
        leaves = [t.clone().requires_grad_() for t in ops]
        y = gated_ffn(*leaves)
        y.backward(dy)
        got = [y.detach(), *(t.grad for t in leaves)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_hidden_values_past_2_31():
    """More than 2^31 hidden values: the last tokens' rows and gradients (all others are zero)."""
    from came_amd import gated_ffn
    T, D, F, E, tail = 131072 + 37, 8, 16392, 8, 60
    (xt, wg, wu, wd), dyt = _operands(tail, D, F, E, BF16, seed=7)
    x, dy = torch.zeros(T, D, dtype=BF16, device="cuda"), torch.zeros(T, E, dtype=BF16, device="cuda")
    x[-tail:], dy[-tail:] = xt, dyt
    want, bound, kept = orc.forward(xt, wg, wu, wd, "silu", BF16)
    grads = orc.backward(kept, dyt)
    with torch.no_grad():
        _check(gated_ffn(x, wg, wu, wd)[-tail:], want, bound, "y without gradients")
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*leaves)
    _check(y[-tail:], want, bound, "y")
    assert (y[:-tail] == 0).all()
    y.backward(dy)
    _check(x.grad[-tail:], *grads["x"], "gradient of x")
    assert (x.grad[:-tail] == 0).all()
    for name, leaf in zip(NAMES[1:], leaves[1:]):
        _check(leaf.grad, *grads[name], f"gradient of {name}")


def test_on_another_stream_and_in_a_graph():
    from came_amd import gated_ffn
    ops, dy = _operands(130, 128, 200, 128, BF16, seed=1)
    with torch.no_grad():
        want = gated_ffn(*ops)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = gated_ffn(ops[0] * 1, *ops[1:])
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, want)
        graph = torch.cuda.CUDAGraph()
        x = ops[0].clone()
        one = x[:1]
        gated_ffn(one, *ops[1:])
        with torch.cuda.graph(graph):
            y = gated_ffn(x, *ops[1:])
            y1 = gated_ffn(one, *ops[1:])
        for k in range(3):
            x.copy_(torch.randn(x.shape, device="cuda"))
            graph.replay()
            assert torch.equal(y, gated_ffn(x, *ops[1:])) and torch.equal(y1, gated_ffn(x[:1], *ops[1:]))


def test_refusals_on_the_gpu():
    from came_amd import gated_ffn
    (x, wg, wu, wd), _ = _operands(4, 8, 16, 8, BF16)
    with pytest.raises(RuntimeError, match="x is torch.bfloat16"):
        gated_ffn(x, wg.float(), wu, wd)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        gated_ffn(x.double(), wg, wu, wd)
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(x, wg, wu, wd, activation="relu")
    for bad in ((x[:, :7], wg, wu, wd), (x, wg, wu[:8], wd), (x, wg, wu, wd[:, :8]), (x, wg[:0], wu[:0], wd[:, :0]),
                (x, wg[0], wu[0], wd)):
        with pytest.raises(ValueError, match="gated_ffn"):
            gated_ffn(*bad)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*leaves)
    dx, = torch.autograd.grad(y.float().sum(), leaves[:1], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.float().sum().backward()
