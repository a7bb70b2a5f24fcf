"""The global gradient norm and the clip by it against sums in 64 bits: types, sizes about chunk edges, more tensors than
a launch's table, empty, strided and unaligned ones, norms below and above the bound, infinities and NaN, repeatability."""
import math

import pytest
import torch

from oracle import adamw_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# fp32 sums of at most 8 squares in a row a lane, 64 in all before fp64: (8 + 3) roundings of positive terms at most,
# the square root halves that, and one rounding of the result and its square root
TOL = 8 * 2.0**-24


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _grads(sizes, dtypes, seed, offset=0, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        buf = torch.zeros(n + offset, dtype=dt, device="cuda")
        buf[offset:] = (torch.randn(n, generator=gen) * scale).to(dt).cuda()
        out.append(buf[offset:])
    return out


def _params(grads):
    ps = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("sizes", [[1], [7, 8, 9], [16383, 16384, 16385], [0, 5, 0], [100003, 1, 40000], [37] * 500,
                                   [3000000, 17]])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
def test_norm_and_clip(sizes, dtypes, offset):
    import came_amd
    grads = _grads(sizes, dtypes, len(sizes), offset)
    want = orc.norm64([g.cpu() for g in grads])
    norm = came_amd.grad_norm(grads)
    assert norm.shape == () and norm.dtype == F32
    assert abs(float(norm) - want) <= TOL * want
    before = [g.clone() for g in grads]
    ps = _params(grads)
    assert torch.equal(came_amd.clip_grad_norm_(ps, 2 * want), norm)  # the norm is below: nothing changes
    assert all(torch.equal(p.grad, b) for p, b in zip(ps, before))
    assert torch.equal(came_amd.clip_grad_norm_(ps, 0.25 * want), norm)
    factor = 0.25 * want / (float(norm) + 1e-6)
    for p, b in zip(ps, before):
        x = b.double() * factor
        unit = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}[b.dtype]
        tol = x.abs() * (unit + 8 * 2.0**-24) + (2.0**-25 if b.dtype == F16 else 0)
        assert ((p.grad.double() - x).abs() <= tol).all()


def test_parameters_without_gradients_and_strided_ones():
    import came_amd
    a = torch.nn.Parameter(torch.zeros(40, 50, device="cuda"))
    a.grad = torch.randn(50, 40, device="cuda").t()
    b = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    kept = a.grad.clone()
    want = orc.norm64([kept.cpu()])
    norm = came_amd.clip_grad_norm_([b, a], 1.0)
    assert abs(float(norm) - want) <= TOL * want
    assert ((a.grad.double() - kept.double() / (want + 1e-6)).abs() <= 1e-6 * kept.double().abs()).all()
    assert b.grad is None
    assert float(came_amd.clip_grad_norm_([b], 1.0)) == 0.0
    assert abs(float(came_amd.clip_grad_norm_(a, 0.5)) - 1.0) < 1e-5  # a single tensor
    assert float(came_amd.grad_norm([torch.zeros(0, device="cuda")])) == 0.0


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_norms_that_are_not_finite(bad):
    import came_amd
    grads = _grads([1000, 20000], (F32,), 0)
    grads[1][777] = bad
    ps = _params([g.clone() for g in grads])
    with pytest.raises(RuntimeError, match="not finite"):
        came_amd.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert torch.equal(ps[0].grad, grads[0])
    norm = float(came_amd.clip_grad_norm_(ps, 1.0))
    assert math.isinf(norm) if math.isinf(bad) else math.isnan(norm)
    if math.isinf(bad):
        assert (ps[0].grad == 0).all() and torch.isnan(ps[1].grad[777])
    else:
        assert torch.isnan(ps[0].grad).all()


def test_the_same_gradients_give_the_same_bits():
    import came_amd
    grads = _grads([1000003, 5, 77777], (F32, BF16), 3)
    norms = {float(came_amd.grad_norm(grads)) for _ in range(20)}
    assert len(norms) == 1


def test_in_a_graph():
    """The tensor list travels in the kernels' arguments: a captured clip replays on new values in the same buffers."""
    import came_amd
    grads = _grads([70001, 300], (F32,), 1)
    ps = _params(grads)
    came_amd.clip_grad_norm_(ps, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = came_amd.clip_grad_norm_(ps, 0.01)
    for k in range(3):
        new = _grads([70001, 300], (F32,), 10 + k)
        for g, x in zip(grads, new):
            g.copy_(x)
        eager = _params([x.clone() for x in new])
        graph.replay()
        want = came_amd.clip_grad_norm_(eager, 0.01)
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        assert all(torch.equal(g, e.grad) for g, e in zip(grads, eager))
