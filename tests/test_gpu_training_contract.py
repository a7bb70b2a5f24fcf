"""What programs count on around AdamW, the clip and the gated feed-forward block beside their formulas."""
import copy

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _classes():
    import came_amd
    return came_amd.AdamW, came_amd.AdamW8bit


class Named(torch.Tensor):
    """A subclass without dispatch of its own: its values are its storage's."""


@pytest.mark.parametrize("strided", [False, True])
def test_gradients_of_a_simple_subclass(strided):
    import came_amd
    g = torch.randn(40, 50, device="cuda")
    g = g.t() if strided else g
    want = float(g.double().norm())
    p = torch.nn.Parameter(torch.zeros(g.shape, device="cuda"))
    p.grad = g.clone(memory_format=torch.preserve_format).as_subclass(Named)
    assert abs(float(came_amd.grad_norm([p.grad])) / want - 1) < 1e-6
    assert abs(float(came_amd.clip_grad_norm_([p], 1.0)) / want - 1) < 1e-6
    assert abs(float(p.grad.as_subclass(torch.Tensor).double().norm()) - 1) < 1e-5
    q = torch.nn.Parameter(torch.zeros(g.shape, device="cuda"))
    q.grad = p.grad.as_subclass(torch.Tensor).clone()
    a, b = came_amd.AdamW([p], max_grad_norm=0.5), came_amd.AdamW([q], max_grad_norm=0.5)
    a.step()
    b.step()
    assert a.state[p]["step"] == 1 and torch.equal(p, q) and torch.equal(a.last_grad_norm, b.last_grad_norm)


@pytest.mark.parametrize("cls", range(2))
@pytest.mark.parametrize("transposed", [False, True])
def test_a_step_between_forward_and_backward_is_seen(cls, transposed):
    """The block's backward pass uses the weights of the forward one: where a step has changed them it raises."""
    import came_amd
    w = [torch.randn(*s, device="cuda") * 0.1 for s in ((72, 64), (72, 64), (64, 72))]
    w = [torch.nn.Parameter(t.t().contiguous().t() if transposed else t) for t in w]
    opt = _classes()[cls](w)
    y = came_amd.gated_ffn(torch.randn(20, 64, device="cuda"), *w)
    y.backward(torch.ones_like(y), retain_graph=True)
    before = [p._version for p in w]
    opt.step()
    assert all(p._version > b for p, b in zip(w, before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))


@pytest.mark.parametrize("transposed", [False, True])
def test_a_clip_advances_the_gradients_versions(transposed):
    import came_amd
    p = torch.nn.Parameter(torch.zeros(30, 20, device="cuda"))
    p.grad = torch.randn(20, 30, device="cuda").t() if transposed else torch.randn(30, 20, device="cuda")
    before = p.grad._version
    came_amd.grad_norm([p.grad])
    assert p.grad._version == before
    came_amd.clip_grad_norm_([p], 0.5)
    assert p.grad._version > before


def test_inference_tensors_are_stepped_and_clipped():
    """They have no version; a step and a clip write them as others."""
    import came_amd
    with torch.inference_mode():
        p = torch.nn.Parameter(torch.ones(100, device="cuda"), requires_grad=False)
        p.grad = torch.ones(100, device="cuda")
    assert abs(float(came_amd.clip_grad_norm_([p], 1.0)) - 10) < 1e-4
    opt = came_amd.AdamW([p], lr=0.1, weight_decay=0.0)
    opt.step()
    assert (p - 0.9).abs().max() < 1e-4


@pytest.mark.parametrize("dual", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_raise(dual, grad):
    """There are none: without an error they would read as zero."""
    import came_amd
    ops = [torch.randn(*s, device="cuda") for s in ((5, 16), (24, 16), (24, 16), (16, 24))]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        ops[dual] = forward_ad.make_dual(ops[dual], torch.ones_like(ops[dual]))
        with pytest.raises(RuntimeError, match="forward-mode|forward mode|forward AD|jvp"):
            came_amd.gated_ffn(*ops)


@pytest.mark.parametrize("transform", ["jvp", "vmap", "grad", "jacfwd"])
def test_function_transforms_raise(transform):
    import came_amd
    ops = [torch.randn(*s, device="cuda") for s in ((5, 16), (24, 16), (24, 16), (16, 24))]

    def fn(x):
        y = came_amd.gated_ffn(x, *ops[1:])
        return y.sum() if transform == "grad" else y

    func = torch.func
    call = dict(jvp=lambda: func.jvp(fn, (ops[0],), (torch.ones_like(ops[0]),)), vmap=lambda: func.vmap(fn)(ops[0][None]),
                grad=lambda: func.grad(fn)(ops[0]), jacfwd=lambda: func.jacfwd(fn)(ops[0]))[transform]
    with pytest.raises(RuntimeError):
        call()


@pytest.mark.parametrize("grad", [False, True])
def test_traces_raise(grad):
    """A trace would hold the result's allocation and not what fills it."""
    import came_amd
    ops = [torch.randn(*s, device="cuda") for s in ((5, 16), (24, 16), (24, 16), (16, 24))]
    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="gated_ffn.*trace"):
        torch.jit.trace(lambda x: came_amd.gated_ffn(x, *ops[1:]), (ops[0],), check_trace=False)


@pytest.mark.parametrize("cls", range(2))
@pytest.mark.parametrize("transposed", [False, True])
def test_a_refused_step_is_not_counted(cls, transposed):
    p = torch.randn(30, 20, device="cuda")
    p = torch.nn.Parameter(p.t() if transposed else p)
    p.grad = torch.randn(p.shape, device="cuda")
    before = p.detach().clone()
    opt = _classes()[cls]([p], lr=1e-2)
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(RuntimeError, match="lr"):
        opt.step()
    assert torch.equal(p, before) and opt.state[p].get("step", 0) == 0
    opt.param_groups[0]["lr"] = 1e-2
    opt.step()
    assert opt.state[p]["step"] == 1 and not torch.equal(p, before)


def test_gradients_that_are_negative_views():
    import came_amd
    ops = [torch.randn(*s, device="cuda") for s in ((5, 16), (24, 16), (24, 16), (16, 24))]
    dy = torch.randn(5, 16, device="cuda")
    a, b = ([t.clone().requires_grad_() for t in ops] for _ in range(2))
    came_amd.gated_ffn(*a).backward(torch._neg_view(dy))
    came_amd.gated_ffn(*b).backward(-dy)
    assert all(torch.equal(s.grad, t.grad) for s, t in zip(a, b))
    for cls in _classes():
        p, q = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2))
        g = torch.randn(300, device="cuda")
        p.grad, q.grad = torch._neg_view(g), -g
        a, b = cls([p], lr=0.1), cls([q], lr=0.1)
        for _ in range(2):  # the second with the states that the first has made
            a.step()
            b.step()
            assert torch.equal(p, q)


def test_a_kept_norm_keeps_no_workspace():
    """A program that keeps every step's norm keeps a few bytes a step."""
    import came_amd
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = torch.ones(100, device="cuda")
    opt = came_amd.AdamW([p], max_grad_norm=1.0)
    opt.step()
    for norm in (came_amd.grad_norm([p.grad]), came_amd.clip_grad_norm_([p], 1.0), opt.last_grad_norm):
        assert norm.untyped_storage().nbytes() <= 8


def test_copies_of_an_optimizer_clip_as_it_does():
    for cls in _classes():
        p = torch.nn.Parameter(torch.ones(100, device="cuda"))
        p.grad = torch.ones(100, device="cuda")
        opt = cls([p], max_grad_norm=1e-3)
        opt.step()
        two = copy.deepcopy(opt)
        q = two.param_groups[0]["params"][0]
        q.grad = p.grad.clone()
        opt.step()
        two.step()
        assert torch.equal(p, q) and torch.equal(opt.last_grad_norm, two.last_grad_norm)


def test_a_checkpoint_of_a_transposed_parameter_continues():
    """torch keeps its moments in the parameter's order; the next steps agree within float32 rounding (three roundings of the
    parameter and of an update of at most a few lr a step)."""
    import came_amd
    u, lr = 2.0**-24, 1e-2
    gen = torch.Generator().manual_seed(4)
    p = torch.nn.Parameter(torch.randn(60, 50, generator=gen).cuda().t())
    ref = torch.optim.AdamW([p], lr=lr, weight_decay=0.1, foreach=False)
    p.grad = torch.randn(50, 60, generator=gen).cuda()
    ref.step()
    q = torch.nn.Parameter(p.detach().clone())
    opt = came_amd.AdamW([q], lr=lr, weight_decay=0.1)
    opt.load_state_dict(ref.state_dict())
    for _ in range(3):
        p.grad = torch.randn(50, 60, generator=gen).cuda()
        q.grad = p.grad.clone()
        ref.step()
        opt.step()
    assert ((p - q).abs() <= 3 * (8 * u * p.abs() + 64 * u * lr)).all()


@pytest.mark.parametrize("kind", ["again", "overlapping"])
def test_gradients_that_share_memory_are_scaled_one_after_another(kind):
    """As in torch, a gradient counts in the norm and is scaled as often as it is listed, and so is what two have in common."""
    import came_amd
    n = 40_000_000
    buf = torch.randn(n + 1000, device="cuda")
    views = {"again": [buf, buf, buf], "overlapping": [buf[1000:], buf[:n], buf[500:700]]}[kind]
    before, times = buf.double(), torch.zeros(n + 1000, device="cuda", dtype=torch.float64)
    want = float(torch.stack([v.double().square().sum() for v in views]).sum().sqrt())
    params = []
    for v in views:
        params.append(torch.nn.Parameter(torch.empty_like(v)))
        params[-1].grad = v
        times[v.storage_offset() : v.storage_offset() + v.numel()] += 1
    norm = came_amd.clip_grad_norm_(params, 0.5 * want)
    assert abs(float(norm) / want - 1) < 1e-6
    x = before * (0.5 * want / (want + 1e-6)) ** times
    assert ((buf.double() - x).abs() <= x.abs() * (3 * 10 * 2.0**-24)).all()  # a factor and a product each time
