"""What programs count on around AdamW and the gradient clip, on the host: nothing is left out in silence, copies and
checkpoints keep what a step goes by."""
import copy
import pickle
import types

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._pytree import tree_map

import came_amd


class Elsewhere(torch.Tensor):
    """A subclass that says it is on the GPU and keeps its values in a tensor of its own, as distributed tensors do."""

    @staticmethod
    def __new__(cls, inner):
        t = torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device="cuda:0")
        t.inner = inner
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        bare = lambda x: x.inner if isinstance(x, Elsewhere) else x  # noqa: E731
        out = func(*tree_map(bare, args), **tree_map(bare, kwargs or {}))
        return tree_map(lambda x: Elsewhere(x) if isinstance(x, torch.Tensor) else x, out)


@pytest.fixture
def elsewhere(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
    p = torch.nn.Parameter(Elsewhere(torch.zeros(4)))
    p.grad = Elsewhere(torch.full((4,), 100.0))
    return p


def test_a_clip_that_cannot_be_taken_raises(elsewhere):
    with pytest.raises(RuntimeError, match="clip_grad_norm_: tensor subclasses"):
        came_amd.clip_grad_norm_([elsewhere], 1.0)
    with pytest.raises(RuntimeError, match="grad_norm: tensor subclasses"):
        came_amd.grad_norm([elsewhere.grad])


@pytest.mark.parametrize("cls", [came_amd.AdamW, came_amd.AdamW8bit])
def test_a_step_whose_clip_cannot_be_taken_raises(cls, elsewhere):
    with pytest.raises(RuntimeError, match="tensor subclasses"):
        cls([elsewhere], max_grad_norm=1.0).step()


def test_compressed_sparse_gradients_are_refused():
    p = torch.nn.Parameter(torch.eye(3))
    g = torch.eye(3).to_sparse_csr()
    with pytest.raises(RuntimeError, match="sparse"):
        came_amd.grad_norm([g])


def test_absmax_of_another_device_is_refused():
    from came_amd import blockwise_quantization as bq
    for dtype, call in ((torch.uint8, lambda q, a: bq.dequantize_second_moment(q, a, block_size=64)),
                        (torch.int8, lambda q, a: bq.dequantize_blockwise(q, a, signed=True, block_size=64))):
        q = Elsewhere(torch.zeros(100, dtype=dtype))
        with pytest.raises(RuntimeError, match="codes on cuda:0, absmax on cpu"):
            call(q, torch.ones(2))
        with pytest.raises(ValueError, match="fewer entries"):
            call(q, Elsewhere(torch.ones(1)))


@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_of_the_feed_forward_block_is_refused(grad):
    w = torch.zeros(24, 16)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(5, 16), torch.ones(5, 16))
        with pytest.raises(RuntimeError, match="forward-mode"):
            came_amd.gated_ffn(x, w, w, w.t())


def test_a_trace_of_the_feed_forward_block_is_refused():
    w = torch.zeros(24, 16)
    with pytest.raises(RuntimeError, match="gated_ffn: cannot be traced"):
        torch.jit.trace(lambda x: came_amd.gated_ffn(x, w, w, w.t()), (torch.zeros(5, 16),), check_trace=False)


@pytest.mark.parametrize("cls", [came_amd.AdamW, came_amd.AdamW8bit])
@pytest.mark.parametrize("bound", [None, 0.0, 2.5])
@pytest.mark.parametrize("way", [copy.deepcopy, lambda opt: pickle.loads(pickle.dumps(opt))], ids=["deepcopy", "pickle"])
def test_copies_keep_the_clip_bound(cls, bound, way):
    opt = cls([torch.nn.Parameter(torch.zeros(3))], max_grad_norm=bound)
    two = way(opt)
    assert two.max_grad_norm == bound and two.last_grad_norm is None
    two.step()  # no gradient: nothing to do
    two.load_state_dict(opt.state_dict())
    assert two.max_grad_norm == bound


def _stepped(p, **kw):
    """A torch.optim.AdamW over p after a step."""
    opt = torch.optim.AdamW([p], **kw)
    p.grad = torch.ones_like(p)
    opt.step()
    return opt


@pytest.mark.parametrize("option", ["amsgrad", "maximize"])
def test_options_that_the_step_does_not_have_are_refused(option):
    p = torch.nn.Parameter(torch.zeros(5))
    opt = came_amd.AdamW([p], lr=0.5)
    with pytest.raises(ValueError, match=option):
        opt.load_state_dict(_stepped(p, **{option: True}).state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and not opt.param_groups[0].get(option) and not opt.state
    opt.load_state_dict(_stepped(p, lr=0.25).state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and opt.state[p]["step"] == 1
    with pytest.raises(ValueError, match=option):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))], option: True})
    assert len(opt.param_groups) == 1
    for cls in (came_amd.AdamW, came_amd.AdamW8bit):
        with pytest.raises(ValueError, match=option):
            cls([{"params": [p], option: True}])
        cls([{"params": [p], option: False}])


@pytest.mark.parametrize("p", [torch.randn(6, 4).t(), torch.randn(2, 3, 4, 5).to(memory_format=torch.channels_last)],
                         ids=["transposed", "channels_last"])
def test_moments_in_the_order_of_a_strided_parameter_are_taken(p):
    p = torch.nn.Parameter(p)
    ref = torch.optim.AdamW([p])
    p.grad = torch.randn(p.shape).contiguous()
    ref.step()
    assert not ref.state[p]["exp_avg"].is_contiguous()
    opt = came_amd.AdamW([p])
    opt.load_state_dict(ref.state_dict())
    for key in ("exp_avg", "exp_avg_sq"):
        got = opt.state[p][key]
        assert got.is_contiguous() and torch.equal(got, ref.state[p][key])
        assert got.data_ptr() != ref.state[p][key].data_ptr()


@pytest.mark.parametrize("wrong", ["type", "size", "missing", "groups"])
def test_a_refused_load_leaves_the_optimizer_as_it_was(wrong):
    p, q = torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(7))
    opt = came_amd.AdamW([p, q], lr=0.5)
    opt.load_state_dict(_two(p, q).state_dict())
    opt.param_groups[0]["lr"] = 0.5
    kept = copy.deepcopy(opt.state_dict())
    saved = _two(p, q, lr=0.25).state_dict()
    st = saved["state"][1]  # of the second parameter: the first one's is fine
    if wrong == "type":
        st["exp_avg"] = st["exp_avg"].half()
    elif wrong == "size":
        st["exp_avg_sq"] = torch.zeros(6)
    elif wrong == "missing":
        del st["exp_avg"]
    else:
        saved["param_groups"][0]["params"].append(2)
    with pytest.raises((RuntimeError, ValueError)):
        opt.load_state_dict(saved)
    now = opt.state_dict()
    assert now["param_groups"] == kept["param_groups"]
    for k, st in kept["state"].items():
        for key, v in st.items():
            w = now["state"][k][key]
            assert torch.equal(v, w) if isinstance(v, torch.Tensor) else v == w


def _two(p, q, **kw):
    """A torch.optim.AdamW over both after a step."""
    opt = torch.optim.AdamW([p, q], **kw)
    p.grad, q.grad = torch.randn(5), torch.randn(7)
    opt.step()
    return opt


@pytest.mark.parametrize("norm_type", [2.0, 1.0, 2, float("inf"), "inf"])
def test_a_norm_type_in_torchs_place_is_refused(norm_type):
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(TypeError, match="always the 2-norm"):
        came_amd.clip_grad_norm_([p], 1.0, norm_type)
    for flag in (True, False):
        assert float(came_amd.clip_grad_norm_([p], 1.0, flag)) == 0.0


@pytest.mark.parametrize("cls", [came_amd.AdamW, came_amd.AdamW8bit])
def test_a_parameter_that_appears_twice_is_refused(cls):
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    for params in ([p, q, p], iter([p, p]), [{"params": [q]}, {"params": (p, p)}], [{"params": iter([q, q])}],
                   [("first", p), ("second", p)]):
        with pytest.raises(ValueError, match="appears twice"):
            cls(params)
    for params in ([p, q], iter([p, q]), [{"params": iter([p])}, {"params": q}], [("first", p), ("second", q)]):
        assert sum(len(g["params"]) for g in cls(params).param_groups) == 2


def test_hooks_of_a_load_are_heard():
    p = torch.nn.Parameter(torch.zeros(5, dtype=torch.bfloat16))
    saved = _stepped(torch.nn.Parameter(torch.zeros(5))).state_dict()
    opt = came_amd.AdamW([p])

    def hook(_, given):
        state = {k: {key: v if key == "step" else v + 1 / 3 for key, v in st.items()} for k, st in given["state"].items()}
        return {**given, "state": state}

    opt.register_load_state_dict_pre_hook(hook)
    opt.load_state_dict(saved)
    for key in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(opt.state[p][key], saved["state"][0][key] + 1 / 3)
