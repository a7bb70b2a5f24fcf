"""The gated feed-forward block with a down projection that is a slice of columns of a wider matrix whose rows lie an odd number of
elements apart (a shard, for instance): the columns beside it, NaN here, are not the operand's."""
import pytest
import torch

from oracle import ffn_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T", [1, 17, 48, 130, 700])
@pytest.mark.parametrize("hidden,before,after", [(129, 2, 0), (129, 0, 2), (64, 4, 3), (65, 2, 2), (1001, 6, 0), (2731, 2730, 0),
                                                 (8, 2, 1)])
def test_a_slice_of_odd_strided_rows(T, hidden, before, after, dtype):
    from came_amd import gated_ffn
    D, E = 72, 200
    gen = torch.Generator().manual_seed(T + hidden)
    x, wg, wu, wd = ((torch.randn(*s, generator=gen) * s[1] ** -0.5).to(dtype).cuda()
                     for s in ((T, D), (hidden, D), (hidden, D), (E, hidden)))
    wide = torch.full((E, before + hidden + after), float("nan"), dtype=dtype, device="cuda")
    assert wide.stride(0) % 2 == 1
    wide[:, before : before + hidden] = wd
    ops = [x, wg, wu, wide[:, before : before + hidden]]
    want, bound, kept = orc.forward(*ops, "silu", dtype)
    leaves = [t.detach().requires_grad_() for t in ops]
    dy = torch.randn(T, E, generator=gen).to(dtype).cuda()
    y = gated_ffn(*leaves)
    y.backward(dy)
    with torch.no_grad():
        alone = gated_ffn(*ops)
    for got in (y.detach(), alone):
        assert ((got.cpu().double() - want).abs() <= bound).all()
    grads = orc.backward(kept, dy)
    for leaf, name in zip(leaves, ("x", "w_gate", "w_up", "w_down")):
        g, b = grads[name]
        assert ((leaf.grad.cpu().double() - g).abs() <= b).all(), name
