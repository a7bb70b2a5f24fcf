"""AdamW's states past 2^31 elements: every state tensor of the last elements, against the definition in 64 bits."""
import pytest
import torch

from oracle import adamw_oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0**-24
BETAS = (0.9, 0.999)


@pytest.mark.parametrize("bits", [32, 8])
def test_states_past_2_31_elements(bits):
    """From zero moments, m = (1 - b1) g and v = (1 - b2) g^2 in float32: a rounding of the coefficient, of g^2 and of the product,
    within 4 units.  8-bit blocks are counted from the tensor's start, so the last block may be short."""
    import came_amd
    from came_amd import blockwise_quantization as bq
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    n, tail, B = (1 << 31) + 1027, 5000, 256
    gen = torch.Generator().manual_seed(8)
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = (torch.randn(tail, generator=gen) * torch.exp(torch.randn(tail, generator=gen))).to(torch.bfloat16)
    p.grad[-tail:] = g.cuda()
    opt = (came_amd.AdamW8bit if bits == 8 else came_amd.AdamW)([p], lr=1e-2)
    opt.step()
    m1, v1 = orc.moments64(g, torch.zeros(tail), torch.zeros(tail), BETAS)
    st = opt.state[p]
    if bits == 32:
        assert ((st["exp_avg"][-tail:].cpu().double() - m1).abs() <= 4 * U * m1.abs()).all()
        assert ((st["exp_avg_sq"][-tail:].cpu().double() - v1).abs() <= 4 * U * v1).all()
        assert int(st["exp_avg_sq"][: n - tail].count_nonzero()) == 0
        return
    start = (n - tail) // B * B  # the block that the tail begins in
    pad = torch.zeros(n - tail - start, dtype=torch.float64)
    m1, v1 = torch.cat([pad, m1]), torch.cat([pad, v1])
    for values, key in ((m1, "exp_avg_absmax"), (v1, "exp_avg_sq_absmax")):
        top = torch.stack([b.abs().max() for b in values.split(B)])
        got = st[key].cpu().double()
        assert got.numel() == -(-n // B) and (got[: start // B] == 1).all()
        assert ((got[start // B :] - top).abs() <= 4 * U * top).all()
    at = slice(start // B, None)
    hm = bq.dequantize_blockwise(st["exp_avg_q"][start:], st["exp_avg_absmax"][at], signed=True, block_size=B).cpu().double()
    hv = bq.dequantize_second_moment(st["exp_avg_sq_q"][start:], st["exp_avg_sq_absmax"][at], block_size=B).cpu().double()
    top = st["exp_avg_absmax"][at].cpu().double().repeat_interleave(B)[: m1.numel()]
    assert ((hm - m1).abs() <= top * (0.5 / 127 + 8 * U)).all()
    top = st["exp_avg_sq_absmax"][at].cpu().double().repeat_interleave(B)[: v1.numel()] * 8 / 15
    grid = torch.maximum(v1 / 8, top * 2.0**-33)  # a step of the grid is at most an eighth of the value
    assert ((hv - v1).abs() <= grid * (1 + 1e-6) + v1 * 8 * U).all()
    assert int(st["exp_avg_sq_q"][:start].count_nonzero()) == 0
