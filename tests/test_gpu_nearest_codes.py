"""The 8-bit codes of the fp32 norm, whose products have 48 bits: ties, and values nearer to a border between two codes than 64
bits tell."""
import pytest
import torch

from oracle import lm_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("h,w,code", [((15865167, 14861102), (15345633, 15672959), 121), ((8715477, 4698892), (10378235, 13262443), 87)])
@pytest.mark.parametrize("D", [2, 300, 3000, 20000])
def test_values_nearer_to_a_border_than_64_bits_tell(h, w, code, D):
    from came_amd import rms_norm_int8
    x, weight = torch.zeros(1, D), torch.ones(D)
    x[0, :2], weight[:2] = torch.tensor(h, dtype=torch.float32), torch.tensor(w, dtype=torch.float32)
    for sign in (1, -1):
        x[0, 1] *= sign
        q, _ = rms_norm_int8(x.cuda(), weight.cuda())
        assert q[0, :2].tolist() == [127, code * int(torch.sign(x[0, 1]))] and not q[0, 2:].any()


@pytest.mark.parametrize("T,D", [(2000, 60), (300, 700), (40, 5000), (7, 30000)])
def test_ties_of_products(T, D):
    """Values (2k + 1) / 254 of the row's largest, all by one weight of 24 bits."""
    from came_amd import rms_norm_int8
    gen = torch.Generator().manual_seed(D)
    m = 2 * torch.randint(1, 2**24 // 127 // 2, (T, 1), generator=gen)
    k = torch.randint(0, 127, (T, D), generator=gen)
    x = ((2 * k + 1) * m // 2).float() * (2.0 * torch.randint(0, 2, (T, D), generator=gen) - 1)
    at = torch.randint(0, D, (T, 1), generator=gen)
    x.scatter_(1, at, 127.0 * m.float())
    weight = torch.full((D,), float(2**23 + 1 + 2 * int(torch.randint(0, 2**22 - 1, (), generator=gen))))
    want = (torch.sign(x) * (k + k % 2)).to(torch.int8).scatter_(1, at, torch.tensor(127, dtype=torch.int8).expand(T, 1))
    q, _ = rms_norm_int8(x.cuda(), weight.cuda())
    assert torch.equal(orc.rms_norm_int8(x, weight, 1e-6)[0], want)
    assert torch.equal(q.cpu(), want)
