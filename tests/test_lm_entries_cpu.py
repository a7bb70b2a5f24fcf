"""What the C entries of a language model's operators refuse, on the host, beside what test_lm_operators_cpu.py has."""
import ctypes

import pytest

from came_amd import _lib as L

P = 0x1000  # an aligned address that nothing reads: what is refused launches nothing


@pytest.mark.parametrize("eps", [1e39, 1.7e308])
def test_the_norm_refuses_an_eps_that_is_infinite_in_float32(eps):
    lib, n = L.load(), L.Came8RmsNorm(4, 8, 8, 8, eps, L.CAME8_BF16, 0)
    ref = ctypes.byref(n)
    for rc in (lib.came8_rms_norm_forward(ref, P, P, P, P, P, None), lib.came8_rms_norm_int8(ref, P, P, P, P, 16, P, P, None),
               lib.came8_rms_norm_backward(ref, P, P, P, P, P, P, P, 1 << 50, None)):
        assert rc == L.CAME8_EINVAL
        with pytest.raises(RuntimeError, match="eps"):
            L.check(rc, "norm")
