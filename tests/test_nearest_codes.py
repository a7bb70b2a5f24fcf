"""Codes of values next to a border between two, on the CPU: the kernels' rule (came_amd/csrc/came8_codes.h) and the oracle's
against whole numbers of any size."""
import ctypes
import os
import shutil
import subprocess
from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import lm_oracle as orc

HERE = os.path.dirname(os.path.abspath(__file__))
U = 2.0**-24


def nearest(p, a):
    """127 p / a to nearest, ties to even, of two numbers that are held exactly."""
    e = Fraction(float(p)) * 127 / Fraction(float(a))
    k = e.numerator // e.denominator
    rest = e - k
    return k + (1 if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and k % 2) else 0)


def pairs(n, rng):
    """Values p and largest ones a >= |p|, products of two float32 numbers each: exact ties, what is as near to one as such products
    come by chance, and values anywhere."""
    half = n // 2
    m, w = rng.integers(1, 2**24 // 127 // 2, half) * 2, rng.integers(2**23, 2**24, half)
    k = rng.integers(0, 127, half)
    p = ((2 * k + 1) * m // 2).astype(np.float64) * w * rng.choice([-1.0, 1.0], half)  # (2k + 1) / 254 of the largest
    a = (127 * m).astype(np.float64) * w
    h, w = rng.integers(2**23, 2**24, n - half), rng.integers(2**23, 2**24, n - half)
    b = h.astype(np.float64) * w
    k, v = rng.integers(0, 127, n - half), rng.integers(2**23, 2**24, n - half)
    g = np.rint((k + 0.5) * b / 127 / v)
    g = np.where(g < 2**24, g, 2**24 - 1)
    fits = np.abs(g * v) <= b
    any_h = rng.integers(0, h + 1)  # anywhere
    return np.concatenate([p, (g * v)[fits], any_h.astype(np.float64) * w]), np.concatenate([a, b[fits], b])


# h and w of a row of two values: the second's quotient is 2e-15 from a border, nearer than 64 bits tell
KNOWN = [((15865167, 14861102), (15345633, 15672959), 121), ((8715477, 4698892), (10378235, 13262443), 87)]


def test_known_rows():
    for h, w, code in KNOWN:
        p, a = float(h[1] * w[1]), float(h[0] * w[0])
        assert nearest(p, a) == code != round(p * 127 / a)


def test_the_kernels_rule(tmp_path):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("g++ not available")
    out = str(tmp_path / "codes.so")
    subprocess.run([cc, "-O1", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC", "-o", out, os.path.join(HERE, "native", "codes.cpp")],
                   check=True)
    fn = ctypes.CDLL(out).nearest_codes
    fn.restype, fn.argtypes = None, [ctypes.c_void_p] * 5 + [ctypes.c_long]
    rng = np.random.default_rng(0)
    p, a = pairs(40_000, rng)
    for h, w, _ in KNOWN:
        p, a = np.append(p, float(h[1] * w[1])), np.append(a, float(h[0] * w[0]))
    want = np.array([nearest(*v) for v in zip(p, a)])
    assert (np.rint(p * 127 / a) != want).sum() > 100  # what 64 bits get wrong
    for scale in (2.0**-52, 1.0, 2.0**60):  # powers of two move no code
        q = p * 127 / a
        for off in (-1e-4, -3e-5, -1e-7, 0.0, 1e-7, 3e-5, 1e-4):  # what a quotient in 32 bits may be off by
            x = (q + off * 0.9).astype(np.float32)
            c = np.rint(x)
            got = np.zeros(len(p), np.float32)
            args = [np.ascontiguousarray(t) for t in (x, c, p * scale, a * scale)]
            fn(*[t.ctypes.data for t in args], got.ctypes.data, len(got))
            assert (got == want).all()


def test_the_oracles_codes():
    rng = np.random.default_rng(1)
    p, a = pairs(20_000, rng)
    got = orc.codes(torch.from_numpy(p), torch.from_numpy(a))
    assert got.tolist() == [nearest(*v) for v in zip(p, a)]
    for h, w, code in KNOWN:
        x, weight = torch.tensor([h], dtype=torch.float32), torch.tensor(w, dtype=torch.float32)
        assert orc.rms_norm_int8(x, weight, 1e-6)[0].tolist() == [[127, code]]
