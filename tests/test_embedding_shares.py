"""Where the embedding's gradient notes which tokens cross from a share of the sorted positions to the next, on the CPU
(came_amd/csrc/came8_shares.h): every share's end once, inside the list, up to the longest list that is accepted."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
MOST = (1 << 31) - 1  # positions


@pytest.fixture(scope="module")
def ends(tmp_path_factory):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("shares") / "shares.so")
    subprocess.run([cc, "-O1", "-std=c++17", "-shared", "-fPIC", "-o", out, os.path.join(HERE, "native", "shares.cpp")], check=True)
    fn = ctypes.CDLL(out).share_ends
    i64 = ctypes.c_int64
    fn.restype, fn.argtypes = i64, [i64, i64, i64, ctypes.c_void_p, i64]

    def call(start, count, share):
        pairs = np.zeros((4096, 2), np.int64)
        n = fn(start, count, share, pairs.ctypes.data, len(pairs))
        assert n <= len(pairs)
        return [tuple(map(int, p)) for p in pairs[:n]]

    return call


def _share(positions):
    return max(16, -(-positions // 2048))


def _expected(start, count, share):
    """From the definition, in whole numbers of any size."""
    out = []
    for s in range(start // share, (start + count) // share):
        begins, goes_on = start >= s * share, start + count > (s + 1) * share
        out.append((s, (start + count - 1) // share if begins and goes_on else -1))
    return out


@pytest.mark.parametrize("positions", [MOST, MOST - 1, MOST - (1 << 20), (1 << 31) - (1 << 21), 1 << 30, 100_000, 40])
def test_tokens_near_the_end_of_a_list(ends, positions):
    share = _share(positions)
    shares = -(-positions // share)
    for back in {1, 2, share // 2, share - 1, share, share + 1, 2 * share, 5 * share + 3, positions}:
        for left in {0, 1, share // 2, share}:  # positions behind the token's
            start, count = max(0, positions - back), min(back, positions) - left
            if count < 0:
                continue
            got = ends(start, count, share)
            assert got == (_expected(start, count, share) if count else [])
            assert all(0 <= s < shares and -1 <= last < shares for s, last in got)


@pytest.mark.parametrize("positions", [MOST, 70_000, 333])
def test_every_share_ends_once(ends, positions):
    rng = np.random.default_rng(positions)
    share = _share(positions)
    cuts = np.unique(np.concatenate([[0, positions], rng.integers(0, positions, 400), [max(0, positions - share // 2)]]))
    seen = [s for a, b in zip(cuts[:-1], cuts[1:]) for s, _ in ends(int(a), int(b - a), share)]
    assert seen == list(range(positions // share))
