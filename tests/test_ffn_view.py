"""Where the feed-forward products' loads may reach, on the CPU: the bounds that the kernels give the hardware
(came_amd/csrc/came8_view.h) end with the operand's last element, to the word, and the shifted loads of 16-bit rows an odd
number of elements apart (csrc/came8_ffn.h: Stage with ODD), which ask for words past a row's end, get none past that."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
NOWHERE = 0x80000000
STEP = 128  # bytes of k


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("view") / "view.so")
    subprocess.run([cc, "-O1", "-std=c++17", "-shared", "-fPIC", "-o", out, os.path.join(HERE, "native", "ffn_view.cpp")],
                   check=True)
    so = ctypes.CDLL(out)
    i64 = ctypes.c_int64
    so.view_bytes.restype, so.view_bytes.argtypes = i64, [ctypes.c_int, i64, i64, i64, i64]
    so.buffer_bytes.restype, so.buffer_bytes.argtypes = ctypes.c_int32, [i64]
    return so


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("elem", [2, 4])
def test_a_view_ends_with_the_last_element(lib, rows, elem):
    for extent in (1, 2, 63, 64, 200):
        for K in (1, 7, 8, 64, 129):
            for gap in (0, 1, 2, 9, 1000):
                ld = ((K if rows else extent) + gap) * elem
                r, k = np.arange(extent)[:, None], np.arange(K)[None]
                end = int((r * ld + k * elem if rows else k * ld + r * elem).max()) + elem
                assert lib.view_bytes(rows, extent, K, ld, elem) == end
                assert end <= lib.buffer_bytes(end) < end + 4


def test_the_bound_of_large_and_empty_views(lib):
    assert lib.buffer_bytes(0) == lib.buffer_bytes(-128) == 0
    assert lib.buffer_bytes(1 << 40) == 0x7FFFFFFC


@pytest.mark.parametrize("tile", [64, 128])
@pytest.mark.parametrize("rows,K,ld", [(1, 1, 1), (64, 63, 63), (65, 64, 65), (200, 8, 17), (130, 129, 131), (70, 100, 1001),
                                       (128, 1001, 1003), (2048, 2731, 5461)])
def test_shifted_loads_stay_inside(lib, rows, K, ld, tile):
    """Every word that a load gets lies between the matrix's first byte and the word that holds its last one."""
    last = ((rows - 1) * ld + K) * 2
    threads = np.arange(256)
    for m0 in range(0, rows, tile):
        whole = lib.view_bytes(1, rows - m0, K, ld * 2, 2)
        for at in range(0, K * 2, STEP):
            bound = lib.buffer_bytes(whole - at)
            off = np.where((threads & 7) * 8 >= K - at // 2, NOWHERE, (threads >> 3) * ld * 2 + (threads & 7) * 16)
            shift = off & 2
            for i in range(tile * 8 // 256):
                words = (off - shift + i * 32 * ld * 2)[:, None] + 4 * np.arange(5)
                got = words[words < bound] + m0 * ld * 2 + at
                assert got.size == 0 or (got.min() >= 0 and got.max() + 4 <= (last + 3) // 4 * 4)
