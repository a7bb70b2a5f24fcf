"""The norm's launches on the CPU (came_amd/csrc/came8_rms_grid.h): work items stay below 2^32 in each dimension for all rows and
widths that are accepted."""
import ctypes
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ITEMS = 1 << 32
THREADS = 1024  # at most


@pytest.fixture(scope="module")
def grid(tmp_path_factory):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("grid") / "grid.so")
    subprocess.run([cc, "-O1", "-std=c++17", "-shared", "-fPIC", "-o", out, os.path.join(HERE, "native", "rms_grid.cpp")], check=True)
    so = ctypes.CDLL(out)
    for name, n in (("max_dim", 0), ("row_groups", 2), ("column_groups", 2), ("join_groups", 1)):
        getattr(so, name).restype, getattr(so, name).argtypes = ctypes.c_int64, [ctypes.c_int64] * n
    return so


def test_launches_of_the_widest_rows(grid):
    most = grid.max_dim()
    assert most == 1 << 30
    for dim in (1, 31, 32, 33, 16385, 40001, 1 << 25, (1 << 27) - 1, 1 << 27, (1 << 27) + 33, most - 1, most):
        assert 0 < grid.join_groups(dim) * THREADS < ITEMS
        assert grid.join_groups(dim) == min(-(-dim // 32), 1 << 20)  # no workgroup without columns
        for vec in (4, 8):
            groups = grid.column_groups(dim, vec)
            assert 0 < groups * THREADS < ITEMS and groups * THREADS * vec >= dim


def test_launches_of_many_rows(grid):
    for rows in (1, 2, 1 << 20, (1 << 20) + 1, (1 << 31) - 1):
        for per in (1, 4, 16):
            groups = grid.row_groups(rows, per)
            assert 0 < groups * THREADS < ITEMS and groups * per < rows + per
            assert groups * per >= rows or groups == 1 << 20  # in turns
