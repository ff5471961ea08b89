"""Layer norm's copies of a row take every element of it and nothing in front of the tensor or behind its end, whatever the width.  What the
kernels call is compiled here for the host."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

SOURCE = """
#include "fda_norm_copy.h"
extern "C" int room(long long left, int width, int each) { return fda_norm::room_of(left, width, each); }
extern "C" int copied(int column, int width, int each, int room) { return fda_norm::copied_elements(column, width, each, room); }
"""


@pytest.fixture(scope="module")
def copies(tmp_path_factory):
    path = tmp_path_factory.mktemp("copies")
    (path / "copies.cpp").write_text(SOURCE)
    out = str(path / "copies.so")
    subprocess.check_call([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "ops3d_b200", "csrc"),
                           str(path / "copies.cpp"), "-o", out])
    lib = ctypes.CDLL(out)
    lib.room.argtypes, lib.copied.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int], [ctypes.c_int] * 4
    return lib


# Elements of a vector of the rows' type, and of a 16-byte unit of the copied tensor: 16-bit rows, an fp32 residual beside them, fp32 rows.
@pytest.mark.parametrize("vector,each", [(8, 8), (8, 4), (4, 4)])
@pytest.mark.parametrize("width", [*range(1, 34), 63, 65, 259])
def test_copies_stay_inside_the_tensor(copies, width, vector, each):
    for rows in range(1, 19):
        total = rows * width
        for row in range(rows + 3):                               # a team's last steps lead behind the last row
            room = copies.room(rows - row, width, each)
            taken = set()
            for column in range(-(row * width % vector), width + 2 * vector, each):
                n = copies.copied(column, width, each, room)
                start = row * width + column
                assert 0 <= n <= each and (n == 0 or (start % each == 0 and 0 <= start and start + n <= total))
                assert n in (0, each) or start + n == total       # cut off at the tensor's end only
                taken.update(range(start, start + n))
            assert row >= rows or taken.issuperset(range(row * width, (row + 1) * width))


def test_many_rows_left(copies):
    """Rows left of which the elements do not fit 32 bits, and rows far behind the last."""
    for width in (1, 7, 4097, (1 << 26) - 1):
        assert copies.copied(-3, width, 8, copies.room(1 << 31, width, 8)) == 8
        assert copies.copied(-3, width, 8, copies.room(1 << 40, width, 8)) == 8
        assert copies.copied(0, width, 8, copies.room(-(1 << 40), width, 8)) == 0
        assert copies.copied(width - 1, width, 8, copies.room(1, width, 8)) == 1
