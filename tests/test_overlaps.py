"""Which arrays' rows meet (csrc/paging.h), on the CPU: plain integer arithmetic, built here with the host
compiler and compared with every row against every other."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

from numrs_amd import _lib as L

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "numrs_amd", "csrc")

WRAPPER = """
#include "paging.h"
extern "C" int rows_meet(int64_t a, int64_t na, int64_t la, int64_t b, int64_t nb, int64_t lb, int64_t rows) {
  return paging::rows_meet({reinterpret_cast<const float *>(a), na, la}, {reinterpret_cast<const float *>(b), nb, lb}, rows);
}
"""


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlaps")
    src, so = d / "overlaps.cpp", d / "overlaps.so"
    src.write_text(WRAPPER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    f"-I{os.path.dirname(L.HEADER_PATH)}", str(src), "-o", str(so)], check=True)
    fn = ctypes.CDLL(str(so)).rows_meet
    fn.argtypes = [ctypes.c_int64] * 7
    return fn


def test_against_every_pair_of_rows(meet):
    base, some = 1 << 40, [0, 0]
    for na, nb, rows in itertools.product((1, 2, 5), (1, 3), (1, 2, 4)):
        for la, lb in itertools.product({na, na + 1, na + nb, 9}, {nb, nb + 2, na + nb, 9}):
            a = np.arange(rows)[:, None] * la + np.arange(na)
            for d in range(-4 * 9 - 6, 4 * 9 + 7):
                b = d + np.arange(rows)[:, None] * lb + np.arange(nb)
                want = bool(np.intersect1d(a, b).size)
                some[want] += 1
                assert bool(meet(base, na, la, base + 4 * d, nb, lb, rows)) == want, (na, la, nb, lb, rows, d)
    assert min(some) > 1000


def test_large_and_empty(meet):
    base, rows, ld = 1 << 46, 2 ** 30, 2 ** 31 - 1
    assert not meet(base, 8, 8, base, 8, 8, 0) and not meet(base, 0, 8, base, 8, 8, 5)
    assert meet(base, 8, ld, base + 4 * (rows - 1) * ld, 8, ld, rows)
    assert meet(base + 4 * (rows - 1) * ld, 8, ld, base, 8, ld, rows)
    assert not meet(base, 8, ld, base + 4 * rows * ld, 8, ld, rows)
    assert not meet(base, 8, ld, base + 4 * (5 * ld + 8), 8, ld, rows)
    assert meet(base, 8, ld, base + 4 * (5 * ld + 7), 8, ld, rows)
    assert meet(base, 8, ld, base - 4 * (5 * ld + 7), 8, ld, rows)
    assert not meet(base, 8, ld, base - 4 * (5 * ld + 8), 8, ld, rows)
    # half an element
    assert meet(base, 8, 16, base + 31, 8, 16, 4) and not meet(base, 8, 16, base + 32, 8, 16, 4)
