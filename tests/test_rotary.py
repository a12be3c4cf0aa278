"""Descriptions of a rotation that are refused (csrc/rotary.h), on the CPU: plain arithmetic, built here
with the host compiler, and the Python side's own checks."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

import numrs_amd as nr
from numrs_amd import _lib as L

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "numrs_amd", "csrc")
INCLUDE = os.path.dirname(L.HEADER_PATH)

WRAPPERS = """
#include "rotary.h"
extern "C" {
const char *refuse_rotary(const numrs_hip_rotary *r, int64_t dh, int *code) { return rotary::refuse_rotary(r, dh, code); }
const char *refuse_eps(float eps) { return rotary::refuse_eps(eps); }
int lanes_of(int64_t dh) { return rotary::lanes_of(dh); }
double turns_of(const numrs_hip_rotary *r, int i, int *dims, int *pairs) {
  const rotary::Turn t = rotary::turn_of(r);
  *dims = t.dims, *pairs = t.pairs;
  return t.turns[i];
}
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("rotary")
    src, so = d / "rotary.cpp", d / "rotary.so"
    src.write_text(WRAPPERS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    f"-I{INCLUDE}", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    i64, i, p = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p
    for name, res, args in (("refuse_rotary", ctypes.c_char_p, [p, i64, p]), ("lanes_of", i, [i64]),
                            ("refuse_eps", ctypes.c_char_p, [ctypes.c_float]),
                            ("turns_of", ctypes.c_double, [p, i, p, p])):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def _refused(lib, spec, dh):
    code = ctypes.c_int(0)
    why = lib.refuse_rotary(ctypes.byref(spec) if spec is not None else None, dh, ctypes.byref(code))
    return (why, code.value) if why else None


def test_rotations_that_are_refused(lib):
    ok = nr.Rotary(64).spec
    assert _refused(lib, None, 64) is None and _refused(lib, ok, 64) is None and _refused(lib, ok, 128) is None
    assert _refused(lib, L.RotarySpec(None, 0, 0), 8) is None
    assert _refused(lib, ok, 56)[1] == L.E_SHAPE  # more columns than the head has
    for dims in (-8, 4, 12, 63, 136):
        assert _refused(lib, L.RotarySpec(ok.freqs, dims, 0), 128)[1] == L.E_SHAPE
    for layout in (-1, 2):
        assert _refused(lib, L.RotarySpec(ok.freqs, 64, layout), 64)[1] == L.E_INVALID
    assert _refused(lib, L.RotarySpec(None, 8, 0), 64)[1] == L.E_INVALID
    for bad in (math.nan, math.inf, -math.inf, 1.1e6):
        assert _refused(lib, nr.Rotary(8, freqs=[1, 1, bad, 1]).spec, 8)[1] == L.E_INVALID
    assert _refused(lib, nr.Rotary(8, freqs=[0, -1, 1e6, 1e-300]).spec, 8) is None


def test_eps_that_are_refused(lib):
    assert lib.refuse_eps(0.0) is None and lib.refuse_eps(1e-6) is None and lib.refuse_eps(1e30) is None
    for bad in (-1e-9, math.nan, math.inf, -math.inf):
        assert lib.refuse_eps(bad)


def test_lanes_and_turns(lib):
    assert [lib.lanes_of(d) for d in (8, 16, 24, 32, 40, 64, 72, 80, 96, 120, 128)] == [0, 1, 2, 2, 3, 3, 4, 4, 4, 4, 4]
    r = nr.Rotary(128, 96, base=500000.0, layout="pairs")
    dims, pairs = ctypes.c_int(), ctypes.c_int()
    for i in range(48):
        t = lib.turns_of(ctypes.byref(r.spec), i, ctypes.byref(dims), ctypes.byref(pairs))
        assert abs(t * 2 * math.pi / 500000.0 ** (-2 * i / 96) - 1) <= 4 * 2.0 ** -52
    assert (dims.value, pairs.value) == (96, 1)
    lib.turns_of(None, 0, ctypes.byref(dims), ctypes.byref(pairs))
    assert dims.value == 0


def test_python_rotary():
    r = nr.Rotary(80, 40)
    assert np.allclose(r.freqs, 10000.0 ** (-np.arange(0, 40, 2) / 40)) and r.spec.dims == 40
    assert nr.Rotary(64).dims == 64 and nr.Rotary(64, freqs=np.ones(32)).freqs.tolist() == [1.0] * 32
    for args, kw in (((64, 7), {}), ((64, 72), {}), ((64, 0), {}), ((64,), {"layout": "odd"}), ((64,), {"base": 0}),
                     ((64,), {"freqs": [1.0]}), ((4,), {})):
        with pytest.raises(ValueError):
            nr.Rotary(*args, **kw)


def test_a_description_keeps_its_frequencies():
    """`spec` holds an address: what it leads to lives as long as it does, and is what `freqs` shows."""
    r = nr.Rotary(64, freqs=np.arange(32.0))
    spec = r.spec
    del r
    others = [np.full(32, 7.0) for _ in range(4)]  # takes the place of what was given back
    assert spec.freqs[:32] == list(range(32))
    r = nr.Rotary(64)
    with pytest.raises(AttributeError):
        r.freqs = np.zeros(32)
    r.freqs[3] = 0.25
    assert r.spec.freqs[:32] == r.freqs.tolist()
    del others
