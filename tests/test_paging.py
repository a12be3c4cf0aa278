"""Where a cached token lies and which descriptions are refused (csrc/paging.h), on the CPU: the
header's functions are plain integer arithmetic that the kernels share, built here with the host
compiler."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

from numrs_amd import KVPages
from numrs_amd import _lib as L

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "numrs_amd", "csrc")
INCLUDE = os.path.dirname(L.HEADER_PATH)

WRAPPERS = """
#include "paging.h"
extern "C" {
int page_of(const int32_t *row, int64_t m, int shift, int64_t pages, int64_t pos) {
  return paging::page_of(row, m, shift, pages, pos);
}
int64_t page_base(int64_t p, int64_t hk, int64_t h, int shift, int64_t dh) {
  return paging::page_base(p, hk, h, shift, dh);
}
int64_t value_code(int64_t slot, int64_t d, int64_t dh) { return paging::value_code(slot, d, dh); }
int64_t held(int64_t len, int64_t m, int shift) { return paging::held(len, m, shift); }
int log2_of(int64_t n) { return paging::log2_of(n); }
const char *refuse_cache(const numrs_hip_kv_cache *c, int *code) { return paging::refuse_cache(c, code); }
const char *refuse_table(const void *t, int64_t m, const void *l, int64_t n, int *code) {
  return paging::refuse_table(t, m, l, n, code);
}
const char *refuse_heads(int64_t h, int64_t hk, int64_t dh) { return paging::refuse_heads(h, hk, dh); }
int bad_grid(int64_t n) { return paging::bad_grid(n); }
int bad_stride(int64_t ld, int64_t w) { return paging::bad_stride(ld, w); }
int64_t packed_total(const int64_t *l, int64_t n) { return paging::packed_total(l, n); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("paging")
    src, so = d / "paging.cpp", d / "paging.so"
    src.write_text(WRAPPERS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    f"-I{INCLUDE}", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    i64, i, p = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p
    for name, res, args in (("page_of", i, [p, i64, i, i64, i64]), ("held", i64, [i64, i64, i]),
                            ("page_base", i64, [i64, i64, i64, i, i64]), ("value_code", i64, [i64] * 3),
                            ("log2_of", i, [i64]), ("refuse_cache", ctypes.c_char_p, [p, p]),
                            ("refuse_table", ctypes.c_char_p, [p, i64, p, i64, p]),
                            ("refuse_heads", ctypes.c_char_p, [i64] * 3), ("bad_stride", i, [i64] * 2),
                            ("bad_grid", i, [i64]), ("packed_total", i64, [p, i64])):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def test_no_table_and_no_position_leads_outside_the_cache(lib):
    pages, shift, hk, dh = 5, 4, 3, 24
    size = pages * hk * (1 << shift) * dh
    bad = [-1, -2**31, 5, 6, 2**31 - 1]
    for row in itertools.chain(itertools.product([0, 4, *bad], repeat=2), [(3, 1)]):
        r = np.array(row, np.int32)
        for pos in (-2**31, -17, -1, 0, 1, 15, 16, 31, 32, 47, 2**31 - 1, 2**40):
            p = lib.page_of(r.ctypes.data, len(row), shift, pages, pos)
            good = 0 <= pos < 32 and 0 <= row[pos // 16] < pages
            assert p == (row[pos // 16] if good else -1), (row, pos)
            if p < 0:
                continue
            for h in range(hk):
                base, slot = lib.page_base(p, hk, h, shift, dh), pos % 16
                assert base == (p * hk + h) * 16 * dh
                assert 0 <= base + slot * dh + dh - 1 < size
                codes = {lib.value_code(slot, d, dh) for d in range(dh)}
                assert len(codes) == dh and 0 <= min(codes) and max(codes) < 16 * dh


def test_codes_of_a_page_do_not_collide(lib):
    for dh in (8, 40, 128):
        at = [lib.value_code(s, d, dh) for s in range(64) for d in range(dh)]
        assert sorted(at) == list(range(64 * dh))
        assert lib.value_code(5, 3, dh) == (1 * dh + 3) * 4 + 1


def test_offsets_pass_32_bits(lib):
    assert lib.page_base(2**20, 8, 7, 8, 128) == (2**20 * 8 + 7) * 256 * 128


def test_lengths_stay_within_the_table(lib):
    for n, m, shift, want in ((0, 3, 4, 0), (-5, 3, 4, 0), (48, 3, 4, 48), (49, 3, 4, 48),
                              (2**31 - 1, 3, 4, 48), (2**31 - 1, 2**31 - 1, 16, 2**31 - 1)):
        assert lib.held(n, m, shift) == want
    assert [lib.log2_of(n) for n in (16, 64, 65536)] == [4, 6, 16]


def _cache(**change):
    args = dict(k=64, v=128, k_scale=256, v_scale=512, pages=7, page_size=16, kv_heads=2, head_dim=40,
                format=L.KV_INT8)
    args.update(change)
    return KVPages(*(args[f] for f, _ in KVPages._fields_))


@pytest.mark.parametrize("change,code", [
    ({}, 0), ({"format": L.KV_F32, "k_scale": None, "v_scale": None}, 0), ({"page_size": 65536}, 0),
    ({"format": 2}, L.E_INVALID), ({"format": -1}, L.E_INVALID), ({"k": None}, L.E_INVALID),
    ({"v": None}, L.E_INVALID), ({"k_scale": None}, L.E_INVALID), ({"v_scale": None}, L.E_INVALID),
    ({"k": 72}, L.E_INVALID), ({"v": 130}, L.E_INVALID), ({"v_scale": 516}, L.E_INVALID),
    ({"page_size": 8}, L.E_SHAPE), ({"page_size": 48}, L.E_SHAPE), ({"page_size": 0}, L.E_SHAPE),
    ({"page_size": -16}, L.E_SHAPE), ({"page_size": 131072}, L.E_SHAPE), ({"kv_heads": 0}, L.E_SHAPE),
    ({"kv_heads": 65536}, L.E_SHAPE), ({"head_dim": 0}, L.E_SHAPE), ({"head_dim": 12}, L.E_SHAPE),
    ({"head_dim": 136}, L.E_SHAPE), ({"pages": 0}, L.E_SHAPE), ({"pages": 2**31}, L.E_SHAPE),
    ({"pages": 2**31 - 1, "page_size": 65536, "kv_heads": 65535, "head_dim": 128}, L.E_SHAPE)])
def test_cache_descriptions(lib, change, code):
    got, cache = ctypes.c_int(0), _cache(**change)
    why = lib.refuse_cache(ctypes.addressof(cache), ctypes.byref(got))
    assert (why is None) == (code == 0)
    if code:
        assert got.value == code and why


def test_null_cache_tables_heads_and_strides(lib):
    got = ctypes.c_int(0)
    assert lib.refuse_cache(None, ctypes.byref(got)) and got.value == L.E_INVALID
    for t, m, n_ptr, n, code in ((8, 1, 8, 3, 0), (None, 1, None, 0, 0), (None, 1, 8, 3, L.E_INVALID),
                                 (8, 1, None, 3, L.E_INVALID), (8, 0, 8, 3, L.E_SHAPE),
                                 (8, 2**31, 8, 3, L.E_SHAPE), (8, 1, 8, -1, L.E_INVALID),
                                 (8, 1, 8, 2**24, L.E_SHAPE)):
        why = lib.refuse_table(t, m, n_ptr, n, ctypes.byref(got))
        assert (why is None) == (code == 0) and (code == 0 or got.value == code)
    for h, hk, dh, ok in ((8, 8, 64, 1), (8, 1, 8, 1), (32, 4, 128, 1), (8, 3, 64, 0), (0, 1, 64, 0),
                          (8, 0, 64, 0), (-8, -1, 64, 0), (65536, 1, 64, 0), (8, 8, 0, 0), (8, 8, 4, 0),
                          (8, 8, 60, 0), (8, 8, 136, 0), (4, 8, 64, 0)):
        assert (lib.refuse_heads(h, hk, dh) is None) == bool(ok), (h, hk, dh)
    assert not lib.bad_stride(64, 64) and lib.bad_stride(63, 64) and lib.bad_stride(-1, 64)
    assert lib.bad_stride(2**31, 64)
    # 256 threads each: 2^32 - 1 at most
    assert not lib.bad_grid(2**24 - 1) and lib.bad_grid(2**24)


def test_packed_totals(lib):
    def total(*lengths):
        a = np.array(lengths, np.int64)
        return lib.packed_total(a.ctypes.data, len(a))
    assert total() == 0 and total(0, 0) == 0 and total(3, 0, 5) == 8
    assert total(2**30) == 2**30 and total(2**30, 1) == -1 and total(5, -1) == -1
    assert total(2**62, 2**62, 2**62) == -1


def test_null_contexts_are_refused():
    lib, out = L.load(), ctypes.c_void_p()
    c = _cache()
    assert lib.numrs_hip_seqs_create(None, None, 0, ctypes.byref(out)) == L.E_INVALID
    assert lib.numrs_hip_seqs_destroy(None) == 0 and lib.numrs_hip_seqs_total(None) == -1
    assert lib.numrs_hip_attention_packed_forward(None, None, *[None, 8, None, None, 8, None, 8, None],
                                                  1, 1, 8) == L.E_INVALID
    assert lib.numrs_hip_attention_packed_backward(
        None, None, None, 8, None, None, 8, None, None, 8, None, None, None, None, 1, 1, 8, 0) == L.E_INVALID
    for fn in (lib.numrs_hip_kv_cache_write, lib.numrs_hip_kv_cache_read):
        assert fn(None, ctypes.byref(c), None, None, None, 8, None, 1, None) == L.E_INVALID
    assert lib.numrs_hip_attention_paged(None, ctypes.byref(c), None, 8, 1, None, 1, None, 1, None,
                                         8) == L.E_INVALID
    assert lib.numrs_hip_tensor_attention_packed_qkv(None, None, 1, 1, ctypes.byref(out)) == L.E_INVALID
    assert lib.numrs_hip_tensor_attention_packed(None, None, None, None, 1, 1,
                                                 ctypes.byref(out)) == L.E_INVALID
    assert lib.numrs_hip_tensor_attention_paged(None, None, 1, None, 1, None,
                                                ctypes.byref(out)) == L.E_INVALID
