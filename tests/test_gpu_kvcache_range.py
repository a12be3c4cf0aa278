"""Attention over a paged cache where cached values differ in size, against float64 with the bounds of
test_gpu_packed.py: a score is one product here, so its error is that of its roundings, ten operations'
worth of it, for the keys that a row attends to (a probability above 2^-100)."""
import ctypes
import math

import numpy as np
import pytest

import numrs_amd as nr
from conftest import assert_bits, rand
from numrs_amd import _lib as L
from numrs_amd import nn
from test_gpu_kvcache import U2, _Paged, _stands_for

pytestmark = pytest.mark.gpu


def _run(c, s, q, k, v, H):
    """Rows written into the cache of `s` and attended to by one query a sequence: [n, H, dh]."""
    n, dh = len(s.lengths), s.dh
    s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
    out, qd = c.empty((n, H * dh)), c.to_device(q)
    c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(s.cache.pages), qd.ptr, H * dh, H,
                                                s.td.ptr, s.table.shape[1], s.ends.ptr, n, out.ptr, H * dh))
    return out.numpy().reshape(n, H, dh)


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("n", [40, 1500])
@pytest.mark.parametrize("gap", [0, 13, 20, 30, 60, 500])
def test_a_value_far_above_the_others(hip_ctx, gap, n, format):
    """A token with 2^-gap of the others' probability and a value 2^min(gap, 60) times theirs; of 500, none of it."""
    c, H, Hk, dh, rng = hip_ctx, 8, 2, 64, np.random.default_rng(gap + n)
    s = _Paged(c, [n, 70], 16, Hk, dh, format, rng)
    T = n + 70
    k, v, q = np.zeros((T, Hk * dh), np.float32), rand(rng, (T, Hk * dh)), np.zeros((2, H * dh), np.float32)
    q[:, ::dh] = 8
    # a row of one value has the code 127 for it: the cache holds it to a rounding
    k[:, ::dh] = rng.uniform(-1, 1, (T, Hk)).astype(np.float32)
    for at in (7, n + 33):
        k[at, ::dh] = -np.float32(gap * math.log(2))
        v[at] *= np.float32(2.0 ** min(gap, 60))
    got = _run(c, s, q, k, v, H)
    K, V = (_stands_for(x.reshape(T, Hk, dh), format).astype(np.float64) for x in (k, v))
    at = 0
    for i, m in enumerate(s.lengths):
        for h in range(H):
            x, y = K[at:at + m, h // (H // Hk), 0], V[at:at + m, h // (H // Hk)]
            p = np.exp(x - x.max())
            p /= p.sum()
            f = 2 * U2 * 10 * abs(x[p > 2.0 ** -100]).max() + U2 * (m + 8)
            ref, err = p @ y, f * (p @ abs(y))
            d = abs(got[i, h] - ref)
            assert (d <= err).all(), f"row {i}, head {h}: off by {(d / err).max():.2g} of the bound"
            # besides the worst case: sums of fp32 terms, and a score's three roundings at the gap's size
            norm = 2e-6 + 3 * min(gap, 60) * math.log(2) * U2 / 2
            assert np.linalg.norm(d) <= norm * np.linalg.norm(ref), f"row {i}, head {h}: {np.linalg.norm(d):.2g}"
        at += m


def test_the_lowest_scores(hip_ctx):
    """One token whose score, in base 2, lies between fp32's lowest and -3.4e38: its value is the result."""
    c, H, Hk, dh = hip_ctx, 2, 1, 64
    s = _Paged(c, [1], 16, Hk, dh, "int8", np.random.default_rng(0))
    k, q = np.zeros((1, dh), np.float32), np.zeros((1, H * dh), np.float32)
    v = rand(np.random.default_rng(1), (1, dh))
    k[0, 0] = -2.0 ** 66
    q[0, ::dh] = 3.4015e38 / (math.log2(math.e) / 8) / 2.0 ** 66
    got = _run(c, s, q, k, v, H)
    want = _stands_for(v.reshape(1, Hk, dh), "int8").reshape(dh)
    assert (abs(got[0] - want) <= 9 * U2 * abs(want)).all()


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_shared_pages_of_a_large_and_of_a_small_cache(hip_ctx, format):
    """600 sequences on the same 64 pages, 1.2 GB and more read by one call: the pages of a cache of 260 MB and
    more, which is read past the caches, and of one that is said to end behind them, which is not."""
    c, rng, page, H, Hk, dh, n = hip_ctx, np.random.default_rng(29), 64, 4, 2, 128, 600
    token = Hk * dh * (8 if format == "f32" else 2)
    cache = nr.KVCache(270_000_000 // (token * page), page, Hk, dh, format, ctx=c)
    seqs, table = nr.PackedSequences([4096], ctx=c), c.to_device(np.arange(64, dtype=np.int32)[None])
    k, v = (c.to_device(rand(rng, (4096, Hk * dh))) for _ in range(2))
    cache.write(seqs, k, v, table, c.to_device(np.array([4096], np.int32)))
    lengths = rng.integers(3900, 4097, n).astype(np.int32)
    q, ends = c.to_device(rand(rng, (n, H * dh))), c.to_device(lengths)
    td = c.to_device(np.repeat(np.arange(64, dtype=np.int32)[None], n, 0))
    got = []
    for pages in (cache.pages.pages, 64):
        cache.pages.pages = pages
        out = c.empty((n, H * dh))
        c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(cache.pages), q.ptr, H * dh, H, td.ptr,
                                                    64, ends.ptr, n, out.ptr, H * dh))
        got.append(out.numpy())
    assert np.isfinite(got[0]).all() and (got[0] != 0).any(1).all()
    assert_bits(got[1], got[0])


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_more_rows_than_the_caches_hold(hip_ctx, format):
    """134 MB of keys and values, which are written and read back past the caches, and one row fewer, which are
    not: to the bit."""
    c, rng, page, Hk, dh, n = hip_ctx, np.random.default_rng(30), 256, 8, 128, 2 ** 14 + 1
    k, v = rand(rng, (n, Hk * dh)), rand(rng, (n, Hk * dh))
    kd, vd = c.to_device(k), c.to_device(v)
    pages = -(-n // page)
    table = c.to_device(np.arange(pages, dtype=np.int32)[None])
    for m in (n, n - 1):
        cache, seqs = nr.KVCache(pages, page, Hk, dh, format, ctx=c), nr.PackedSequences([m], ctx=c)
        ends = c.to_device(np.array([m], np.int32))
        cache.write(seqs, kd, vd, table, ends)
        for got, x in zip(cache.read(seqs, table, ends), (k, v)):
            assert_bits(got.numpy(), _stands_for(x[:m].reshape(m, Hk, dh), format).reshape(m, Hk * dh))


def test_decode_that_would_be_recorded_leaves_the_cache(hip_ctx):
    """A step outside no_grad() is refused before anything is written."""
    before = nr.default_context()
    nr.set_default_context(hip_ctx)
    try:
        c, rng, d, H, Hk, dh = hip_ctx, np.random.default_rng(31), 32, 4, 2, 16
        attn = nn.CausalSelfAttention(*(rand(rng, s, 0.2) for s in ((H * dh, d), (Hk * dh, d), (Hk * dh, d), (d, H * dh))),
                                      heads=H, kv_heads=Hk)
        s = _Paged(c, [5, 20], 16, Hk, dh, "f32", rng)
        for a in (s.cache.k, s.cache.v):
            a.fill(3.0)
        ones, x = nr.PackedSequences([1, 1]), nr.Tensor.new(rand(rng, (2, d)))
        with pytest.raises(nr.HipError, match="no backward"):
            attn.decode(x, ones, s.cache, s.td, s.ends)
        assert all((a == 3).all() for a in s.raw())
        with nr.no_grad():
            attn.decode(x, ones, s.cache, s.td, s.ends)
        assert not (s.raw()[0] == 3).all()
    finally:
        nr.set_default_context(before)
